"""The softmax of the rules on logits where logits are far from zero or temperatures far from one.

Logits here meet no rule but the temperature, so they enter exactly and only
differences to the largest one matter.  With D = (largest - x) / temperature, an
exponent -D is a difference, a constant over the temperature and a product, each within
2^-24 of itself, and the constant's own rounding: 4 * 2^-24 * D in all, in one step or
two (an entry to its CTA's largest, that to the row's).  An exponential is within
2^-22; there are two.  The sum of positive terms takes at most 48 additions in a
thread and 20 between threads, warps and CTAs, 2^-24 each, and is off by the mean of
what its terms are, 4 * 2^-24 * E[D]; three more roundings make the result.  So a
probability is compared relative to
    4 * 2^-24 * (D + E[D]) + 4 * 2^-22 + 72 * 2^-24,
and 2^-126 absolutely (smaller exponentials count as 0).
"""
from __future__ import annotations

import pytest
import torch

from wal2026_b200.logits import logit_rules

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32 = torch.float32


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _softmax(logits, temperature):
    """(probabilities, bound) in 64 bits; a quotient past fp32's range counts as an infinity."""
    t = temperature.double()[:, None, None]
    x = logits.double()
    q = x / t
    q = torch.where(q.float().isinf(), q.float().double(), q)
    top, most = q.amax(-1, keepdim=True), x.amax(-1, keepdim=True)
    d = torch.where(q == float("-inf"), float("inf"), torch.where(q == top, 0.0, (most - x) / t))
    e = torch.exp(-d)
    p = e / e.sum(-1, keepdim=True)
    mean = (p * torch.where(p > 0, d, 0.0)).sum(-1, keepdim=True)
    rel = 4 * 2.0 ** -24 * (torch.where(d.isinf(), 0.0, d) + mean) + 4 * 2.0 ** -22 + 72 * 2.0 ** -24
    return p.nan_to_num(0.0), (p * rel).nan_to_num(0.0) + 2.0 ** -126


def _check(logits, temperature=None):
    B, T, V = logits.shape
    out = torch.full((B, T, V), float("nan"), device=DEV)
    logit_rules(logits, out, temperature=temperature)
    want, bound = _softmax(logits, torch.ones(B, device=DEV) if temperature is None else temperature)
    off = (out.double() - want).abs()
    assert bool((off <= bound).all()), (float((off / bound).nan_to_num(9e9).max()), int((~(off <= bound)).sum()))
    assert bool(((out.double().sum(-1) - 1).abs() < 2.0 ** -16).all())
    return out


def _blocks(V, which):
    """Entries of some of the eight CTAs that share a row of V > 16384: blocks of 128 are dealt out in turn."""
    i = torch.arange(V, device=DEV)
    return torch.isin((i >> 7) & 7, torch.tensor(which, device=DEV))


@pytest.mark.parametrize("low", [-1e4, -1e6, -1e9, -1e10, -1e20, -1e29, -1e33, torch.finfo(F32).min, float("-inf")])
@pytest.mark.parametrize("V", [300, 5000, 20000, 150001])
def test_rows_masked_by_low_numbers(low, V):
    temps = torch.tensor([0.1, 0.3, 0.5, 0.7, 0.8, 1.0, 1.2, 1e-3], device=DEV)
    B = len(temps)
    logits = 3 * torch.randn(B, 2, V, device=DEV, generator=_gen(V))
    # whole CTAs are left with nothing else, and in the second rows scattered entries too
    logits[:, :, _blocks(V, [1, 4, 5])] = low
    logits[:, 1][torch.rand(B, V, device=DEV, generator=_gen(1)) < 0.3] = low
    _check(logits, temps)
    _check(logits)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, F32])
def test_rows_all_of_one_low_number(dtype):
    for low in (-1e4, -6e4) if dtype == torch.float16 else (-1e9, -1e10, -1e20, -1e29, 1e10, 1e29, 3e38, -3e38):
        for V in (7, 300, 20000):
            logits = torch.full((2, 1, V), low, device=DEV).to(dtype)
            out = _check(logits, torch.tensor([1.0, 1.3], device=DEV))
            assert bool((out - 1.0 / V).abs().max() <= 2.0 ** -20 / V)


@pytest.mark.parametrize("V", [1000, 20000, 140000])
@pytest.mark.parametrize("temp", [1e-38, 1e-20, 1e-12, 2.0 ** -40 * (1 - 2.0 ** -24), 2.0 ** -40, 1e-9, 1e-8, 1e-6, 1e-4, 0.01, 0.1, 3.0,
                                  1e6, 2.0 ** 40, 2.0 ** 40 * (1 + 2.0 ** -23), 1e30, 3e38, float("inf")])
def test_temperatures_of_every_size(V, temp):
    g = _gen(V)
    logits = 8 * torch.randn(4, 2, V, device=DEV, generator=g)
    logits[1] += 30.0
    logits[2] = 18.75 + logits[2] * 1e-3
    logits[3, :, 5] = logits[3, :, V - 1] = logits[3].amax(-1)  # a tie, in different CTAs of longer rows
    t = torch.full((4,), temp, device=DEV)
    _check(logits, t)
    _check(logits.to(torch.bfloat16), t)


@pytest.mark.parametrize("temp", [0.01, 0.1, 0.6, 1.0])
@pytest.mark.parametrize("shift", [0.0, 1e2, 1e4, 3e5, 2e6, 1e7])
def test_logits_away_from_zero(temp, shift):
    logits = 2 * torch.randn(8, 3, 33000, device=DEV, generator=_gen(3)) + shift
    logits[4:] -= 2 * shift
    _check(logits, torch.full((8,), temp, device=DEV))


def test_numbers_at_both_ends_of_the_range():
    big = torch.finfo(F32).max
    logits = torch.randn(6, 1, 20000, device=DEV, generator=_gen(7))
    logits[:, 0, 17], logits[:, 0, 9000] = -big, big
    logits[1, 0, 9001] = big * (1 - 2.0 ** -20)
    logits[2] = logits[2] * (big / 8)
    logits[3] = logits[3] * 1e-40
    logits[4] = logits[4] * (big / 8)
    logits[4, 0, 9000] = 0.0
    _check(logits, torch.tensor([1.0, big / 4, big / 2, 1e-40, 1e38, 0.25], device=DEV))


def test_an_infinite_temperature_and_infinite_logits():
    inf = float("inf")
    logits = torch.randn(3, 1, 20000, device=DEV, generator=_gen(8))
    logits[0, 0, 4], logits[0, 0, 9000], logits[1, 0, 5] = inf, inf, -inf  # inf / inf is no number: left out
    logits[2] = -inf
    out = torch.full_like(logits, float("nan"))
    logit_rules(logits, out, temperature=torch.full((3,), inf, device=DEV))
    assert bool((out[2] == 0).all())
    for b in range(2):
        left = logits[b, 0].isfinite()
        assert bool((out[b, 0, ~left] == 0).all())
        assert bool(((out[b, 0, left] * int(left.sum()) - 1).abs() < 2.0 ** -20).all())
