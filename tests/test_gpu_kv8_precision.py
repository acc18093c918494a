"""Precision of the 8-bit cache: weights of the attention for every row tile and code type, and what a rejected token leaves.

Bounds, against the softmax in 64 bits over the cache's own values.  The output
is rounded once to bf16: 2^-8 of the value.  A weight is the sum of two bf16
numbers: the first leaves at most 2^-8 of it, the second at most 2^-8 of that,
so 2^-16 of the weight.  Scores of a few units in fp32 move a weight by 2^-18 or
so (a product of 128 terms in 8 steps), the base-two exponential by 2^-22, and
sums over a few hundred positions by 2^-18; together they stay below another
2^-16.  So an element is off by at most 2^-8 of its size and 2^-15 of the
weighted mean of |v|.
"""
from __future__ import annotations

import math

import pytest
import torch

from wal2026_b200.kv8 import (CODE_MAX, PagedKV8Cache, kv8_append, kv8_attention, kv8_attention_workspace,
                              kv8_read)

from .test_gpu_kv8 import DEV, E4M3, INT8, _attention64, _filled, _gen, _i32, _tables

pytestmark = pytest.mark.gpu
ROWS = [8, 16, 24, 32, 48, 64, 96]  # query rows per kv head: one call of each row tile


def _attend(cache, q, table, lens, scale=None):
    B, hq = table.shape[0], q.shape[1] // cache.head_dim
    out = torch.full(q.shape, float("nan"), dtype=torch.bfloat16, device=DEV)
    kv8_attention(cache, 0, q, table, _i32(lens), out, kv8_attention_workspace(cache, B, hq, q.shape[0] // B), scale=scale)
    return out.double()


def _bound(want, mag):
    return 2.0 ** -8 * want.abs() + 2.0 ** -15 * mag + 1e-30


def _check(out, want, mag):
    bad = ~((out - want).abs() <= _bound(want, mag))  # a NaN is bad too
    assert not bool(bad.any()), (int(bad.sum()), float((out - want).abs().max()))


@pytest.mark.parametrize("above", [7.9, 7.9972, 7.998, 7.9999, 8.0, 8.1])
@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("rows", ROWS)
def test_a_later_score_just_above_the_running_maximum(rows, dtype, above):
    # the running maximum may lag by 8: weights near 2^8, blocks of one V scale.  The tiles of positions 0 and 128 go to
    # one warp group, whatever the row tile, and one CTA takes the whole sequence.
    P, n = 64, 160
    for hd in (64, 128):
        cache = _filled(1, 3, 1, P, hd, dtype, rows)
        cache.codes.view(torch.uint8)[0, 0] = 0
        cache.codes[0, 0, 2, 0, 0, 0] = 1
        cache.scales[:] = 1.0
        q = torch.zeros(1, rows * hd, dtype=torch.bfloat16, device=DEV)
        q.view(rows, hd)[:, 0] = 1.0
        table, scale = _i32([[0, 1, 2]]), above * math.log(2.0)
        _check(_attend(cache, q, table, [n - 1], scale), *_attention64(cache, 0, q, table, [n - 1], [1], scale))


@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("rows,T", [(r, 1) for r in ROWS] + [(20, 5), (36, 9), (130, 65)])
def test_outputs_within_the_stated_precision(rows, T, dtype):
    P, hd, lens = 32, 128, [0, 300, 77]
    ends = [n + T for n in lens]
    pages = sum(-(-n // P) for n in ends)
    cache = _filled(1, pages, 2, P, hd, dtype, rows)
    table = _tables(ends, P, pages, 2)
    q = torch.randn(3 * T, 2 * (rows // T) * hd, device=DEV, generator=_gen(rows)).to(torch.bfloat16)
    _check(_attend(cache, q, table, lens), *_attention64(cache, 0, q, table, lens, [T] * 3, hd ** -0.5))


@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("rows", ROWS)
def test_both_parts_of_a_weight_count(rows, dtype):
    # two positions of opposite values and nearly equal weights: what is left is what one bf16 weight would lose
    P, hd = 16, 64
    cache = PagedKV8Cache.allocate(1, 1, 1, hd, page_size=P, dtype=dtype, device=DEV)
    top = CODE_MAX[dtype]
    cache.codes[0, 0, 0, 0, 1, 0] = -1
    cache.codes[0, 1, 0, 0, 0], cache.codes[0, 1, 0, 0, 1] = top, -top
    cache.scales[:] = 1.0
    q = torch.zeros(1, rows * hd, dtype=torch.bfloat16, device=DEV)
    q.view(rows, hd)[:, 0] = torch.linspace(0.001, 0.08, rows, device=DEV)
    table = _i32([[0]])
    want, mag = _attention64(cache, 0, q, table, [1], [1], 1.0)
    _check(_attend(cache, q, table, [1], 1.0), want, mag)
    x = torch.exp(-q.double().view(rows, hd)[:, :1])  # weight of the second position over the first's
    once = (top * (1 - x.to(torch.bfloat16).double()) / (1 + x)).expand(rows, hd).reshape(1, -1)
    assert bool(((once - want).abs() > _bound(want, mag)).any())  # the bound would show a weight of one bf16 number


@pytest.mark.parametrize("dtype", [E4M3, INT8])
def test_a_rejected_token_leaves_its_scale(dtype):
    # a large draft re-rounds the earlier codes of its block once, and later tokens keep its scale; a block that the
    # draft itself began is begun anew
    P, hd, top = 16, 64, CODE_MAX[dtype]
    cache = PagedKV8Cache.allocate(1, 2, 1, hd, page_size=P, dtype=dtype, device=DEV)
    rows = torch.randn(12, 3 * hd, device=DEV, generator=_gen(4)).to(torch.bfloat16)
    big, table, q = rows[10:11] * 50, _i32([[1, 0]]), torch.empty(12, hd, dtype=torch.bfloat16, device=DEV)

    def append(x, n):
        kv8_append(cache, 0, x, 1, table, _i32([n]), q[:x.shape[0]])

    def read(n):
        k, v = (torch.empty(1, 1, n, hd, device=DEV) for _ in range(2))
        kv8_read(cache, 0, table, _i32([0]), _i32([n]), k, v)
        return torch.stack([k, v]).double()

    append(rows[:10], 0)
    before = read(10)
    append(big, 10)
    scale = cache.scales[0, :, 1, 0].clone()
    assert torch.equal(scale, big.float().view(3, hd)[1:].abs().amax(1) * (torch.ones((), device=DEV) / top))
    after, s = read(10), scale.double().view(2, 1, 1, 1, 1)
    step = s if dtype == INT8 else (before.abs() * 2.0 ** -3).clamp(min=2.0 ** -9 * s)  # between codes
    assert bool(((after - before).abs() <= 0.5 * step + 1e-6 * before.abs()).all())
    append(rows[11:], 10)  # in the draft's place
    assert torch.equal(cache.scales[0, :, 1, 0], scale) and torch.equal(read(10).float(), after.float())
    append(rows[:6], 10)   # up to the block's end
    append(big, 16)        # begins the next block
    append(rows[11:], 16)
    assert torch.equal(cache.scales[0, :, 0, 0], rows[11].float().view(3, hd)[1:].abs().amax(1) * (torch.ones((), device=DEV) / top))
