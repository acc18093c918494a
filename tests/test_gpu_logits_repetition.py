"""The repetition penalty divides: a quotient is the nearest fp32 number, so that equal logits stay equal."""
from __future__ import annotations

import pytest
import torch

from wal2026_b200.logits import logit_rules

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _logits(B, V, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return 4 * torch.randn(B, 1, V, device=DEV, generator=g), 1 + torch.rand(B, device=DEV, generator=g)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V", [1000, 5001, 40000, 140000])
@pytest.mark.parametrize("scale", [1.0, 1e-30, 1e30])
def test_penalised_logits_are_the_nearest_numbers(dtype, V, scale):
    x, rep = _logits(3, V, V)
    x, rep = x.to(dtype), rep * scale
    seen = torch.arange(0, V, 3, device=DEV, dtype=torch.int32).repeat(3, 1)
    out = torch.empty(3, 1, V, device=DEV)
    logit_rules(x, out, text=seen, lens=torch.full((3,), seen.shape[1] - 1, dtype=torch.int32, device=DEV), repetition=rep, softmax=False)
    f, r = x.float(), rep[:, None, None]
    want = torch.where(torch.arange(V, device=DEV) % 3 == 0, torch.where(f > 0, f / r, f * r), f)
    assert torch.equal(out, want)


def test_greedy_choice_between_a_penalised_logit_and_its_equal():
    # rows where x * (1 / r) is not the number next to x / r
    x, rep = _logits(4096, 1, 5)
    x = x.abs() + 0.5
    q = x[:, 0, 0] / rep
    off = q != x[:, 0, 0] * (1.0 / rep)
    assert int(off.sum()) > 100
    for first in (0, 1):  # the penalised one before or behind its equal: the first one is taken
        logits = torch.full((4096, 1, 200), -50.0, device=DEV)
        logits[:, 0, 20 if first else 150] = q
        logits[:, 0, 100] = x[:, 0, 0]
        out = torch.empty_like(logits)
        logit_rules(logits, out, text=torch.full((4096, 1), 100, dtype=torch.int32, device=DEV),
                    lens=torch.zeros(4096, dtype=torch.int32, device=DEV), repetition=rep, temperature=torch.zeros(4096, device=DEV))
        assert bool((out[:, 0, 20 if first else 100] == 1.0).all())
