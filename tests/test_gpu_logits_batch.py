"""Rules on logits where clusters of CTAs take several rows, and where vocabularies take the largest kernel.

The reference and its tolerance are those of ``test_gpu_logits``.
"""
from __future__ import annotations

import pytest
import torch

from tests.test_gpu_logits import BF, DEV, F32, HF, _check, _f32, _i32, _inputs
from wal2026_b200.logits import logit_rules, pack_mask

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("B,T,V", [(40, 3, 33000), (30, 5, 16388), (150, 3, 5000), (140, 4, 2047)])
def test_every_rule_where_rows_exceed_the_clusters(dtype, B, T, V):
    # 32 clusters of eight CTAs, 64 of four and 256 single CTAs run at a time, so each has rows of several sequences
    logits, rules, allowed = _inputs(B, T, V, 120, 5, dtype, V + B)
    _check(logits, allowed, **rules)
    rules["new_lens"] = _i32([(T, 1, 0, T - 1)[b % 4] for b in range(B)])
    _check(logits, allowed, **rules)
    _check(logits, allowed, softmax=False, **rules)


def test_a_row_gives_the_same_bits_alone_and_in_a_batch():
    B, T, V = 50, 4, 20000
    logits, rules, allowed = _inputs(B, T, V, 400, 7, BF, 31)
    out = _check(logits, allowed, **rules)
    mask = pack_mask(allowed)
    for b in (0, 1, 17, 31, 32, 49):
        one = torch.empty(1, T, V, device=DEV)
        logit_rules(logits[b:b + 1], one, mask=mask[b:b + 1], **{k: v[b:b + 1] for k, v in rules.items()})
        assert torch.equal(one[0], out[b])


def test_greedy_rows_between_others_of_the_same_clusters():
    B, T, V = 70, 2, 33000
    logits, rules, allowed = _inputs(B, T, V, 60, 3, BF, 8)
    rules["temperature"] = torch.where(torch.arange(B, device=DEV) % 3 == 1, 0.0, rules["temperature"])
    out = _check(logits, allowed, **rules)
    assert bool((out[1::3].amax(-1) == 1).all())


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("V", [131072, 131073, 131076, 151936, 256000, 393215])
def test_every_rule_in_large_vocabularies(dtype, V):
    logits, rules, allowed = _inputs(2, 2, V, 500, 9, dtype, V)
    _check(logits, allowed, **rules)
    _check(logits, allowed, softmax=False, **rules)
    _check(logits, None, temperature=_f32([0.0, 0.7]))


def test_more_rows_than_clusters_in_a_large_vocabulary():
    # 16 clusters of eight CTAs with an SM each
    logits, rules, allowed = _inputs(20, 2, 151936, 90, 4, BF, 3)
    _check(logits, allowed, **rules)
    rules["new_lens"] = _i32([(2, 1, 0)[b % 3] for b in range(20)])
    _check(logits, allowed, **rules)


@pytest.mark.parametrize("V", [151936, 200001])
def test_padding_and_strides_in_a_large_vocabulary(V):
    logits, rules, allowed = _inputs(2, 3, V, 50, 3, BF, V)
    wide = torch.zeros(2, 4, V + 5, dtype=BF, device=DEV)
    wide[:, 1:, 2:2 + V] = logits
    out = torch.full((2, 4, V + 7), 7.0, device=DEV)
    view = out[:, :3, 3:3 + V]
    logit_rules(wide[:, 1:, 2:2 + V], view, mask=pack_mask(allowed), **rules)
    want = _check(logits, allowed, **rules)
    assert torch.equal(view, want) or bool(((view - want).abs() <= want * 2.0 ** -18).all())
    view.fill_(7.0)
    assert bool((out == 7.0).all())  # nothing else was written
