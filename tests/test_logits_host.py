"""What the rules on logits refuse, and their masks, without a GPU."""
from __future__ import annotations

import ctypes

import pytest
import torch

from wal2026_b200 import _abi
from wal2026_b200.logits import LogitRules, logit_rules, pack_mask

ARG, SHAPE, ALIGN = _abi.WAL_ERR_INVALID_ARGUMENT, _abi.WAL_ERR_SHAPE, _abi.WAL_ERR_ALIGNMENT
P256 = 0x10000  # an aligned address that no refused call touches
CALL = dict(rules=None, logits=P256, dtype=_abi.WAL_BF16, ld_seq=2000, ld_row=1000, B=2, T=2, V=1000, out=P256, out_seq=2000,
            out_row=1000, softmax=1, stream=None)


def _rules(**kw):
    base = dict(text=P256, ld_text=50, text_len=50, lens=P256, repetition=P256, bias_ids=P256, bias=P256, num_bias=4, mask=P256,
                mask_seq=64, mask_row=32, temperature=P256)
    return _abi.LogitRules(**(base | kw))


def _call(rules, **change):
    args = dict(CALL, **change)
    args["rules"] = None if rules is None else ctypes.byref(rules)
    return _abi.load().wal_logit_rules_apply(*args.values())


@pytest.mark.parametrize("change,want", [
    (dict(text=None), ARG), (dict(lens=None), ARG), (dict(bias=None), ARG), (dict(bias_ids=None), ARG),
    (dict(bias=None, bias_ids=None), ARG), (dict(num_bias=1025), SHAPE), (dict(num_bias=-1), SHAPE), (dict(ld_text=49), SHAPE),
    (dict(text_len=-1), SHAPE), (dict(text_len=1 << 20, ld_text=1 << 20), SHAPE), (dict(mask_seq=-1), SHAPE), (dict(mask_row=-1), SHAPE)])
def test_rules_refused(change, want):
    assert _call(_rules(**change)) == want


@pytest.mark.parametrize("change,want", [
    (dict(logits=None), ARG), (dict(out=None), ARG), (dict(dtype=5), _abi.WAL_ERR_UNSUPPORTED), (dict(B=0), SHAPE), (dict(T=0), SHAPE),
    (dict(V=0), SHAPE), (dict(V=393217, ld_row=393217, out_row=393217), SHAPE), (dict(B=1 << 20, T=1 << 20), SHAPE),
    (dict(ld_row=999), SHAPE), (dict(ld_seq=-1), SHAPE), (dict(out_row=999), SHAPE), (dict(out_seq=1999), SHAPE),
    (dict(logits=P256 + 1), ALIGN), (dict(out=P256 + 2), ALIGN)])
def test_call_refused(change, want):
    assert _call(None) == ARG
    assert _call(_rules(), **change) == want


def test_masks_are_words_of_32_tokens():
    allowed = torch.zeros(2, 70, dtype=torch.bool)
    allowed[0, [0, 31, 32, 69]] = True
    allowed[1] = True
    words = pack_mask(allowed)
    assert words.dtype == torch.int32 and words.tolist() == [[1 - 2 ** 31, 1, 32], [-1, -1, 63]]


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError):
        logit_rules(torch.zeros(1, 1, 8), torch.zeros(1, 1, 8))
    assert not LogitRules(temperature=torch.ones(1)).penalises() and LogitRules(presence=torch.ones(1)).penalises()
