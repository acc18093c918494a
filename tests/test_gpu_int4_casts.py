"""4-bit linears on the GPU after their module, or the stack that holds them, was cast, copied or moved."""
from __future__ import annotations

import copy

import pytest
import torch

from tests.test_gpu_int4 import BF, DEV, F32, _check, _gen, _layer
from wal2026_b200.llama import LlamaShape, dense_llama

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cast", ["bfloat16", "half", "float", "double"])
def test_int4_products_after_a_cast(cast):
    layer, w = _layer(200, 512, 64, True, 6, bias=True)
    x = torch.randn(3, 512, device=DEV, generator=_gen(5)).to(BF)
    want, y = torch.empty(3, 200, device=DEV), torch.empty(3, 200, device=DEV)
    layer.gemv_into(x, want)
    dense = layer.reconstruct_weight(F32)
    getattr(layer, cast)()
    layer.gemv_into(x, y)
    assert torch.equal(y, want) and torch.equal(layer.reconstruct_weight(F32), dense)
    _check(layer, w, x, y)
    layer.cpu().to(DEV, dtype=getattr(torch, {"half": "float16"}.get(cast, cast if cast == "bfloat16" else "float32")))
    layer.gemv_into(x, y)
    assert torch.equal(y, want)


def test_a_cast_stack_keeps_its_4_bit_head():
    stack = dense_llama(LlamaShape(layers=1, hidden=256, mlp=512, heads=4, kv_heads=2, vocab=1000), seed=3)
    stack.quantize_head(64, zero_points=True)
    x = torch.randn(5, 256, device=DEV, generator=_gen(1)).to(BF)
    want = stack.logits(x)
    stack.to(torch.bfloat16)
    assert torch.equal(stack.logits(x), want)


def test_int4_copies_multiply_alone():
    layer, _ = _layer(48, 256, 32, True, 2, bias=True)
    x = torch.randn(2, 256, device=DEV, generator=_gen(3)).to(BF)
    want, y = torch.empty(2, 48, device=DEV), torch.empty(2, 48, device=DEV)
    layer.gemv_into(x, want)
    other = copy.deepcopy(layer)
    layer.packed.zero_()
    other.gemv_into(x, y)
    assert torch.equal(y, want)
