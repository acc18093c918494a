"""What casts, copies and replaced buffers do to a 4-bit linear, without a GPU."""
from __future__ import annotations

import copy
import pickle

import pytest
import torch
from torch import nn

from wal2026_b200.int4 import Int4Linear

BUFFERS = ("packed", "scales", "zeros", "bias")


def _linear(zeros=True, bias=True):
    """A layer of 16 x 64 as its constructor leaves it, but for the packing, which runs on the GPU."""
    layer = object.__new__(Int4Linear)
    nn.Module.__init__(layer)
    layer.group_size, layer.out_features, layer.in_features = 64, 16, 64
    g = torch.Generator().manual_seed(1)
    layer.register_buffer("packed", torch.randint(0, 256, (512,), dtype=torch.uint8, generator=g))
    layer.register_buffer("scales", torch.rand(16, generator=g).to(torch.float16))
    layer.register_buffer("zeros", torch.randint(0, 16, (16,), dtype=torch.uint8, generator=g) if zeros else None)
    layer.register_buffer("bias", torch.randn(16, generator=g).to(torch.bfloat16) if bias else None)
    layer._layer_cache = None
    layer.layer_struct()
    return layer


def _same(a, b):
    for name in BUFFERS:
        x, y = getattr(a, name), getattr(b, name)
        assert (x is None) == (y is None)
        assert x is None or (x.dtype == y.dtype and torch.equal(x, y)), name


@pytest.mark.parametrize("cast", ["bfloat16", "half", "float", "double"])
@pytest.mark.parametrize("inside", [False, True])
def test_casts_leave_the_weights_alone(cast, inside):
    layer, want = _linear(), _linear()
    holder = nn.ModuleDict({"layer": layer, "other": nn.Linear(4, 4)}) if inside else layer
    getattr(holder, cast)()
    _same(layer, want)
    holder.to(dtype=getattr(torch, {"half": "float16", "float": "float32", "double": "float64"}.get(cast, cast)))
    _same(layer, want)
    if inside:
        assert holder["other"].weight.dtype != torch.float32 or cast == "float"
    s = layer.layer_struct()
    assert (s.packed, s.scales, s.zeros, s.bias) == tuple(getattr(layer, n).data_ptr() for n in BUFFERS)


def test_type_and_meta_device():
    layer, want = _linear(), _linear()
    layer.type(torch.float32)
    _same(layer, want)
    layer.to("meta", torch.float32)
    assert all(getattr(layer, n).device.type == "meta" for n in BUFFERS)
    assert [getattr(layer, n).dtype for n in BUFFERS] == [getattr(want, n).dtype for n in BUFFERS]


@pytest.mark.parametrize("name,dtype", [("scales", torch.bfloat16), ("scales", torch.float32), ("bias", torch.float16),
                                        ("packed", torch.int32), ("zeros", torch.int16)])
def test_buffers_of_another_type_are_refused(name, dtype):
    layer = _linear()
    setattr(layer, name, getattr(layer, name).to(dtype))
    with pytest.raises(ValueError):
        layer.layer_struct()


def test_copies_have_their_own_buffers():
    layer = _linear(zeros=False)
    for other in (copy.deepcopy(layer), pickle.loads(pickle.dumps(layer))):
        _same(other, layer)
        assert other.layer_struct().packed == other.packed.data_ptr() != layer.packed.data_ptr()
    assert layer.layer_struct().packed == layer.packed.data_ptr()
