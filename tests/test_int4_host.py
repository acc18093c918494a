"""What the 4-bit linear refuses and how it quantises, without a GPU."""
from __future__ import annotations

import ctypes

import pytest
import torch

from wal2026_b200 import _abi
from wal2026_b200.int4 import Int4Linear, quantize_int4

ARG, SHAPE, ALIGN = _abi.WAL_ERR_INVALID_ARGUMENT, _abi.WAL_ERR_SHAPE, _abi.WAL_ERR_ALIGNMENT
UNSUPPORTED = _abi.WAL_ERR_UNSUPPORTED
P256 = 0x10000  # an aligned address that no refused call touches


def _layer(**kw):
    return _abi.Int4Layer(**(dict(out_features=32, in_features=256, group_size=64, packed=P256, scales=P256, zeros=None, bias=None) | kw))


GEMV = dict(layer=None, x=P256, x_dtype=_abi.WAL_BF16, M=2, ldx=256, y=P256, ldy=32, y_dtype=_abi.WAL_F32, stream=None)
DEQUANT = dict(layer=None, w=P256, ldw=256, dtype=_abi.WAL_F32, stream=None)
PACK = dict(layer=None, codes=P256, scales=P256, zeros=None, stream=None)


def _call(name, args, layer=None, **change):
    args = dict(args, **change)
    args["layer"] = None if layer is None else ctypes.byref(layer)
    return getattr(_abi.load(), name)(*args.values())


@pytest.mark.parametrize("name,args", [("wal_int4_gemv", GEMV), ("wal_int4_dequant", DEQUANT), ("wal_int4_pack", PACK)])
def test_entry_points_refuse_bad_layers(name, args):
    assert _call(name, args) == ARG
    for change, want in ((dict(packed=None), ARG), (dict(scales=None), ARG), (dict(group_size=48), UNSUPPORTED),
                         (dict(out_features=0), SHAPE), (dict(in_features=0), SHAPE), (dict(in_features=96), SHAPE),
                         (dict(out_features=(1 << 30) + 1), SHAPE), (dict(in_features=1 << 31), SHAPE),
                         (dict(packed=P256 + 8), ALIGN), (dict(scales=P256 + 2), ALIGN), (dict(zeros=P256 + 1), ALIGN)):
        assert _call(name, args, _layer(**change)) == want, change


@pytest.mark.parametrize("change,want", [
    (dict(x=None), ARG), (dict(y=None), ARG), (dict(x_dtype=_abi.WAL_F32), UNSUPPORTED), (dict(y_dtype=3), UNSUPPORTED),
    (dict(M=0), SHAPE), (dict(M=1 << 31), SHAPE), (dict(ldx=248), SHAPE), (dict(ldy=31), SHAPE), (dict(x=P256 + 8), ALIGN),
    (dict(ldx=260), ALIGN), (dict(y=P256 + 2), ALIGN)])
def test_gemv_refusals(change, want):
    assert _call("wal_int4_gemv", GEMV, _layer(), **change) == want


def test_dequant_and_pack_refusals():
    assert _call("wal_int4_dequant", DEQUANT, _layer(), w=None) == ARG
    assert _call("wal_int4_dequant", DEQUANT, _layer(), ldw=255) == SHAPE
    assert _call("wal_int4_dequant", DEQUANT, _layer(), dtype=7) == UNSUPPORTED
    assert _call("wal_int4_dequant", DEQUANT, _layer(), w=P256 + 2) == ALIGN
    assert _call("wal_int4_pack", PACK, _layer(), codes=None) == ARG
    assert _call("wal_int4_pack", PACK, _layer(), scales=None) == ARG
    assert _call("wal_int4_pack", PACK, _layer(), zeros=P256) == ARG  # the layer has no place for them
    assert _call("wal_int4_pack", PACK, _layer(zeros=P256)) == ARG
    assert _abi.load().wal_int4_packed_size(32, 256, 64, None, None) == ARG


def test_packed_size():
    nb, ne = ctypes.c_size_t(0), ctypes.c_size_t(0)
    assert _abi.load().wal_int4_packed_size(33, 96, 32, ctypes.byref(nb), ctypes.byref(ne)) == _abi.WAL_OK
    assert nb.value == 3 * 2 * 512 and ne.value == 3 * 16 * 3


def test_quantize_codes_and_refusals():
    w = torch.tensor([[-7.5, 0.0, 3.0, 7.0] * 8, [0.0] * 32])
    codes, scale, zero = quantize_int4(w, 32)
    assert scale.tolist() == [[1.0], [0.0]] and zero is None
    assert codes[0, :4].tolist() == [0, 8, 11, 15] and codes[1].tolist() == [8] * 32
    codes, scale, zero = quantize_int4(torch.linspace(1.0, 16.0, 32)[None], 32, zero_points=True)
    assert zero.tolist() == [[0]] and int(codes.max()) == 15
    for bad in (dict(group_size=48), dict(group_size=64)):
        with pytest.raises(ValueError):
            quantize_int4(w, **bad)
    w[0, 0] = float("inf")
    with pytest.raises(ValueError):
        quantize_int4(w, 32)


def test_module_refusals():
    codes, scales = torch.zeros(4, 64, dtype=torch.uint8), torch.ones(4, 1, dtype=torch.float16)
    for args in ((codes.int(), scales), (codes[0], scales), (codes, scales.float()), (codes, scales[:3]),
                 (codes, torch.ones(4, 4, dtype=torch.float16)), (codes, scales, torch.zeros(4, 1)),
                 (codes, scales, None, torch.zeros(5)), (codes, scales)):
        with pytest.raises(ValueError):
            Int4Linear(*args)
