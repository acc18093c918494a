"""What the groups and the attention of shared prefixes refuse, without a GPU."""
from __future__ import annotations

import ctypes

import pytest
import torch

from wal2026_b200 import _abi
from wal2026_b200.kv8 import kv_pages_groups

ARG, SHAPE, ALIGN = _abi.WAL_ERR_INVALID_ARGUMENT, _abi.WAL_ERR_SHAPE, _abi.WAL_ERR_ALIGNMENT
P256 = 0x10000  # an aligned address that no refused call touches
ATTN = dict(cache=None, layer=1, q=P256, ld_q=256, B=2, T=3, hq=4, table=P256, ld_table=5, max_pages=5, lens=P256,
            new_lens=None, groups=P256, scale=0.1, out=P256, ld_out=256, ws=P256, ws_bytes=1 << 40, status=None, stream=None)
GROUPS = dict(table=P256, ld_table=6, lens=P256, rows=4, width=6, page_size=16, least=32, groups=P256, stream=None)


def _c(**kw):
    base = dict(codes=P256, scales=P256, num_pages=8, layers=2, kv_heads=2, page_size=16, head_dim=64, kind=0)
    return _abi.KV8Cache(**(base | kw))


def _call(name, args, **change):
    args = dict(args, **change)
    if isinstance(args.get("cache"), _abi.KV8Cache):
        args["cache"] = ctypes.byref(args["cache"])
    return getattr(_abi.load(), name)(*args.values())


@pytest.mark.parametrize("change,want", [
    (dict(cache=None), ARG), (dict(cache=_c(head_dim=96)), _abi.WAL_ERR_UNSUPPORTED), (dict(layer=2), SHAPE), (dict(q=None), ARG),
    (dict(table=None), ARG), (dict(lens=None), ARG), (dict(groups=None), ARG), (dict(out=None), ARG), (dict(ws=None), ARG),
    (dict(B=0), SHAPE), (dict(T=0), SHAPE), (dict(hq=5), SHAPE), (dict(max_pages=0), SHAPE), (dict(ld_table=4), SHAPE),
    (dict(ld_q=248), SHAPE), (dict(ld_out=248), SHAPE), (dict(B=4097), SHAPE), (dict(B=1 << 20, T=1 << 20), SHAPE),
    (dict(q=P256 + 8), ALIGN), (dict(out=P256 + 4), ALIGN), (dict(ws=P256 + 16), ALIGN), (dict(ld_q=260), ALIGN),
    (dict(ws_bytes=0), _abi.WAL_ERR_BUFFER_TOO_SMALL), (dict(ws_bytes=1 << 20), _abi.WAL_ERR_BUFFER_TOO_SMALL)])
def test_shared_attention_refusals(change, want):
    assert _call("wal_kv8_attention_shared", dict(ATTN, cache=_c()), **change) == want


def test_shared_workspace_holds_the_plain_one_and_refuses_invalid_shapes():
    lib, ok = _abi.load(), _c()
    sizes = [lib.wal_kv8_attention_shared_workspace(ctypes.byref(ok), 3, T, 4) for T in range(1, 100)]
    assert all(a <= b for a, b in zip(sizes, sizes[1:])) and sizes[0] > lib.wal_kv8_attention_workspace(ctypes.byref(ok), 3, 1, 4)
    for c, B, T, hq in ((None, 1, 1, 2), (ok, 0, 1, 2), (ok, 1, 0, 2), (ok, 1, 1, 0), (ok, 1, 1, 3), (ok, 4097, 1, 2)):
        assert lib.wal_kv8_attention_shared_workspace(None if c is None else ctypes.byref(c), B, T, hq) == 0


def test_groups_refusals():
    for key, value in GROUPS.items():
        if value == P256:
            assert _call("wal_kv_pages_groups", GROUPS, **{key: None}) == ARG, key
    for change in (dict(rows=0), dict(rows=4097), dict(width=0), dict(ld_table=5), dict(page_size=0), dict(least=0),
                   dict(width=1 << 28, ld_table=1 << 28), dict(width=1 << 31, ld_table=1 << 31)):
        assert _call("wal_kv_pages_groups", GROUPS, **change) == SHAPE, change


def test_cpu_tensors_are_refused():
    table = torch.zeros(2, 3, dtype=torch.int32)
    with pytest.raises(ValueError):
        kv_pages_groups(table, torch.zeros(2, dtype=torch.int32), 16, torch.zeros(4, 2, dtype=torch.int32))
