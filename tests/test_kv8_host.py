"""What the paged 8-bit cache and the draft verification refuse, without a GPU."""
from __future__ import annotations

import ctypes

import pytest
import torch

from wal2026_b200 import _abi
from wal2026_b200.kv8 import (PagedKV8Cache, kv8_append, kv8_attention, kv8_attention_workspace, kv8_read,
                              kv_pages_assign, kv_pages_compact, kv_pages_copy)
from wal2026_b200.speculative import verify_drafts

ARG, SHAPE, ALIGN = _abi.WAL_ERR_INVALID_ARGUMENT, _abi.WAL_ERR_SHAPE, _abi.WAL_ERR_ALIGNMENT
UNSUPPORTED, SMALL = _abi.WAL_ERR_UNSUPPORTED, _abi.WAL_ERR_BUFFER_TOO_SMALL
P256 = 0x10000  # an aligned address that no refused call touches


def _c(**kw):
    base = dict(codes=P256, scales=P256, num_pages=8, layers=2, kv_heads=2, page_size=16, head_dim=64, kind=0)
    return _abi.KV8Cache(**(base | kw))


def _call(name, args, **change):
    args = dict(args, **change)
    c = args.get("cache")
    if isinstance(c, _abi.KV8Cache):
        args["cache"] = ctypes.byref(c)
    return getattr(_abi.load(), name)(*args.values())


APPEND = dict(cache=None, layer=1, qkv=P256, ld_qkv=512, B=2, T=3, hq=4, table=P256, ld_table=5, max_pages=5, lens=P256,
              new_lens=None, cos=P256, sin=P256, max_pos=10, q_out=P256, ld_q=256, stream=None)
READ = dict(cache=None, layer=1, B=2, table=P256, ld_table=5, max_pages=5, first=P256, count=P256, L=4, k=P256, v=P256,
            dtype=_abi.WAL_F32, stream=None)
ATTN = dict(cache=None, layer=1, q=P256, ld_q=256, B=2, T=3, hq=4, table=P256, ld_table=5, max_pages=5, lens=P256,
            new_lens=None, scale=0.1, out=P256, ld_out=256, ws=P256, ws_bytes=1 << 40, stream=None)
BAD_CACHE = [(dict(codes=None), ARG), (dict(scales=None), ARG), (dict(num_pages=0), SHAPE), (dict(layers=1), SHAPE),
             (dict(kv_heads=0), SHAPE), (dict(page_size=48), UNSUPPORTED), (dict(head_dim=96), UNSUPPORTED),
             (dict(kind=2), UNSUPPORTED), (dict(codes=P256 + 8), ALIGN)]


@pytest.mark.parametrize("name,args", [("wal_kv8_append", APPEND), ("wal_kv8_read", READ), ("wal_kv8_attention", ATTN)])
def test_entry_points_refuse_bad_caches(name, args):
    assert _call(name, args) == ARG
    for change, want in BAD_CACHE:
        assert _call(name, args, cache=_c(**change)) == want, change
    assert _call(name, args, cache=_c(), layer=2) == SHAPE
    assert _call(name, args, cache=_c(), layer=-1) == SHAPE


@pytest.mark.parametrize("change,want", [
    (dict(qkv=None), ARG), (dict(table=None), ARG), (dict(lens=None), ARG), (dict(q_out=None), ARG), (dict(cos=None), ARG),
    (dict(sin=None), ARG), (dict(B=0), SHAPE), (dict(T=0), SHAPE), (dict(hq=3), SHAPE), (dict(hq=0), SHAPE),
    (dict(max_pages=0), SHAPE), (dict(ld_table=4), SHAPE), (dict(ld_qkv=504), SHAPE), (dict(ld_q=248), SHAPE),
    (dict(max_pos=0), SHAPE), (dict(B=1 << 31), SHAPE), (dict(max_pages=1 << 28, ld_table=1 << 28), SHAPE),
    (dict(qkv=P256 + 2), ALIGN), (dict(q_out=P256 + 8), ALIGN), (dict(cos=P256 + 4), ALIGN), (dict(ld_qkv=516), ALIGN),
    (dict(ld_q=260), ALIGN)])
def test_append_refusals(change, want):
    assert _call("wal_kv8_append", APPEND, cache=_c(), **change) == want


@pytest.mark.parametrize("change,want", [
    (dict(table=None), ARG), (dict(first=None), ARG), (dict(count=None), ARG), (dict(k=None), ARG), (dict(v=None), ARG),
    (dict(dtype=_abi.WAL_F16), UNSUPPORTED), (dict(B=0), SHAPE), (dict(L=0), SHAPE), (dict(max_pages=6), SHAPE),
    (dict(L=1 << 31), SHAPE), (dict(k=P256 + 4), ALIGN), (dict(v=P256 + 8), ALIGN)])
def test_read_refusals(change, want):
    assert _call("wal_kv8_read", READ, cache=_c(), **change) == want


@pytest.mark.parametrize("change,want", [
    (dict(q=None), ARG), (dict(table=None), ARG), (dict(lens=None), ARG), (dict(out=None), ARG), (dict(ws=None), ARG),
    (dict(B=0), SHAPE), (dict(T=0), SHAPE), (dict(hq=5), SHAPE), (dict(max_pages=0), SHAPE), (dict(ld_table=4), SHAPE),
    (dict(ld_q=248), SHAPE), (dict(ld_out=248), SHAPE), (dict(B=1 << 20, T=1 << 20), SHAPE), (dict(q=P256 + 8), ALIGN),
    (dict(out=P256 + 4), ALIGN), (dict(ws=P256 + 16), ALIGN), (dict(ld_q=260), ALIGN), (dict(ld_out=258), ALIGN),
    (dict(ws_bytes=0), SMALL)])
def test_attention_refusals(change, want):
    assert _call("wal_kv8_attention", ATTN, cache=_c(), **change) == want


def test_attention_workspace_of_invalid_shapes_is_zero():
    lib = _abi.load()
    ok = _c()
    assert lib.wal_kv8_attention_workspace(ctypes.byref(ok), 3, 2, 4) > 0
    for c, B, T, hq in ((None, 1, 1, 2), (ok, 0, 1, 2), (ok, 1, 0, 2), (ok, 1, 1, 0), (ok, 1, 1, 3)):
        assert lib.wal_kv8_attention_workspace(None if c is None else ctypes.byref(c), B, T, hq) == 0


def test_attention_workspace_never_shrinks_with_more_tokens():
    lib, c = _abi.load(), _c()
    sizes = [lib.wal_kv8_attention_workspace(ctypes.byref(c), 3, T, 4) for T in range(1, 200)]
    assert all(a <= b for a, b in zip(sizes, sizes[1:]))


ASSIGN = dict(table=P256, ld_table=6, rows_in=3, parent=P256, keep=P256, add=P256, rows=4, width=6, num_pages=9, page_size=16,
              out=P256, ld_out=6, ref=P256, src=P256, dst=P256, info=P256, stream=None)
COMPACT = dict(table=P256, ld_table=6, lens=P256, rows=4, width=6, num_pages=9, page_size=16, out=P256, ld_out=6, remap=P256,
               src=P256, dst=P256, info=P256, stream=None)


@pytest.mark.parametrize("name,args", [("wal_kv_pages_assign", ASSIGN), ("wal_kv_pages_compact", COMPACT)])
def test_page_refusals(name, args):
    for key, value in args.items():
        if value == P256:
            assert _call(name, args, **{key: None}) == ARG, key
    for key in ("rows", "width", "num_pages", "page_size"):
        assert _call(name, args, **{key: 0}) == SHAPE, key
    assert _call(name, args, ld_table=5) == SHAPE and _call(name, args, ld_out=5) == SHAPE
    assert _call(name, args, width=1 << 28, ld_table=1 << 28, ld_out=1 << 28) == SHAPE
    if name == "wal_kv_pages_assign":
        assert _call(name, args, rows=16384) == SHAPE and _call(name, args, rows_in=0) == SHAPE


def test_copy_refusals():
    args = dict(cache=_c(), src=P256, dst=P256, n=3, stream=None)
    assert _call("wal_kv_pages_copy", args, cache=None) == ARG
    assert _call("wal_kv_pages_copy", args, src=None) == ARG and _call("wal_kv_pages_copy", args, dst=None) == ARG
    assert _call("wal_kv_pages_copy", args, n=0) == SHAPE
    assert _call("wal_kv_pages_copy", args, cache=_c(head_dim=32)) == UNSUPPORTED


VERIFY = dict(target=P256, tseq=3000, trow=1000, draft=P256, dseq=2000, drow=1000, drafts=P256, ldd=2, dlens=None, u=P256, ldu=3,
              B=2, T=2, V=1000, acc=P256, tok=P256, ldt=3, stream=None)


@pytest.mark.parametrize("change,want", [
    (dict(target=None), ARG), (dict(drafts=None), ARG), (dict(u=None), ARG), (dict(acc=None), ARG), (dict(tok=None), ARG),
    (dict(B=0), SHAPE), (dict(B=65536), SHAPE), (dict(T=-1), SHAPE), (dict(T=4097), SHAPE), (dict(V=0), SHAPE),
    (dict(V=(1 << 22) + 1), SHAPE), (dict(trow=999), SHAPE), (dict(drow=0), SHAPE), (dict(tseq=-1), SHAPE), (dict(ldd=1), SHAPE),
    (dict(ldu=2), SHAPE), (dict(ldt=2), SHAPE)])
def test_verify_refusals(change, want):
    assert _call("wal_verify_drafts", VERIFY, **change) == want


# ------------------------------------------------------------ Python checks

def _cache(**kw):
    return PagedKV8Cache.allocate(**(dict(layers=1, num_pages=4, kv_heads=2, head_dim=64, page_size=16, device="cpu") | kw))


def test_cache_checks():
    c = _cache()
    assert c.codes.shape == (1, 2, 4, 2, 16, 64) and c.bytes_per_token() == 2 * 2 * 64.25
    assert _cache(dtype=torch.float8_e4m3fn).codes.dtype == torch.float8_e4m3fn
    for kw in (dict(page_size=8), dict(head_dim=80), dict(num_pages=0), dict(dtype=torch.uint8)):
        with pytest.raises(ValueError):
            _cache(**kw)
    with pytest.raises(ValueError, match="contiguous"):
        PagedKV8Cache(c.codes.transpose(2, 3), torch.zeros(1, 2, 2, 4))
    with pytest.raises(ValueError, match="scales"):
        PagedKV8Cache(c.codes, c.scales.half())


def _z(*shape, dtype=torch.int32):
    return torch.zeros(shape, dtype=dtype)


def test_calls_refuse_cpu_tensors():
    c, bf = _cache(), torch.bfloat16
    tab, ln = _z(2, 3), _z(2)
    with pytest.raises(ValueError, match="CUDA"):
        kv8_append(c, 0, _z(2, 512, dtype=bf), 4, tab, ln, _z(2, 256, dtype=bf))
    with pytest.raises(ValueError, match="CUDA"):
        kv8_read(c, 0, tab, ln, ln, _z(2, 2, 5, 64, dtype=bf), _z(2, 2, 5, 64, dtype=bf))
    with pytest.raises(ValueError, match="CUDA"):
        kv8_attention(c, 0, _z(2, 256, dtype=bf), tab, ln, _z(2, 256, dtype=bf), _z(256, dtype=torch.uint8))
    with pytest.raises(ValueError, match="CUDA"):
        kv_pages_assign(tab, ln, ln, ln, 16, _z(2, 3), _z(4), ln, ln, ln)
    with pytest.raises(ValueError, match="CUDA"):
        kv_pages_compact(tab, ln, 16, _z(2, 3), _z(4), _z(4), _z(4), _z(2))
    with pytest.raises(ValueError, match="CUDA"):
        kv_pages_copy(c, ln, ln)
    with pytest.raises(ValueError, match="CUDA"):
        verify_drafts(_z(2, 2, 9, dtype=torch.float32), None, _z(2, 1), _z(2, 2, dtype=torch.float32), ln, _z(2, 2))
    with pytest.raises(ValueError, match="invalid attention shape"):
        kv8_attention_workspace(c, 2, 3)


def test_shapes_and_types_are_checked_before_the_device():
    tab, ln = _z(2, 3), _z(2)
    with pytest.raises(ValueError, match="pages per row"):
        kv_pages_assign(tab, ln, ln, ln, 16, _z(2, 4), _z(4), ln, ln, ln)
    with pytest.raises(ValueError, match="keep"):
        kv_pages_assign(tab, ln, ln.long(), ln, 16, _z(2, 3), _z(4), ln, ln, ln)
    with pytest.raises(ValueError, match="shape of table"):
        kv_pages_compact(tab, ln, 16, _z(3, 3), _z(4), _z(4), _z(4), _z(2))
    f = torch.float32
    with pytest.raises(ValueError, match="target"):
        verify_drafts(_z(2, 2, 9, dtype=torch.float64), None, _z(2, 1), _z(2, 2, dtype=f), ln, _z(2, 2))
    with pytest.raises(ValueError, match="draft must"):
        verify_drafts(_z(2, 2, 9, dtype=f), _z(2, 2, 9, dtype=f), _z(2, 1), _z(2, 2, dtype=f), ln, _z(2, 2))
    with pytest.raises(ValueError, match="tokens"):
        verify_drafts(_z(2, 2, 9, dtype=f), None, _z(2, 1), _z(2, 2, dtype=f), ln, _z(2, 1))


def test_nothing_is_launched_where_the_arguments_do_not_fit(monkeypatch):
    # arguments that the fast checks refuse are refused, whether or not the search for the reason finds one
    import wal2026_b200.kv8 as kv8
    import wal2026_b200.speculative as speculative

    launched = []
    for module in (kv8, speculative):
        monkeypatch.setattr(module, "_cuda", lambda device: None)  # CPU tensors: the fast checks fail, no reason is found
        monkeypatch.setattr(module, "_call", lambda *a: launched.append(a))
    c, bf, f = _cache(), torch.bfloat16, torch.float32
    tab, ln, out = _z(2, 3), _z(2), _z(2, 3)
    calls = [lambda: kv8_append(c, 0, _z(2, 512, dtype=bf), 4, tab, ln, _z(2, 256, dtype=bf)),
             lambda: kv8_read(c, 0, tab, ln, ln, _z(2, 2, 5, 64, dtype=bf), _z(2, 2, 5, 64, dtype=bf)),
             lambda: kv8_attention(c, 0, _z(2, 256, dtype=bf), tab, ln, _z(2, 256, dtype=bf), _z(256, dtype=torch.uint8)),
             lambda: kv_pages_assign(tab, ln, ln, ln, 16, out, _z(4), ln, ln, ln),
             lambda: kv_pages_compact(tab, ln, 16, out, _z(4), _z(4), _z(4), _z(2)),
             lambda: kv_pages_copy(c, ln, ln),
             lambda: verify_drafts(_z(2, 2, 9, dtype=f), None, _z(2, 1), _z(2, 2, dtype=f), ln, _z(2, 2))]
    for call in calls:
        with pytest.raises(ValueError, match="do not fit together"):
            call()
    assert not launched


def test_sizes_whose_indexes_would_pass_32_bits_are_refused():
    big = 1 << 30
    for name, args in (("wal_kv_pages_assign", ASSIGN), ("wal_kv_pages_compact", COMPACT)):
        wide = dict(ld_table=1 << 31, ld_out=1 << 31)
        assert _call(name, args, num_pages=big + 1) == SHAPE            # strided loops over the pages
        assert _call(name, args, width=big + 1, page_size=1, **wide) == SHAPE  # chunks of 512 entries
        assert _call(name, args, width=715827882, page_size=3, **wide) == SHAPE  # tokens rounded up to pages
        assert _call(name, args, width=1, page_size=big + 2) == SHAPE
    # wanted pages of all rows together
    assert _call("wal_kv_pages_assign", ASSIGN, rows=16, width=1 << 27, page_size=8, ld_table=1 << 27, ld_out=1 << 27) == SHAPE
    # the end of an attention tile
    for pages in ((1 << 27) - 1, (1 << 27) - 2):
        assert _call("wal_kv8_attention", ATTN, cache=_c(), max_pages=pages, ld_table=1 << 27) == SHAPE
