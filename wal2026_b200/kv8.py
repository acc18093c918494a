"""Paged KV cache held in 8 bits, the attention that reads it, and its pages (C ABI wrappers).

``PagedKV8Cache`` wraps two tensors: codes ``[layers, 2, pages, kv_heads,
page_size, head_dim]`` (int8, or float8_e4m3fn) and fp32 scales ``[layers, 2,
pages, kv_heads]``; a value is code * scale.  Index 0 of the second axis is K,
1 is V.  Sequences own rows of an int32 page table; tables, lengths and counts
stay on the device, so a decoding loop never waits for the host.

A step of T new tokens per sequence (T = 1: plain decoding; more: a prompt, or
drafts to verify):

    kv_pages_assign / kv_pages_copy   room for the tokens, in pages of their own
    kv8_append                        rotary positions, q out, k and v stored   (per layer)
    kv8_attention                     causal attention of the T tokens          (per layer)

``lens`` always counts the positions a sequence held before the step's tokens.
Each call launches on the current stream of its tensors' device; none has a CPU
path, allocates or synchronises.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch import Tensor

from . import _abi

PAGE_SIZES = (16, 32, 64)
HEAD_DIMS = (64, 128)
_KIND = {torch.int8: _abi.WAL_KV_INT8, torch.float8_e4m3fn: _abi.WAL_KV_E4M3}
CODE_MAX = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


class PagedKV8Cache:
    """Codes and scales of a paged 8-bit KV cache; ``allocate`` makes a zero-filled one."""

    def __init__(self, codes: Tensor, scales: Tensor):
        if codes.dtype not in _KIND:
            raise ValueError(f"cache codes must be int8 or float8_e4m3fn, got {codes.dtype}")
        if codes.dim() != 6 or codes.shape[1] != 2:
            raise ValueError("cache codes must be [layers, 2, pages, kv_heads, page_size, head_dim]")
        if scales.dtype != torch.float32 or tuple(scales.shape) != tuple(codes.shape[:4]):
            raise ValueError("cache scales must be fp32 [layers, 2, pages, kv_heads]")
        if not (codes.is_contiguous() and scales.is_contiguous()):
            raise ValueError("cache codes and scales must be contiguous")
        if codes.device != scales.device:
            raise ValueError("cache codes and scales must be on one device")
        self.layers, _, self.num_pages, self.kv_heads, self.page_size, self.head_dim = (int(v) for v in codes.shape)
        if self.page_size not in PAGE_SIZES or self.head_dim not in HEAD_DIMS:
            raise ValueError(f"page_size must be one of {PAGE_SIZES} and head_dim one of {HEAD_DIMS}")
        if codes.numel() == 0:
            raise ValueError("cache has no pages")
        self.codes, self.scales = codes, scales
        self.device, self.index = codes.device, codes.get_device()
        self._c = _abi.KV8Cache(codes.data_ptr(), scales.data_ptr(), self.num_pages, self.layers, self.kv_heads,
                                self.page_size, self.head_dim, _KIND[codes.dtype])
        self._ref = ctypes.byref(self._c)

    @classmethod
    def allocate(cls, layers: int, num_pages: int, kv_heads: int, head_dim: int, *, page_size: int = 64,
                 dtype: torch.dtype = torch.int8, device="cuda") -> "PagedKV8Cache":
        if dtype not in _KIND:
            raise ValueError(f"cache codes must be int8 or float8_e4m3fn, got {dtype}")
        shape = (layers, 2, num_pages, kv_heads, page_size, head_dim)
        codes = torch.zeros(shape, dtype=torch.int8, device=device).view(dtype)
        return cls(codes, torch.zeros(shape[:4], dtype=torch.float32, device=device))

    def bytes_per_token(self) -> float:
        """Device bytes one position takes over all layers."""
        return 2 * self.layers * self.kv_heads * (self.head_dim + 4 / self.page_size)


# Argument checks.  A call first asks whether everything is as it should be, in
# as few attribute reads as that takes (a step makes two such calls per layer,
# and a read costs about 0.1 us); only where it is not do the functions of the
# names below look for the reason and raise it.

_I32, _BF16, _F32 = torch.int32, torch.bfloat16, torch.float32
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _on(device: torch.device, **tensors: Optional[Tensor]) -> None:
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} is on {t.device}, expected {device}")


def _i32(name: str, t: Tensor, *shape: int) -> None:
    if t.dtype != torch.int32 or tuple(t.shape) != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of shape {list(shape)}")


def _is_i32(t: Tensor, shape: tuple, index: int) -> bool:
    return t.dtype is _I32 and t.shape == shape and t.is_contiguous() and t.get_device() == index


def _table(name: str, t: Tensor) -> tuple[int, int]:
    if t.dtype != torch.int32 or t.dim() != 2 or t.stride(1) != 1 or t.stride(0) < t.shape[1]:
        raise ValueError(f"{name} must be int32 [rows, pages] with contiguous rows")
    return t.shape


def _rows(name: str, t: Tensor, width: int) -> int:
    if t.dtype != torch.bfloat16 or t.dim() != 2 or t.shape[1] != width or t.stride(1) != 1:
        raise ValueError(f"{name} must be bf16 [tokens, {width}] with contiguous rows")
    return t.shape[0]


def _cuda(device: torch.device) -> None:
    if device.type != "cuda":
        raise ValueError("the paged cache runs on CUDA tensors only")


def _batch(rows: int, table: Tensor, lens: Tensor, new_lens: Optional[Tensor]) -> None:
    B, _ = _table("table", table)
    if B == 0 or rows == 0 or rows % B:
        raise ValueError(f"{rows} token rows do not split over {B} sequences")
    _i32("lens", lens, B)
    if new_lens is not None:
        _i32("new_lens", new_lens, B)


_entry: dict = {}


def _call(index: int, name: str, *args) -> None:
    """One entry point on the current stream of device ``index``."""
    fn = _entry.get(name)
    if fn is None:
        fn = _entry[name] = getattr(_abi.load(), name)
    if _abi._raw_stream is not None and index == _current_device():
        st = fn(*args, _abi._raw_stream(index))
    else:
        with torch.cuda.device(index):
            st = fn(*args, _abi.stream_handle(torch.device("cuda", index)))
    if st:
        _abi.check(st, name)


def _step(cache: PagedKV8Cache, x: Tensor, width: int, y: Tensor, hq: int, table: Tensor, lens: Tensor,
          new_lens: Optional[Tensor]) -> Optional[tuple]:
    """(sequences, tokens each, pages, strides of x, y, table) where token rows x [B * T, width] and y [B * T, hq *
    head_dim], a table and lengths all fit to launch."""
    i, ts, xs, x1, y1, t1 = cache.index, table.shape, x.shape, x.stride(), y.stride(), table.stride()
    if (i >= 0 and len(ts) == 2 and len(xs) == 2 and ts[0] > 0 and xs[0] > 0 and xs[0] % ts[0] == 0 and xs[1] == width
            and y.shape == (xs[0], hq * cache.head_dim) and x1[1] == 1 and y1[1] == 1 and t1[1] == 1 and t1[0] >= ts[1]
            and x.dtype is _BF16 and y.dtype is _BF16 and table.dtype is _I32 and x.get_device() == i
            and y.get_device() == i and table.get_device() == i and _is_i32(lens, ts[:1], i)
            and (new_lens is None or _is_i32(new_lens, ts[:1], i))):
        return ts[0], xs[0] // ts[0], ts[1], x1[0], y1[0], t1[0]
    return None


def _why_not_append(cache, qkv, hq, table, lens, q_out, cos, sin, new_lens) -> None:
    _cuda(cache.device)
    hd = cache.head_dim
    M = _rows("qkv", qkv, (hq + 2 * cache.kv_heads) * hd)
    if _rows("q_out", q_out, hq * hd) != M:
        raise ValueError("q_out must have a row for each row of qkv")
    _batch(M, table, lens, new_lens)
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together")
    if cos is not None:
        for name, t in (("cos", cos), ("sin", sin)):
            if t.dtype != torch.float32 or t.dim() != 2 or t.shape[1] != hd // 2 or not t.is_contiguous() or t.shape != cos.shape:
                raise ValueError(f"{name} must be fp32 [max_pos, head_dim / 2] contiguous")
    _on(cache.device, qkv=qkv, q_out=q_out, table=table, lens=lens, new_lens=new_lens, cos=cos, sin=sin)
    raise ValueError("kv8_append: arguments do not fit together")


def kv8_append(cache: PagedKV8Cache, layer: int, qkv: Tensor, hq: int, table: Tensor, lens: Tensor, q_out: Tensor, *,
               cos: Optional[Tensor] = None, sin: Optional[Tensor] = None, new_lens: Optional[Tensor] = None) -> None:
    """Rotate q and k of T new tokens per sequence and store k, v in their pages.

    qkv: bf16 [B * T, (hq + 2 * kv_heads) * head_dim], row b * T + t at position
    lens[b] + t; q_out: bf16 [B * T, hq * head_dim]; cos / sin: fp32 [max_pos,
    head_dim / 2] (rotate-half pairs), or neither.  Rows t >= new_lens[b] are
    padding.  A block's scale grows with its largest value, and its earlier
    codes are re-rounded when it does.  A token that a later call overwrites (a
    draft that was not kept) leaves the scale where it raised it: earlier values
    then carry the coarser rounding.
    """
    hd, max_pos = cache.head_dim, 0
    step = _step(cache, qkv, (hq + 2 * cache.kv_heads) * hd, q_out, hq, table, lens, new_lens)
    fit = step is not None and (cos is None) == (sin is None)
    if fit and cos is not None:
        cs = cos.shape
        max_pos = cs[0] if len(cs) == 2 else 0
        fit = (cs == (max_pos, hd // 2) and sin.shape == cs and cos.dtype is _F32 and sin.dtype is _F32
               and cos.is_contiguous() and sin.is_contiguous() and cos.get_device() == sin.get_device() == cache.index)
    if not fit:
        _why_not_append(cache, qkv, hq, table, lens, q_out, cos, sin, new_lens)
    B, T, pages, ld_x, ld_q, ld_t = step
    _call(cache.index, "wal_kv8_append", cache._ref, layer, qkv.data_ptr(), ld_x, B, T, hq, table.data_ptr(), ld_t, pages,
          lens.data_ptr(), None if new_lens is None else new_lens.data_ptr(), None if cos is None else cos.data_ptr(),
          None if sin is None else sin.data_ptr(), max_pos, q_out.data_ptr(), ld_q)


def _why_not_read(cache, table, first, count, k_out, v_out) -> None:
    _cuda(cache.device)
    B, _ = _table("table", table)
    _i32("first", first, B)
    _i32("count", count, B)
    if k_out.dtype not in (torch.bfloat16, torch.float32) or v_out.dtype != k_out.dtype:
        raise ValueError("k_out and v_out must both be bf16 or fp32")
    L = k_out.shape[2] if k_out.dim() == 4 else 0
    for name, t in (("k_out", k_out), ("v_out", v_out)):
        if tuple(t.shape) != (B, cache.kv_heads, L, cache.head_dim) or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous [{B}, {cache.kv_heads}, L, {cache.head_dim}]")
    _on(cache.device, table=table, first=first, count=count, k_out=k_out, v_out=v_out)
    raise ValueError("kv8_read: arguments do not fit together")


def kv8_read(cache: PagedKV8Cache, layer: int, table: Tensor, first: Tensor, count: Tensor, k_out: Tensor,
             v_out: Tensor) -> None:
    """Values of positions first[b] .. first[b] + count[b] - 1 into k_out, v_out [B, kv_heads, L, head_dim] (bf16 or
    fp32, contiguous); zeros past count[b] and where a position has no page."""
    i, ts, ks, t1 = cache.index, table.shape, k_out.shape, table.stride()
    if not (i >= 0 and len(ts) == 2 and len(ks) == 4 and ks == (ts[0], cache.kv_heads, ks[2], cache.head_dim) and v_out.shape == ks
            and t1[1] == 1 and t1[0] >= ts[1] and table.dtype is _I32 and (k_out.dtype is _F32 or k_out.dtype is _BF16)
            and v_out.dtype is k_out.dtype and k_out.is_contiguous() and v_out.is_contiguous() and table.get_device() == i
            and k_out.get_device() == i and v_out.get_device() == i and _is_i32(first, ts[:1], i) and _is_i32(count, ts[:1], i)):
        _why_not_read(cache, table, first, count, k_out, v_out)
    if ks[2] == 0:
        return
    _call(i, "wal_kv8_read", cache._ref, layer, ts[0], table.data_ptr(), t1[0], ts[1], first.data_ptr(), count.data_ptr(),
          ks[2], k_out.data_ptr(), v_out.data_ptr(), _abi.DTYPE_CODE[k_out.dtype])


def kv8_attention_workspace(cache: PagedKV8Cache, batch: int, hq: int, tokens: int = 1) -> Tensor:
    """Zero-filled scratch for ``kv8_attention`` calls of up to ``batch`` sequences with up to ``tokens`` new tokens each."""
    nbytes = int(_abi.load().wal_kv8_attention_workspace(cache._ref, batch, tokens, hq))
    if nbytes == 0:
        raise ValueError("invalid attention shape")
    return torch.zeros(nbytes, dtype=torch.uint8, device=cache.device)


def _why_not_attention(cache, q, table, lens, out, workspace, new_lens) -> None:
    _cuda(cache.device)
    hd = cache.head_dim
    if q.dim() != 2 or q.shape[1] == 0 or q.shape[1] % (hd * cache.kv_heads):
        raise ValueError("q must be bf16 [tokens, hq * head_dim], hq a multiple of the cache's kv heads")
    M = _rows("q", q, q.shape[1])
    if _rows("out", out, q.shape[1]) != M:
        raise ValueError("out must have a row for each row of q")
    _batch(M, table, lens, new_lens)
    _on(cache.device, q=q, out=out, table=table, lens=lens, new_lens=new_lens, workspace=workspace)
    if not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous")
    raise ValueError("kv8_attention: arguments do not fit together")


def kv8_attention(cache: PagedKV8Cache, layer: int, q: Tensor, table: Tensor, lens: Tensor, out: Tensor,
                  workspace: Tensor, *, new_lens: Optional[Tensor] = None, scale: Optional[float] = None) -> None:
    """out[b * T + t, h] = softmax(scale * q[b * T + t, h] . k_j) v over the positions j <= lens[b] + t of sequence b.

    q, out: bf16 [B * T, hq * head_dim], hq a multiple of the cache's kv heads;
    the T tokens are already stored.  Rows t >= new_lens[b], and rows that have
    no position with a page, are zeros.  ``workspace`` comes from
    ``kv8_attention_workspace`` and is not shared by overlapping calls.
    """
    hd = cache.head_dim
    width = q.shape[-1] if q.dim() else 0
    hq = width // hd
    step = _step(cache, q, width, out, hq, table, lens, new_lens)
    if not (step is not None and width > 0 and width % (hd * cache.kv_heads) == 0
            and workspace.get_device() == cache.index and workspace.is_contiguous()):
        _why_not_attention(cache, q, table, lens, out, workspace, new_lens)
    B, T, pages, ld_q, ld_o, ld_t = step
    _call(cache.index, "wal_kv8_attention", cache._ref, layer, q.data_ptr(), ld_q, B, T, hq, table.data_ptr(), ld_t, pages,
          lens.data_ptr(), None if new_lens is None else new_lens.data_ptr(), hd ** -0.5 if scale is None else scale,
          out.data_ptr(), ld_o, workspace.data_ptr(), workspace.nbytes)


def _why_not_assign(table, parent, keep, add, table_out, ref_out, copy_src, copy_dst, info) -> None:
    _, width = _table("table", table)
    rows, w2 = _table("table_out", table_out)
    if w2 != width:
        raise ValueError("table and table_out must have the same number of pages per row")
    for name, t in (("parent", parent), ("keep", keep), ("add", add), ("copy_src", copy_src), ("copy_dst", copy_dst)):
        _i32(name, t, rows)
    _i32("ref_out", ref_out, ref_out.numel())
    _i32("info", info, 2)
    _cuda(table.device)
    _on(table.device, parent=parent, keep=keep, add=add, table_out=table_out, ref_out=ref_out, copy_src=copy_src,
        copy_dst=copy_dst, info=info)
    raise ValueError("kv_pages_assign: arguments do not fit together")


def kv_pages_assign(table: Tensor, parent: Tensor, keep: Tensor, add: Tensor, page_size: int, table_out: Tensor,
                    ref_out: Tensor, copy_src: Tensor, copy_dst: Tensor, info: Tensor) -> None:
    """Tables of the next step: row b keeps the first keep[b] tokens of row parent[b] and gets room for add[b] more.

    table int32 [rows_in, width]; table_out [rows, width]; ref_out [num_pages];
    the others [rows], info [2].  Forking, truncating, freeing and reserving
    are one call; pass copy_src, copy_dst on to ``kv_pages_copy`` before the
    step's first append.  info = (pages left free, pages wanted but not given);
    ``table`` is left as it was, so a call that could not give every page can be
    repeated after making room.
    """
    index, ts, os, t1, o1 = table.get_device(), table.shape, table_out.shape, table.stride(), table_out.stride()
    rows = os[:1]
    if not (index >= 0 and len(ts) == 2 and len(os) == 2 and ts[1] == os[1] and t1[1] == 1 and o1[1] == 1 and t1[0] >= ts[1]
            and o1[0] >= ts[1] and table.dtype is _I32 and table_out.dtype is _I32 and table_out.get_device() == index
            and _is_i32(parent, rows, index) and _is_i32(keep, rows, index) and _is_i32(add, rows, index)
            and _is_i32(copy_src, rows, index) and _is_i32(copy_dst, rows, index) and _is_i32(info, (2,), index)
            and _is_i32(ref_out, (ref_out.numel(),), index)):
        _why_not_assign(table, parent, keep, add, table_out, ref_out, copy_src, copy_dst, info)
    a, b = table.data_ptr(), table_out.data_ptr()
    if ts[0] and os[0] and a < b + 4 * ((os[0] - 1) * o1[0] + ts[1]) and b < a + 4 * ((ts[0] - 1) * t1[0] + ts[1]):
        raise ValueError("table_out must not overlap table")
    _call(index, "wal_kv_pages_assign", a, t1[0], ts[0], parent.data_ptr(), keep.data_ptr(), add.data_ptr(), os[0], ts[1],
          ref_out.numel(), page_size, b, o1[0], ref_out.data_ptr(), copy_src.data_ptr(), copy_dst.data_ptr(),
          info.data_ptr())


def _why_not_compact(table, lens, table_out, remap, move_src, move_dst, info) -> None:
    rows, _ = _table("table", table)
    if _table("table_out", table_out) != table.shape:
        raise ValueError("table_out must have the shape of table")
    _i32("lens", lens, rows)
    for name, t in (("remap", remap), ("move_src", move_src), ("move_dst", move_dst)):
        _i32(name, t, remap.numel())
    _i32("info", info, 2)
    _cuda(table.device)
    _on(table.device, lens=lens, table_out=table_out, remap=remap, move_src=move_src, move_dst=move_dst, info=info)
    raise ValueError("kv_pages_compact: arguments do not fit together")


def kv_pages_compact(table: Tensor, lens: Tensor, page_size: int, table_out: Tensor, remap: Tensor, move_src: Tensor,
                     move_dst: Tensor, info: Tensor) -> None:
    """Move the used pages to the front of the pool: new table (may be ``table``), remap and moves [num_pages].

    Pass move_src, move_dst on to ``kv_pages_copy``.  info = (used pages, moves).
    """
    index, ts, t1, o1, n = table.get_device(), table.shape, table.stride(), table_out.stride(), remap.numel()
    if not (index >= 0 and len(ts) == 2 and table_out.shape == ts and t1[1] == 1 and o1[1] == 1 and t1[0] >= ts[1]
            and o1[0] >= ts[1] and table.dtype is _I32 and table_out.dtype is _I32 and table_out.get_device() == index
            and _is_i32(lens, ts[:1], index) and _is_i32(remap, (n,), index) and _is_i32(move_src, (n,), index)
            and _is_i32(move_dst, (n,), index) and _is_i32(info, (2,), index)):
        _why_not_compact(table, lens, table_out, remap, move_src, move_dst, info)
    a, b = table.data_ptr(), table_out.data_ptr()
    if (a != b or t1 != o1) and a < b + 4 * ((ts[0] - 1) * o1[0] + ts[1]) and b < a + 4 * ((ts[0] - 1) * t1[0] + ts[1]):
        raise ValueError("table_out must be the table itself or must not overlap it")
    _call(index, "wal_kv_pages_compact", a, t1[0], lens.data_ptr(), ts[0], ts[1], n, page_size, b, o1[0], remap.data_ptr(),
          move_src.data_ptr(), move_dst.data_ptr(), info.data_ptr())


def _why_not_copy(cache, src, dst) -> None:
    _cuda(cache.device)
    _i32("src", src, src.numel())
    _i32("dst", dst, src.numel())
    _on(cache.device, src=src, dst=dst)
    raise ValueError("kv_pages_copy: arguments do not fit together")


def kv_pages_copy(cache: PagedKV8Cache, src: Tensor, dst: Tensor) -> None:
    """Copy page src[i] to dst[i] in every layer (K, V, scales); pairs with an entry that names no page are skipped.

    No dst may be another pair's src or dst.
    """
    n = src.numel()
    if not (cache.index >= 0 and _is_i32(src, (n,), cache.index) and _is_i32(dst, (n,), cache.index)):
        _why_not_copy(cache, src, dst)
    if n:
        _call(cache.index, "wal_kv_pages_copy", cache._ref, src.data_ptr(), dst.data_ptr(), n)
