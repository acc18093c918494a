"""Groups of rows that share their first pages, and their attention, on the GPU.

Groups are compared for equality with a row-by-row restatement; the attention with
the softmax in 64 bits over every row's own positions, as if nothing were shared.
Tolerance: the output is rounded once to bf16 (2^-8 of a value); weights of shared
positions enter the product as f16 (2^-11 each, 2^-32 of the largest where they
are subnormal: n of them at most n 2^-32 of the largest |v|), the others as two
bf16 numbers; the exponents and the sums in 32 bits add less than 2^-13 of the
weighted mean of |v|.
"""
from __future__ import annotations

import pytest
import torch

from wal2026_b200.kv8 import (CODE_MAX, PagedKV8Cache, kv8_attention, kv8_attention_shared, kv8_attention_shared_workspace,
                              kv8_attention_workspace, kv_pages_groups)

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
INT8, E4M3 = torch.int8, torch.float8_e4m3fn


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _filled(pages, hkv, P, hd, dtype, seed, layers=1):
    g = _gen(seed)
    shape = (layers, 2, pages, hkv, P, hd)
    x = (torch.randn(shape, device=DEV, generator=g) * CODE_MAX[dtype] / 4).clamp(-CODE_MAX[dtype], CODE_MAX[dtype])
    codes = x.round().to(INT8) if dtype == INT8 else x.to(E4M3)
    return PagedKV8Cache(codes, torch.rand(shape[:4], device=DEV, generator=g) * (4 / CODE_MAX[dtype]) + 1e-3)


def _forks(prompts, P, T, seed, width=None, stride=None):
    """(table, lens, pages) of rows [(prompt id or None, prompt length, own tokens)]: a prompt's whole pages are common."""
    n, first, rows = 0, {}, []
    for key, length, extra in prompts:
        common = length // P if key is not None else 0
        if key is not None and key not in first:
            first[key] = list(range(n, n + common))
            n += common
        need = -(-(length + extra + T) // P)
        mine = max(0, need - common)
        rows.append((first[key][:common] if key is not None else []) + list(range(n, n + mine)))
        n += mine
    order = torch.randperm(n, generator=torch.Generator().manual_seed(seed)).tolist()
    width = width or max(len(r) for r in rows)
    buf = torch.full((len(rows), stride or width), -7, dtype=torch.int32)
    for b, r in enumerate(rows):
        for j, p in enumerate(r[:width]):
            buf[b, j] = order[p]
    return buf.to(DEV)[:, :width], [a + e for _, a, e in prompts], n


def _groups_reference(table, lens, P, least):
    tab, B, width = table.tolist(), table.shape[0], table.shape[1]
    at, by = (least - 1) // P, {}
    for b in range(B):
        full = min(max(lens[b], 0), width * P - 1) // P
        if full * P // 32 * 32 >= least and at < width and tab[b][at] >= 0:
            by.setdefault(tab[b][at], []).append((b, full))
    order, begin, size, shared = [], [], [], [0] * B
    for members in sorted(by.values()):
        lead, n = members[0]
        for b, full in members:
            k = 0
            while k < min(full, n) and tab[b][k] == tab[lead][k]:
                k += 1
            n = k
        if len(members) > 1 and n * P // 32 * 32 >= least:
            begin.append(len(order))
            size.append(len(members))
            for b, _ in members:
                order.append(b)
                shared[b] = n * P // 32 * 32
    pad = [0] * (B - len(begin))
    return [order + [-1] * (B - len(order)), begin + pad, size + pad, shared]


def _groups(table, lens, P, least):
    out = torch.full((4, table.shape[0]), 99, dtype=torch.int32, device=DEV)
    kv_pages_groups(table, _i32(lens), P, out, least=least)
    return out


@pytest.mark.parametrize("P", [16, 32, 64])
@pytest.mark.parametrize("least", [1, 32, 33, 100, 256])
@pytest.mark.parametrize("rows", [[("a", 300, 5)], [("a", 300, 5), ("a", 300, 0)], [(None, 40, 3)] * 5,
                                  [("a", 300, 5), ("b", 700, 1), ("a", 300, 400), (None, 900, 0), ("b", 700, 0), ("a", 300, 31)],
                                  [("a", 31, 500), ("a", 31, 400), ("b", 64, 0), ("b", 64, 0), ("c", 0, 0), ("c", 0, 0)],
                                  [(i % 37, 200 + 13 * (i % 37), i % 90) for i in range(300)],
                                  [(0, 2000, i) for i in range(70)]])
def test_groups_equal_their_definition(P, least, rows):
    table, lens, _ = _forks(rows, P, 1, 3, stride=200 if len(rows) == 5 else None)
    assert _groups(table, lens, P, least).tolist() == _groups_reference(table, lens, P, least)


def test_groups_of_tables_that_no_fork_makes():
    P = 16
    table = _i32([[1, 2, 3, 4], [1, 2, 9, 4], [1, 2, 3, 4], [9, 2, 3, 4], [-1, 2, 3, 4], [-1, 2, 3, 4], [5, -1, 7, 8], [5, -1, 7, 8],
                  [5, -5, 7, 8]])
    for lens in ([64] * 9, [63] * 9, [0, 64, 64, 64, 64, 64, 64, 64, 64], [33, 1 << 30, -4, 64, 64, 2 ** 31 - 1, 48, 47, 64]):
        for least in (1, 16, 17, 32, 48, 64, 1000, 1 << 40):
            assert _groups(table, lens, P, least).tolist() == _groups_reference(table, lens, P, least), (lens, least)


def test_groups_of_as_many_rows_as_are_allowed():
    rows = [((7919 * i) % 1500, 64 + (i % 2), i % 3) for i in range(4096)]
    table, lens, _ = _forks(rows, 16, 1, 4)
    assert _groups(table, lens, 16, 64).tolist() == _groups_reference(table, lens, 16, 64)
    with pytest.raises(ValueError):
        _groups(torch.zeros(4097, 3, dtype=torch.int32, device=DEV), [1] * 4097, 16, 16)


# ----------------------------------------------------------------- attention

def _attention64(cache, q, table, lens, news, scale, layer):
    B, hkv, P, hd = table.shape[0], cache.kv_heads, cache.page_size, cache.head_dim
    T, hq = q.shape[0] // B, q.shape[1] // hd
    G = hq // hkv
    val = cache.codes[layer].float().double() * cache.scales[layer].double()[..., None, None]
    out, mag = (torch.zeros(B, T, hq, hd, dtype=torch.float64, device=DEV) for _ in range(2))
    most = torch.zeros(B, 1, 1, 1, dtype=torch.float64, device=DEV)
    tab = table.long()
    for b in range(B):
        n_all = min(lens[b] + min(T, news[b]), table.shape[1] * P)
        if news[b] <= 0 or n_all <= 0:
            continue
        pos = torch.arange(n_all, device=DEV)
        page = tab[b, pos // P]
        ok = (page >= 0) & (page < cache.num_pages)
        k, v = (val[i, page.clamp(0, cache.num_pages - 1), :, pos % P].transpose(0, 1) for i in range(2))  # [hkv, n, hd]
        v = torch.where(ok[None, :, None], v, 0.0)
        most[b] = v.abs().max() * n_all
        qb = q.double().view(B, T, hkv, G, hd)[b, :news[b]].permute(1, 0, 2, 3)  # [hkv, t, G, hd]
        x = torch.einsum("htgd,hnd->htgn", qb, k) * scale
        t = torch.arange(min(T, news[b]), device=DEV)
        seen = ok[None, :] & (pos[None, :] <= lens[b] + t[:, None])
        x = x.masked_fill(~seen[None, :, None], float("-inf"))
        w = torch.nan_to_num(torch.softmax(x, -1), nan=0.0)
        out[b, :news[b]] = torch.einsum("htgn,hnd->thgd", w, v).reshape(-1, hq, hd)
        mag[b, :news[b]] = torch.einsum("htgn,hnd->thgd", w, v.abs()).reshape(-1, hq, hd)
    return out.view(B * T, -1), mag.view(B * T, -1), (torch.ones_like(out) * most).view(B * T, -1)


def _check(cache, q, table, lens, groups, news=None, scale=None, layer=0, ws=None):
    B = table.shape[0]
    T, hd = q.shape[0] // B, cache.head_dim
    hq = q.shape[1] // hd
    ws = kv8_attention_shared_workspace(cache, B, hq, T) if ws is None else ws
    out = torch.full(q.shape, float("nan"), dtype=torch.bfloat16, device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    nl = None if news is None else _i32(news)
    kv8_attention_shared(cache, layer, q, table, _i32(lens), groups, out, ws, new_lens=nl, scale=scale, status=status)
    assert status.item() == 0
    want, mag, most = _attention64(cache, q, table, lens, [T] * B if news is None else news, hd ** -0.5 if scale is None else scale, layer)
    bad = ~((out.double() - want).abs() <= 1.01 * 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2.0 ** -13) * mag + 2.0 ** -32 * most + 1e-30)
    assert not bool(bad.any()), (int(bad.sum()), float((out.double() - want).abs().max()))
    again = torch.empty_like(out)
    kv8_attention_shared(cache, layer, q, table, _i32(lens), groups, again, ws, new_lens=nl, scale=scale)
    assert torch.equal(out, again)  # the same bits every time, and the workspace was left ready
    return out


@pytest.mark.parametrize("dtype", [INT8, E4M3])
@pytest.mark.parametrize("P,hd", [(16, 64), (32, 128), (64, 64), (64, 128), (16, 128)])
@pytest.mark.parametrize("hq,hkv,T", [(8, 2, 1), (4, 4, 3), (14, 2, 2), (5, 1, 7)])
def test_shared_attention_matches_softmax_in_64_bits(dtype, P, hd, hq, hkv, T):
    rows = [("a", 300, 5), ("b", 700, 1), ("a", 300, 400), (None, 150, 0), ("b", 700, 0), ("a", 300, 31), (None, 0, 0)]
    table, lens, pages = _forks(rows, P, T, 5)
    cache = _filled(pages, hkv, P, hd, dtype, P + hd + T, layers=2)
    q = (torch.randn(len(lens) * T, hq * hd, device=DEV, generator=_gen(3)) * 2).to(torch.bfloat16)
    groups = _groups(table, lens, P, 64)
    assert int((groups[3] > 0).sum()) == 5
    _check(cache, q, table, lens, groups, layer=1)


@pytest.mark.parametrize("rows,hq,hkv,T,P", [
    ([("a", 4100, i) for i in range(2)], 32, 8, 1, 64),             # two samples
    ([("a", 1000, 7 * i) for i in range(64)], 8, 1, 1, 16),         # four tiles of query rows
    ([("a", 2050, 40 + i) for i in range(9)], 16, 2, 5, 32),        # drafts: three tiles, the last one partly filled
    ([(i % 20, 128 + 32 * (i % 20), i) for i in range(60)], 4, 4, 1, 32),   # many short groups
    ([(i // 3, 500, 3) for i in range(150)], 16, 8, 1, 16),         # more units than SMs
    ([("a", 9000, i) for i in range(3)] + [(None, 5000, 0)], 6, 1, 1, 64),
    ([("a", 257, 0)] * 130, 2, 2, 1, 64)])
def test_shared_attention_over_many_units_and_long_prefixes(rows, hq, hkv, T, P):
    table, lens, pages = _forks(rows, P, T, 1)
    cache = _filled(pages, hkv, P, 128, INT8, len(rows))
    q = torch.randn(len(lens) * T, hq * 128, device=DEV, generator=_gen(len(rows))).to(torch.bfloat16)
    _check(cache, q, table, lens, _groups(table, lens, P, 96))


@pytest.mark.parametrize("dtype", [INT8, E4M3])
def test_shared_attention_with_padding_missing_pages_and_idle_rows(dtype):
    P, hq, hkv, hd, T = 32, 8, 2, 64, 4
    rows = [("a", 500, i) for i in range(5)] + [("b", 260, 3 * i) for i in range(4)]
    table, lens, pages = _forks(rows, P, T, 2, stride=40)
    cache = _filled(pages, hkv, P, hd, dtype, 8)
    groups = _groups(table, lens, P, 64)
    news = [4, 0, 2, 1, 4, 0, 0, 3, 1]
    q = torch.randn(len(rows) * T, hq * hd, device=DEV, generator=_gen(1)).to(torch.bfloat16)
    _check(cache, q, table, lens, groups, news)
    table[:5, 3] = -1                        # a hole in the prefix
    table[2, -2:] = pages                    # no such page, one of them in what was shared
    groups = _groups(table, lens, P, 64)
    assert groups[3, :5].tolist() == [448] * 5
    _check(cache, q, table, lens, groups, news)
    table[5:9, :8] = -1                      # nothing of the prefix is there
    _check(cache, q, table, lens, groups, news)
    table[:] = -1
    assert float(_check(cache, q, table, lens, groups, news).abs().max()) == 0.0


def test_shared_attention_scales_zero_and_very_different():
    P, hq, hkv, hd = 16, 16, 2, 128
    rows = [("a", 1200, 3 * i) for i in range(6)]
    table, lens, pages = _forks(rows, P, 1, 7)
    cache = _filled(pages, hkv, P, hd, INT8, 4)
    g = _gen(11)
    cache.scales.mul_(torch.exp2(torch.randint(-30, 10, cache.scales.shape, device=DEV, generator=g).float()))
    cache.scales[0, 1, ::5] = 0.0           # values of nothing still take weight
    cache.scales[0, 0, ::7] = 0.0
    q = torch.randn(len(rows), hq * hd, device=DEV, generator=g).to(torch.bfloat16)
    q[2] *= 2.0 ** -100
    q[3] *= 2.0 ** 40
    q[4] = 0.0
    groups = _groups(table, lens, P, 64)
    cache.scales[0, 0].clamp_(max=0.05)
    _check(cache, q, table, lens, groups, scale=0.03)


def test_shared_attention_concentrated_on_either_part():
    # scores far apart: a row's weight lies in the prefix alone, or in its own positions alone
    P, hq, hkv, hd = 32, 4, 1, 64
    rows = [("a", 640, 200) for _ in range(4)]
    table, lens, pages = _forks(rows, P, 1, 9)
    cache = _filled(pages, hkv, P, hd, INT8, 6)
    q = torch.randn(4, hq * hd, device=DEV, generator=_gen(6)).to(torch.bfloat16) * 30
    groups = _groups(table, lens, P, 64)
    shared = table[0, :20].long()
    for part in (shared, table[0, 20:].long()):
        keep = cache.scales.clone()
        cache.scales[0, 0, part] = 1e-4
        _check(cache, q, table, lens, groups)
        cache.scales.copy_(keep)


def test_shared_attention_nan_and_infinity_stay_in_their_row():
    P, hq, hkv, hd = 16, 4, 1, 128
    rows = [("a", 400, i) for i in range(5)]
    table, lens, pages = _forks(rows, P, 1, 3)
    cache = _filled(pages, hkv, P, hd, INT8, 2)
    q = torch.randn(5, hq * hd, device=DEV, generator=_gen(2)).to(torch.bfloat16)
    groups, ws = _groups(table, lens, P, 64), kv8_attention_shared_workspace(cache, 5, hq, 1)
    _check(cache, q, table, lens, groups, ws=ws)
    bad = q.clone()
    bad[1, 5], bad[3, 200] = float("nan"), float("inf")
    out = torch.empty_like(q)
    kv8_attention_shared(cache, 0, bad, table, _i32(lens), groups, out, ws)
    assert bool(out[1, :hd].isnan().all()) and bool(out[3, hd:2 * hd].isnan().any())
    # the other rows and heads: rows of a warp share when their references move and which form of exp2 they take, so
    # their bits may differ from the clean call's; their error may not
    want, mag, most = _attention64(cache, q, table, lens, [1] * 5, hd ** -0.5, 0)
    off = (out.double() - want).abs() > 1.01 * 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2.0 ** -13) * mag + 2.0 ** -32 * most
    off[1, :hd] = off[3, hd:2 * hd] = False
    assert not bool(off.any()) and bool(out[[0, 2, 4]].isfinite().all()) and bool(out[1, hd:].isfinite().all())


def test_one_workspace_serves_calls_of_changing_lengths_and_groups():
    P, hq, hkv, hd = 16, 8, 2, 64
    rows = [(i % 2, 900 + 100 * (i % 2), 20 * i) for i in range(8)]
    table, lens, pages = _forks(rows, P, 1, 3)
    cache = _filled(pages, hkv, P, hd, E4M3, 1)
    ws = kv8_attention_shared_workspace(cache, 8, hq, 1)
    for i in range(6):
        now = [max(1, n - 150 * i) for n in lens]
        q = torch.randn(8, hq * hd, device=DEV, generator=_gen(i)).to(torch.bfloat16)
        _check(cache, q, table, now, _groups(table, now, P, 64 if i % 2 else 800), ws=ws)
    none = torch.zeros(4, 8, dtype=torch.int32, device=DEV)
    none[0] = -1
    _check(cache, q, table, lens, none, ws=ws)  # no groups at all


def test_without_groups_the_bits_are_those_of_kv8_attention():
    P, hq, hkv, hd, T = 32, 8, 2, 128, 2
    rows = [(None, 700, 9 * i) for i in range(5)]
    table, lens, pages = _forks(rows, P, T, 3)
    cache = _filled(pages, hkv, P, hd, INT8, 1)
    q = torch.randn(5 * T, hq * hd, device=DEV, generator=_gen(4)).to(torch.bfloat16)
    a, b = torch.empty_like(q), torch.empty_like(q)
    kv8_attention(cache, 0, q, table, _i32(lens), a, kv8_attention_workspace(cache, 5, hq, T))
    kv8_attention_shared(cache, 0, q, table, _i32(lens), _groups(table, lens, P, 64), b, kv8_attention_shared_workspace(cache, 5, hq, T))
    assert torch.equal(a, b)


def test_groups_that_do_not_belong_to_the_table_fault_nothing():
    P, hq, hkv, hd = 16, 8, 2, 64
    rows = [("a", 400, i) for i in range(6)]
    table, lens, pages = _forks(rows, P, 1, 3)
    cache = _filled(pages, hkv, P, hd, INT8, 1)
    q = torch.randn(6, hq * hd, device=DEV, generator=_gen(4)).to(torch.bfloat16)
    out, ws = torch.empty_like(q), kv8_attention_shared_workspace(cache, 6, hq, 1)
    good = _groups(table, lens, P, 64)
    for change in ((0, 2, -1), (0, 0, 6), (0, 1, 2 ** 31 - 1), (1, 0, -3), (1, 0, 7), (1, 0, 2 ** 31 - 1), (2, 0, 2 ** 31 - 1), (2, 0, -1),
                   (2, 1, 5), (3, 0, 2 ** 31 - 1), (3, 0, -2 ** 31), (3, 2, 37), (3, 4, 10 ** 6)):
        bad = good.clone()
        bad[change[0], change[1]] = change[2]
        kv8_attention_shared(cache, 0, q, table, _i32(lens), bad, out, ws)
    torch.cuda.synchronize()
    _check(cache, q, table, lens, good, ws=ws)


def test_shared_attention_on_another_stream_and_captured():
    P, hq, hkv, hd = 32, 8, 2, 128
    rows = [("a", 800, 11 * i) for i in range(5)]
    table, lens, pages = _forks(rows, P, 1, 3)
    cache = _filled(pages, hkv, P, hd, INT8, 1)
    q = torch.randn(5, hq * hd, device=DEV, generator=_gen(4)).to(torch.bfloat16)
    out, ws, ln = torch.empty_like(q), kv8_attention_shared_workspace(cache, 5, hq, 1), _i32(lens)
    groups = torch.empty(4, 5, dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        kv_pages_groups(table, ln, P, groups, least=64)
        kv8_attention_shared(cache, 0, q, table, ln, groups, out, ws)
    s.synchronize()
    assert torch.equal(out, _check(cache, q, table, lens, groups))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv_pages_groups(table, ln, P, groups, least=64)
        kv8_attention_shared(cache, 0, q, table, ln, groups, out, ws)
    ln.sub_(600)
    q.neg_()
    graph.replay()
    now = [n - 600 for n in lens]
    assert torch.equal(out, _check(cache, q, table, now, groups)) and int(groups[3].max()) == 192


def test_shared_refusals():
    cache = _filled(8, 2, 16, 64, INT8, 1)
    table, lens = _i32([[0, 1, 2], [0, 1, 3]]), _i32([40, 40])
    q = torch.zeros(2, 4 * 64, dtype=torch.bfloat16, device=DEV)
    out, groups, ws = torch.empty_like(q), _groups(table, [40, 40], 16, 32), kv8_attention_shared_workspace(cache, 2, 4, 1)
    kv8_attention_shared(cache, 0, q, table, lens, groups, out, ws)
    for change in (dict(groups=groups[:3]), dict(groups=groups.long()), dict(groups=groups.cpu()), dict(q=q[:, :64]), dict(out=out[:1]),
                   dict(lens=lens[:1]), dict(workspace=kv8_attention_workspace(cache, 2, 4, 1)), dict(workspace=ws.cpu()),
                   dict(status=torch.zeros(2, dtype=torch.int32, device=DEV)), dict(layer=1), dict(table=table.long()),
                   dict(new_lens=lens.long())):
        with pytest.raises(ValueError):
            kv8_attention_shared(**(dict(cache=cache, layer=0, q=q, table=table, lens=lens, groups=groups, out=out, workspace=ws) | change))
    for change in (dict(groups=groups.t()), dict(lens=lens.long()), dict(least=0), dict(page_size=0), dict(table=table.cpu())):
        with pytest.raises(ValueError):
            kv_pages_groups(**(dict(table=table, lens=lens, page_size=16, groups=groups) | change))
