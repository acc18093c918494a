"""Paged 8-bit KV cache on the GPU: store, read-back, attention and pages.

Codes, scales, tables and copies are compared for equality with a step-by-step
restatement of their definition; attention with the softmax in 64 bits over the
cache's own values.  Attention's tolerance: the output is rounded once to bf16
(relative 2^-8 of a value), and the weights enter the product in 16-bit floats
(2^-11 each), so an element may be off by 2^-8 of its own size plus 2^-11 times
the weighted mean of |v|, doubled for the sums in 32 bits.
"""
from __future__ import annotations

import pytest
import torch

from wal2026_b200.kv8 import (CODE_MAX, PagedKV8Cache, kv8_append, kv8_attention, kv8_attention_workspace, kv8_read,
                              kv_pages_assign, kv_pages_compact, kv_pages_copy)

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
INT8, E4M3 = torch.int8, torch.float8_e4m3fn


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _filled(layers, pages, hkv, P, hd, dtype, seed):
    g = _gen(seed)
    shape = (layers, 2, pages, hkv, P, hd)
    x = (torch.randn(shape, device=DEV, generator=g) * CODE_MAX[dtype] / 4).clamp(-CODE_MAX[dtype], CODE_MAX[dtype])
    codes = x.round().to(INT8) if dtype == INT8 else x.to(E4M3)
    scales = torch.rand(shape[:4], device=DEV, generator=g) * (4 / CODE_MAX[dtype]) + 1e-3
    return PagedKV8Cache(codes, scales)


def _values(cache, layer=0):
    """[2, pages, hkv, P, hd] fp32, the product rounded once."""
    return cache.codes[layer].float() * cache.scales[layer][..., None, None]


def _tables(lens, P, pages, seed, width=None, stride=None):
    """Rows of distinct pages in random order; int32 [B, width] with rows `stride` apart."""
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    need = [-(-n // P) for n in lens]
    width = width or max(1, max(need))
    buf = torch.full((len(lens), stride or width), -7, dtype=torch.int32)
    for b, n in enumerate(need):
        for j in range(n):
            buf[b, j] = order.pop()
    return buf.to(DEV)[:, :width]


# ----------------------------------------------------------------- attention

def _attention64(cache, layer, q, table, lens, news, scale):
    """(out, mean |v|) in float64; rows b * T + t."""
    B, hkv, P, hd = table.shape[0], cache.kv_heads, cache.page_size, cache.head_dim
    T, hq = q.shape[0] // B, q.shape[1] // hd
    G = hq // hkv
    val = cache.codes[layer].float().double() * cache.scales[layer].double()[..., None, None]
    out = torch.zeros(B, T, hq, hd, dtype=torch.float64, device=DEV)
    mag = torch.zeros_like(out)
    tab = table.tolist()
    for b in range(B):
        for t in range(min(T, news[b])):
            n = min(lens[b] + t + 1, table.shape[1] * P)
            ids = [(tab[b][j // P], j % P) for j in range(n) if 0 <= tab[b][j // P] < cache.num_pages]
            if not ids:
                continue
            pg, sl = (torch.tensor(v, device=DEV) for v in zip(*ids))
            for h in range(hkv):
                k, v = val[0, pg, h, sl], val[1, pg, h, sl]
                w = torch.softmax(q.double().view(B, T, hq, hd)[b, t, h * G:(h + 1) * G] @ k.T * scale, -1)
                out[b, t, h * G:(h + 1) * G] = w @ v
                mag[b, t, h * G:(h + 1) * G] = w @ v.abs()
    return out.view(B * T, -1), mag.view(B * T, -1)


def _check_attention(cache, q, table, lens, news=None, scale=None, layer=0, ws=None):
    B = table.shape[0]
    T, hd = q.shape[0] // B, cache.head_dim
    ws = kv8_attention_workspace(cache, B, q.shape[1] // hd, T) if ws is None else ws
    out = torch.full(q.shape, float("nan"), dtype=torch.bfloat16, device=DEV)
    nl = None if news is None else _i32(news)
    kv8_attention(cache, layer, q, table, _i32(lens), out, ws, new_lens=nl, scale=scale)
    want, mag = _attention64(cache, layer, q, table, lens, news or [T] * B, hd ** -0.5 if scale is None else scale)
    bad = ~((out.double() - want).abs() <= 2 * (2.0 ** -8 * want.abs() + 2.0 ** -11 * mag) + 1e-30)  # a NaN is bad too
    assert not bool(bad.any()), (int(bad.sum()), float((out.double() - want).abs().max()))
    again = torch.empty_like(out)
    kv8_attention(cache, layer, q, table, _i32(lens), again, ws, new_lens=nl, scale=scale)
    assert torch.equal(out, again)  # the same bits every time, and the workspace was left ready
    return out


@pytest.mark.parametrize("dtype", [INT8, E4M3])
@pytest.mark.parametrize("P,hd", [(16, 64), (32, 128), (64, 64), (64, 128), (16, 128)])
@pytest.mark.parametrize("hq,hkv,T", [(8, 2, 1), (4, 4, 3), (14, 2, 2), (5, 1, 7)])
def test_attention_matches_softmax_in_64_bits(dtype, P, hd, hq, hkv, T):
    lens = [0, 1, P - 1, P, 3 * P + 5, 200]
    ends = [n + T for n in lens]
    pages = sum(-(-n // P) for n in ends) + 2
    cache = _filled(2, pages, hkv, P, hd, dtype, P + hd + T)
    q = (torch.randn(len(lens) * T, hq * hd, device=DEV, generator=_gen(3)) * 2).to(torch.bfloat16)
    _check_attention(cache, q, _tables(ends, P, pages, 5), lens, layer=1)


@pytest.mark.parametrize("B,n,hq,hkv,T,P", [(1, 4097, 32, 8, 1, 64), (1, 9001, 8, 1, 4, 16), (3, 2500, 16, 2, 9, 32),
                                            (40, 333, 8, 8, 1, 16), (2, 700, 6, 1, 33, 64)])
def test_attention_over_long_and_split_lengths(B, n, hq, hkv, T, P):
    lens = [max(0, n - 97 * b) for b in range(B)]
    ends = [m + T for m in lens]
    pages = sum(-(-m // P) for m in ends)
    cache = _filled(1, pages, hkv, P, 128, INT8, n)
    q = torch.randn(B * T, hq * 128, device=DEV, generator=_gen(n)).to(torch.bfloat16)
    _check_attention(cache, q, _tables(ends, P, pages, 1), lens)


def test_attention_padding_rows_idle_sequences_and_missing_pages():
    P, hd, T = 16, 64, 4
    lens, news = [30, 0, 17, 100, 5], [4, 0, 2, 1, 9]
    cache = _filled(1, 64, 2, P, hd, INT8, 7)
    table = _tables([n + T for n in lens], P, 64, 2, width=7, stride=9)
    table[0, 1] = -1      # a hole in the middle
    table[3, 2] = 64      # past the pool
    table[4, :] = -5      # nothing at all
    q = torch.randn(len(lens) * T, 8 * hd, device=DEV, generator=_gen(9)).to(torch.bfloat16)
    out = _check_attention(cache, q, table, lens, news).view(len(lens), T, -1)
    assert not out[1].any() and not out[2, 2:].any() and not out[3, 1:].any() and not out[4].any()
    assert out[0].any() and out[2, 0].any()


def test_attention_beyond_the_table_reads_only_the_table():
    cache = _filled(1, 8, 1, 16, 64, INT8, 1)
    table = _tables([32], 16, 8, 3)
    q = torch.randn(2, 64, device=DEV, generator=_gen(2)).to(torch.bfloat16)
    _check_attention(cache, q, table, [1000])


@pytest.mark.parametrize("dtype", [INT8, E4M3])
def test_attention_ignores_what_lies_past_the_length(dtype):
    # a page's unused slots and its neighbours hold every byte there is, the scales of unused pages infinities and NaN
    P, hd = 32, 128
    cache = _filled(1, 6, 1, P, hd, dtype, 11)
    table = _i32([[3, 0, 5]])
    for page in (0, 1, 2, 4, 5):
        cache.codes[0, :, page] = torch.arange(P * hd, device=DEV).view(P, hd).to(torch.uint8).view(dtype)
    want = None
    for junk in (1.0, float("inf"), float("nan")):
        cache.scales[0, :, [1, 2, 4, 0, 5]] = junk
        q = torch.randn(1, 4 * hd, device=DEV, generator=_gen(12)).to(torch.bfloat16)
        out = torch.empty_like(q)
        kv8_attention(cache, 0, q, table, _i32([P - 8]), out, kv8_attention_workspace(cache, 1, 4))
        assert bool(out.isfinite().all())
        assert want is None or torch.equal(out, want)
        want = out
    cache.codes[0, :, 3, :, P - 7:] = torch.full((1,), 0x7F, dtype=torch.uint8, device=DEV).view(dtype)
    out = torch.empty_like(want)
    kv8_attention(cache, 0, q, table, _i32([P - 8]), out, kv8_attention_workspace(cache, 1, 4))
    assert torch.equal(out, want)


def test_attention_extreme_scores_and_scales():
    # one position far above the rest; blocks whose scales differ by 2^40; zero blocks; large and tiny queries
    P, hd, n = 16, 64, 150
    cache = _filled(1, 12, 1, P, hd, INT8, 21)
    cache.scales[0, 0] *= torch.logspace(-3, 3, 12, base=4, device=DEV)[:, None]
    cache.scales[0, 1] *= torch.logspace(-20, 20, 12, base=2, device=DEV)[:, None]
    cache.scales[0, 1, 4] = 0.0
    table = _tables([n], P, 12, 4)
    for size in (1e-30, 1e-3, 1.0, 50.0, 1e4):
        q = (torch.randn(1, 4 * hd, device=DEV, generator=_gen(22)) * size).to(torch.bfloat16)
        _check_attention(cache, q, table, [n - 1])
    _check_attention(cache, torch.zeros(1, 4 * hd, dtype=torch.bfloat16, device=DEV), table, [n - 1])
    q = torch.randn(1, 4 * hd, device=DEV, generator=_gen(23)).to(torch.bfloat16)
    _check_attention(cache, q, table, [n - 1], scale=0.0)
    _check_attention(cache, q, table, [n - 1], scale=-0.3)


def test_attention_of_more_sequences_than_the_balance_sums():
    # 1100 sequences take the path that gives each CTA whole units; some are empty tables, some idle
    P, hd, hq, hkv, B = 16, 64, 4, 2, 1100
    lens = [(i * 7) % 40 for i in range(B)]
    ends = [n + 1 for n in lens]
    pages = sum(-(-n // P) for n in ends)
    cache = _filled(1, pages, hkv, P, hd, E4M3, 51)
    table = _tables(ends, P, pages, 9)
    news = [0 if i % 13 == 5 else 1 for i in range(B)]
    q = torch.randn(B, hq * hd, device=DEV, generator=_gen(52)).to(torch.bfloat16)
    out = torch.full_like(q, float("nan"))
    kv8_attention(cache, 0, q, table, _i32(lens), out, kv8_attention_workspace(cache, B, hq), new_lens=_i32(news))
    for a in range(0, B, 550):  # the same rows in calls that are balanced: the order of sums differs, a rounding at most
        part = torch.empty_like(q[a:a + 550])
        kv8_attention(cache, 0, q[a:a + 550], table[a:a + 550], _i32(lens[a:a + 550]), part,
                      kv8_attention_workspace(cache, 550, hq), new_lens=_i32(news[a:a + 550]))
        diff = (part.float() - out[a:a + 550].float()).abs()
        assert bool((diff <= 2.0 ** -7 * part.float().abs() + 1e-6).all())
    pick = [0, 1, 5, 18, 700, 1099]
    want, mag = _attention64(cache, 0, q[pick], table[pick], [lens[i] for i in pick], [news[i] for i in pick], hd ** -0.5)
    assert bool(((out[pick].double() - want).abs() <= 2 * (2.0 ** -8 * want.abs() + 2.0 ** -11 * mag) + 1e-30).all())


@pytest.mark.parametrize("dtype", [INT8, E4M3])
@pytest.mark.parametrize("hq,T", [(4, 1), (8, 2), (8, 3), (16, 4)])
def test_attention_every_code_counts(dtype, hq, T):
    # each code as a V value at one position that has nearly all the weight, e4m3's subnormals included, and as a K value
    P, hd, n = 64, 64, 256
    codes = torch.arange(256, device=DEV).to(torch.uint8)
    if dtype == INT8:
        codes[128] = 0  # -128 is not a code
    else:
        codes[0x7F], codes[0xFF] = 0, 0  # NaN is none either
    cache = _filled(1, 4, 1, P, hd, dtype, 61)
    cache.scales[:] = 1.0
    cache.codes.view(torch.uint8)[0, 1, :, 0] = codes.view(4, P, 1).expand(4, P, hd)  # V: position j holds code j in every dim
    for shift in (0, 100):
        k = torch.zeros(n, hd, dtype=torch.uint8, device=DEV)
        for d in range(hd):
            k[:, d] = codes.roll(shift + 3 * d)
        cache.codes.view(torch.uint8)[0, 0, :, 0] = k.view(4, P, hd)
        q = (torch.randn(T, hq * hd, device=DEV, generator=_gen(62 + shift)) * 0.02).to(torch.bfloat16)
        _check_attention(cache, q, _i32([[0, 1, 2, 3]]), [n - T])


@pytest.mark.parametrize("hq,T", [(4, 1), (8, 2), (16, 4)])
def test_attention_keeps_a_bad_row_to_itself(hq, T):
    P, hd = 32, 128
    cache = _filled(1, 20, 1, P, hd, INT8, 71)
    table = _tables([500], P, 20, 3)
    q = torch.randn(T, hq * hd, device=DEV, generator=_gen(72)).to(torch.bfloat16)
    ws = kv8_attention_workspace(cache, 1, hq, T)
    good, bad = torch.empty_like(q), torch.empty_like(q)
    kv8_attention(cache, 0, q, table, _i32([500 - T]), good, ws)
    for value in (float("nan"), float("inf")):
        worse = q.clone()
        worse[T - 1, hd + 5] = value  # head 1 of the last token
        kv8_attention(cache, 0, worse, table, _i32([500 - T]), bad, ws)
        assert bool(bad[T - 1, hd:2 * hd].isnan().all())
        rest = torch.ones_like(q, dtype=torch.bool)
        rest[T - 1, hd:2 * hd] = False
        assert torch.equal(bad[rest], good[rest])


def test_attention_strided_rows_one_workspace_and_another_stream():
    P, hd, hq, hkv = 64, 128, 8, 2
    cache = _filled(1, 80, hkv, P, hd, E4M3, 31)
    wide = torch.randn(6, hq * hd + 2 * 512, device=DEV, generator=_gen(32)).to(torch.bfloat16)
    ws = kv8_attention_workspace(cache, 6, hq, 1)
    for lens in ([10, 400, 0, 77, 900, 64], [900, 1, 2, 3, 4, 5]):
        table = _tables([n + 1 for n in lens], P, 80, 6)
        _check_attention(cache, wide[:, 512:512 + hq * hd], table, lens, ws=ws)
        _check_attention(cache, wide[:3, :hq * hd], table[:3], lens[:3], ws=ws)  # a smaller call
    side = torch.cuda.Stream()
    table, ln = _tables([901], P, 80, 6), _i32([900])
    q = wide[:1, :hq * hd].contiguous()
    a, b = torch.empty_like(q), torch.empty_like(q)
    kv8_attention(cache, 0, q, table, ln, a, ws)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kv8_attention(cache, 0, q, table, ln, b, ws)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, b)


def test_attention_workspace_shared_by_steps_of_different_sizes():
    # one workspace for steps of 1 to 30 tokens in turn: each must find its counters at zero
    P, hd, hq, hkv, B = 64, 64, 8, 1, 2
    lens = [3000, 1700]
    cache = _filled(1, 80, hkv, P, hd, INT8, 81)
    table = _tables([n + 30 for n in lens], P, 80, 4)
    ws = kv8_attention_workspace(cache, B, hq, 30)
    for T in (1, 12, 1, 16, 2, 30, 1, 3, 5, 1, 8, 6, 1):
        q = torch.randn(B * T, hq * hd, device=DEV, generator=_gen(T)).to(torch.bfloat16)
        _check_attention(cache, q, table, lens, ws=ws)


def test_attention_offsets_past_32_bits():
    # 2.4e9 code bytes in one pool half: the last page starts past 2^31
    P, hd, hkv, pages = 64, 128, 8, 36700
    codes = torch.zeros(1, 2, pages, hkv, P, hd, dtype=INT8, device=DEV)
    cache = PagedKV8Cache(codes, torch.zeros(1, 2, pages, hkv, device=DEV))
    small = _filled(1, 3, hkv, P, hd, INT8, 41)
    ids = [pages - 1, 3, pages - 2]
    for i, p in enumerate(ids):
        codes[0, :, p] = small.codes[0, :, i]
        cache.scales[0, :, p] = small.scales[0, :, i]
    q = torch.randn(1, 16 * hd, device=DEV, generator=_gen(42)).to(torch.bfloat16)
    outs = []
    for c, t in ((cache, ids), (small, [0, 1, 2])):
        out = torch.empty_like(q)
        kv8_attention(c, 0, q, _i32([t]), _i32([170]), out, kv8_attention_workspace(c, 1, 16))
        outs.append(out)
    assert torch.equal(*outs)
    k, v = (torch.empty(1, hkv, 171, hd, device=DEV) for _ in range(2))
    kv8_read(cache, 0, _i32([ids]), _i32([0]), _i32([171]), k, v)
    want = _values(small)[0].transpose(0, 1).reshape(hkv, -1, hd)[:, :171]
    assert torch.equal(k[0], want)


# ------------------------------------------------------------ store and read

def _code(x, dtype):
    """The nearest code's value: round to nearest even, clamped; NaN gives 0."""
    x = torch.nan_to_num(x.double(), nan=0.0, posinf=1e300, neginf=-1e300).clamp(-CODE_MAX[dtype], CODE_MAX[dtype])
    if dtype == INT8:
        return x.round()
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))  # spacing 2^(e - 3); subnormals below 2^-6
    return torch.round(x * torch.exp2(3 - e)) * torch.exp2(e - 3)


def _f32(x):
    return x.float()


def _append_reference(cache, layer, qkv, hq, table, lens, news, cos, sin):
    """Updates the cache's tensors on the CPU, block by block, and returns (codes as values, scales, q_out)."""
    hkv, P, hd, dt = cache.kv_heads, cache.page_size, cache.head_dim, cache.codes.dtype
    val, sc = cache.codes[layer].float().cpu(), cache.scales[layer].cpu().clone()
    B, tab = table.shape[0], table.tolist()
    T = qkv.shape[0] // B
    x = qkv.float().cpu().view(B, T, hq + 2 * hkv, hd)
    q = torch.zeros(B, T, hq, hd)
    inv = torch.tensor(1.0) / torch.tensor(CODE_MAX[dt])
    for b in range(B):
        m = max(0, min(news[b], T))
        if cos is not None:
            m = max(0, min(m, cos.shape[0] - lens[b]))
            c, s = (t[lens[b]:lens[b] + m].cpu()[:, None] for t in (cos, sin))

            def turn(y):
                y1, y2 = y[..., :hd // 2], y[..., hd // 2:]
                return torch.cat([y1 * c + (-y2) * s, y2 * c + y1 * s], -1)
        else:
            def turn(y):
                return y
        q[b, :m] = turn(x[b, :m, :hq])
        for kv, new in enumerate((turn(x[b, :m, hq:hq + hkv]), x[b, :m, hq + hkv:])):
            for j in range(lens[b] // P, -(-(lens[b] + m) // P) if m else 0):
                page = tab[b][j] if j < len(tab[b]) else -1
                if not 0 <= page < cache.num_pages:
                    continue
                lo, hi = max(lens[b], j * P), min(lens[b] + m, (j + 1) * P)
                for h in range(hkv):
                    y = new[lo - lens[b]:hi - lens[b], h]
                    a = torch.where(y.isfinite(), y.abs(), torch.zeros(())).max()
                    old = sc[kv, page, h].clone() if lo > j * P else torch.zeros(())
                    s1 = torch.maximum(old, a * inv)
                    if s1 > old and lo > j * P:
                        val[kv, page, h, :lo - j * P] = _code(val[kv, page, h, :lo - j * P] * (old / s1), dt).float()
                    sc[kv, page, h] = s1
                    val[kv, page, h, lo - j * P:hi - j * P] = _code(y / s1, dt).float() if s1 > 0 else 0.0
    return val, sc, q.view(B * T, hq * hd).to(torch.bfloat16)


def _rope(max_pos, hd):
    ang = torch.arange(max_pos, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)
    return ang.cos().float().to(DEV), ang.sin().float().to(DEV)


def _check_append(cache, qkv, hq, table, lens, news=None, rope=None, layer=0):
    T = qkv.shape[0] // table.shape[0]
    cos, sin = rope if rope else (None, None)
    want = _append_reference(cache, layer, qkv, hq, table, lens, news or [T] * table.shape[0], cos, sin)
    q = torch.full((qkv.shape[0], hq * cache.head_dim), float("nan"), dtype=torch.bfloat16, device=DEV)
    kv8_append(cache, layer, qkv, hq, table, _i32(lens), q, cos=cos, sin=sin, new_lens=None if news is None else _i32(news))
    assert torch.equal(cache.scales[layer].cpu(), want[1])
    assert torch.equal(cache.codes[layer].float().cpu(), want[0])
    assert torch.equal(q.cpu(), want[2])


@pytest.mark.parametrize("dtype", [INT8, E4M3])
@pytest.mark.parametrize("P,hd", [(16, 64), (32, 128), (64, 64), (64, 128), (32, 64), (16, 128)])
@pytest.mark.parametrize("T", [1, 3, 70])
def test_append_equals_its_definition(dtype, P, hd, T):
    hq, hkv, lens = 4, 2, [0, 1, P - 1, P, 2 * P + 3]
    ends = [n + T for n in lens]
    pages = sum(-(-n // P) for n in ends) + 2
    cache = _filled(2, pages, hkv, P, hd, dtype, T)
    qkv = torch.randn(len(lens) * T, (hq + 2 * hkv) * hd, device=DEV, generator=_gen(T + P)).to(torch.bfloat16)
    _check_append(cache, qkv, hq, _tables(ends, P, pages, 3), lens, rope=_rope(max(ends), hd), layer=1)


@pytest.mark.parametrize("dtype", [INT8, E4M3])
def test_append_token_by_token_grows_scales_and_keeps_earlier_values(dtype):
    P, hd, hkv = 16, 64, 2
    cache = PagedKV8Cache.allocate(1, 4, hkv, hd, page_size=P, dtype=dtype, device=DEV)
    table = _i32([[2, 0, 3]])
    g = _gen(5)
    rows = torch.randn(40, (2 + 2 * hkv) * hd, device=DEV, generator=g) * torch.exp(torch.randn(40, 1, device=DEV, generator=g))
    rows = rows.to(torch.bfloat16)
    for t in range(40):
        _check_append(cache, rows[t:t + 1], 2, table, [t])
    k, v = (torch.empty(1, hkv, 48, hd, device=DEV) for _ in range(2))
    kv8_read(cache, 0, table, _i32([0]), _i32([40]), k, v)
    x = rows.float().view(40, -1, hd)[:, 2:4].transpose(0, 1)
    top = torch.stack([x[:, i:i + 16].abs().amax((1, 2)) for i in (0, 16, 32)])  # [3, hkv]
    # each growth of a block's scale rounds its codes once more: at most 16 roundings of half a code (int8), of 2^-4 of the
    # value (e4m3, whose subnormal codes are spaced 2^-9 of 448)
    for i in range(3):
        d = (k[0, :, 16 * i:16 * i + 16][:, :min(16, 40 - 16 * i)] - x[:, 16 * i:16 * i + 16]).abs()
        lim = 8.5 * top[i][:, None, None] / 127 if dtype == INT8 else x[:, 16 * i:16 * i + 16].abs() * (1.0625 ** 16 - 1) + top[i][:, None, None] * 16 * 2.0 ** -10 / 448
        assert bool((d <= lim).all())
    assert not k[0, :, 40:].any() and not v[0, :, 40:].any()


def test_append_special_values():
    P, hd = 16, 64
    for dtype in (INT8, E4M3):
        cache = _filled(1, 3, 1, P, hd, dtype, 8)
        rows = torch.randn(5, 3 * hd, device=DEV, generator=_gen(9)).to(torch.bfloat16)
        rows[0, hd + 3], rows[1, hd + 5], rows[2, 2 * hd + 1] = float("inf"), float("-inf"), float("nan")
        rows[3, hd:] = 0
        _check_append(cache, rows, 1, _i32([[1]]), [4])
        zero = torch.zeros(2, 3 * hd, dtype=torch.bfloat16, device=DEV)
        _check_append(cache, zero, 1, _i32([[2]]), [0])  # a block of zeros has scale 0
        zero[0, hd:] = float("nan")
        _check_append(cache, zero, 1, _i32([[2]]), [0])
        tiny = (torch.randn(2, 3 * hd, device=DEV, generator=_gen(10)) * 1e-38).to(torch.bfloat16)
        _check_append(cache, tiny, 1, _i32([[2]]), [0])
        huge = (torch.randn(2, 3 * hd, device=DEV, generator=_gen(11)) * 1e38).to(torch.bfloat16)
        _check_append(cache, huge, 1, _i32([[2]]), [2])


def test_append_skips_padding_missing_pages_and_positions_past_the_tables():
    P, hd, hkv, hq, T = 16, 64, 2, 4, 20
    lens, news = [10, 0, 40, 3, 60], [20, 0, 7, -1, 20]
    cache = _filled(1, 20, hkv, P, hd, INT8, 12)
    table = _tables([n + T for n in lens], P, 20, 6, width=4, stride=6)
    table[0, 1] = -1
    qkv = torch.randn(len(lens) * T, (hq + 2 * hkv) * hd + 64, device=DEV, generator=_gen(13)).to(torch.bfloat16)[:, 32:-32]
    _check_append(cache, qkv, hq, table, lens, news, rope=_rope(70, hd))  # positions 70.. have no rotation


@pytest.mark.parametrize("dtype,out", [(INT8, torch.float32), (E4M3, torch.bfloat16), (INT8, torch.bfloat16)])
@pytest.mark.parametrize("P,hd,L", [(16, 64, 37), (64, 128, 130), (32, 128, 1)])
def test_read_gives_the_stored_values(dtype, out, P, hd, L):
    first, count = [0, 5, P, 2 * P + 1, 7], [L, 0, min(3, L), L + 50, -2]
    pages, hkv = 40, 3
    cache = _filled(2, pages, hkv, P, hd, dtype, L)
    table = _tables([400 if P == 64 else 120] * 5, P, pages, 8, stride=11)
    table[0, 1:2] = -1
    k, v = (torch.full((5, hkv, L, hd), float("nan"), device=DEV, dtype=out) for _ in range(2))
    kv8_read(cache, 1, table, _i32(first), _i32(count), k, v)
    val, tab = _values(cache, 1), table.tolist()
    for i, got in enumerate((k, v)):
        want = torch.zeros_like(got)
        for b in range(5):
            for l in range(max(0, min(L, count[b]))):
                j = (first[b] + l) // P
                if j < len(tab[b]) and 0 <= tab[b][j] < pages:
                    want[b, :, l] = val[i, tab[b][j], :, (first[b] + l) % P].to(out)
        assert torch.equal(got, want)


# --------------------------------------------------------------------- pages

def _assign_reference(table, parent, keep, add, P, pages):
    width = len(table[0])
    rows, lost = [], 0
    for p, k in zip(parent, keep):
        k = min(max(k, 0), width * P) if 0 <= p < len(table) else 0
        rows.append([e if 0 <= e < pages else -1 for e in table[p][:-(-k // P)]] if k else [])
    keep = [min(max(k, 0), width * P) if 0 <= p < len(table) else 0 for p, k in zip(parent, keep)]
    add = [max(a, 0) for a in add]
    users = {}
    for r, row in enumerate(rows):
        for j, e in enumerate(row):
            if e >= 0:
                users.setdefault(e, []).append((r, add[r] > 0 and keep[r] % P != 0 and j == len(row) - 1))
    free = [p for p in range(pages) if p not in users]
    src, dst = [-1] * len(rows), [-1] * len(rows)
    out = [list(r) for r in rows]
    for r, row in enumerate(out):
        if add[r] and keep[r] % P and row[-1] >= 0:
            mine = users[row[-1]]
            if len(mine) > 1 and not (all(w for _, w in mine) and mine[0][0] == r):
                if free:
                    src[r], dst[r] = row[-1], free.pop(0)
                else:
                    lost += 1
                row[-1] = dst[r]
        want = -(-(keep[r] + add[r]) // P)
        lost += max(0, want - width) if add[r] else 0
        for _ in range(len(row), min(want, width) if add[r] else len(row)):
            row.append(free.pop(0) if free else -1)
            lost += row[-1] < 0
    ref = [0] * pages
    for row in out:
        for e in row:
            if e >= 0:
                ref[e] += 1
    return [r + [-1] * (width - len(r)) for r in out], ref, src, dst, [ref.count(0), lost]


def _check_assign(table, parent, keep, add, P, pages, stride=None):
    rows, width = len(parent), table.shape[1]
    buf = torch.full((rows, stride or width), 99, dtype=torch.int32, device=DEV)
    ref, src, dst, info = (torch.full((n,), 77, dtype=torch.int32, device=DEV) for n in (pages, rows, rows, 2))
    before = table.clone()
    kv_pages_assign(table, _i32(parent), _i32(keep), _i32(add), P, buf[:, :width], ref, src, dst, info)
    want = _assign_reference(table.tolist(), parent, keep, add, P, pages)
    got = (buf[:, :width], ref, src, dst, info)
    for name, g, w in zip(("table", "ref", "src", "dst", "info"), got, want):
        assert g.tolist() == w, name
    assert torch.equal(table, before)
    return got


@pytest.mark.parametrize("P", [16, 64])
@pytest.mark.parametrize("seed", range(6))
def test_assign_equals_its_definition(P, seed):
    rng = torch.Generator().manual_seed(seed)

    def ints(lo, hi, n):
        return torch.randint(lo, hi, (n,), generator=rng).tolist()

    rows_in, rows = 9, 13 + seed
    lens = ints(0, 6 * P, rows_in)
    pages = (40, 60, 200)[seed % 3]  # the first cannot hold everything
    table = _tables(lens, P, max(pages, 60), seed, width=8)
    parent = ints(-2, rows_in + 1, rows)
    keep = [min(k, lens[p]) if 0 <= p < rows_in else k for p, k in zip(parent, ints(-3, 6 * P, rows))]
    add = [a if a > 0 else 0 for a in ints(-P, 2 * P, rows)]
    add[0] = 9 * P  # more than a row holds
    _check_assign(table, parent, keep, add, P, pages, stride=8 + seed)


def test_assign_shared_last_pages():
    P = 16
    table = _i32([[4, 7, -1], [2, 9, 5]])
    # three writers of page 7: the lowest keeps it; with a reader all of them copy; a longer row holds page 9 whole
    _check_assign(table, [0, 0, 0], [20, 20, 20], [1, 1, 1], P, 12)
    _check_assign(table, [0, 0, 0], [20, 20, 20], [1, 0, 1], P, 12)
    _check_assign(table, [1, 1], [20, 48], [3, 0], P, 12)
    _check_assign(table, [0, 0], [16, 16], [1, 1], P, 12)  # nothing partly filled: nothing to copy
    _check_assign(table, [0, 1], [0, 0], [0, 0], P, 12)    # everything freed
    _check_assign(table, [0, 0], [20, 20], [1, 1], P, 10)


def test_assign_many_rows_and_pages():
    P, rows = 16, 3000
    lens = [(37 * i) % 200 for i in range(rows)]
    need = sum(-(-n // P) for n in lens)
    table = _tables(lens, P, need + rows, 2)
    _check_assign(table, [i if i % 5 else i // 2 for i in range(rows)], [n if i % 5 else lens[i // 2] for i, n in enumerate(lens)],
                  [i % 3 for i in range(rows)], P, need + rows)


def test_assign_as_many_rows_as_it_takes():
    P, rows = 16, 16383
    table = _i32([[0, 1]])
    # every row continues one sequence: page 0 is shared, page 1 copied by all but the first, and a page runs short
    _check_assign(table, [0] * rows, [20] * rows, [1] * rows, P, rows)


@pytest.mark.parametrize("P,pages,rows,hi", [(16, 50, 4, 100), (64, 3000, 40, 2000), (32, 8, 1, 0), (16, 2049, 300, 90)])
def test_compact_equals_its_definition(P, pages, rows, hi):
    lens = [(hi * (i + 1)) // rows - (i % 3 if hi else 0) for i in range(rows)]
    table = _tables(lens, P, pages, 3, width=max(1, -(-hi // P)) + 1)
    if rows > 3:
        lens[2] = lens[3]
        table[2] = table[3]  # a shared prefix
    for out in (torch.empty_like(table), table):
        tab = table.tolist()
        remap, src, dst = (torch.full((pages,), 9, dtype=torch.int32, device=DEV) for _ in range(3))
        info = torch.empty(2, dtype=torch.int32, device=DEV)
        kv_pages_compact(table, _i32(lens), P, out, remap, src, dst, info)
        used = sorted({e for row, n in zip(tab, lens) for e in row[:-(-n // P)] if e >= 0})
        moves = list(zip([p for p in used if p >= len(used)], [p for p in range(len(used)) if p not in set(used)]))
        new = {p: p for p in used} | dict(moves)
        pad = [-1] * (pages - len(moves))
        assert info.tolist() == [len(used), len(moves)]
        assert src.tolist() == [m[0] for m in moves] + pad and dst.tolist() == [m[1] for m in moves] + pad
        assert remap.tolist() == [new.get(p, -1) for p in range(pages)]
        assert out.tolist() == [[new[e] if j < -(-n // P) else -1 for j, e in enumerate(row)] for row, n in zip(tab, lens)]


@pytest.mark.parametrize("dtype,layers,hkv,P,hd", [(INT8, 3, 2, 16, 64), (E4M3, 1, 8, 64, 128), (INT8, 2, 5, 32, 64)])
def test_copy_moves_pages_of_every_layer(dtype, layers, hkv, P, hd):
    pages = 100
    cache = _filled(layers, pages, hkv, P, hd, dtype, layers)
    codes, scales = cache.codes.view(torch.uint8).clone(), cache.scales.clone()
    perm = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).tolist()
    src, dst = perm[:40], perm[40:80]
    src[3], dst[5], src[7], dst[9] = -1, -1, pages, 1 << 30  # skipped
    for s, d in zip(src, dst):
        if 0 <= s < pages and 0 <= d < pages:
            codes[:, :, d], scales[:, :, d] = codes[:, :, s], scales[:, :, s]
    kv_pages_copy(cache, _i32(src), _i32(dst))
    assert torch.equal(cache.codes.view(torch.uint8), codes) and torch.equal(cache.scales, scales)


def test_fork_append_and_attend_like_separate_sequences():
    # a prompt shared by three samples and then written by each gives what three caches of their own give
    P, hd, hq, hkv, n = 16, 64, 4, 2, 37
    g = _gen(77)
    shared = PagedKV8Cache.allocate(2, 30, hkv, hd, page_size=P, device=DEV)
    single = PagedKV8Cache.allocate(2, 30, hkv, hd, page_size=P, device=DEV)
    prompt = torch.randn(n, (hq + 2 * hkv) * hd, device=DEV, generator=g).to(torch.bfloat16)
    nxt = torch.randn(3, (hq + 2 * hkv) * hd, device=DEV, generator=g).to(torch.bfloat16)
    t0, t1 = torch.full((1, 5), -1, dtype=torch.int32, device=DEV), torch.empty(3, 5, dtype=torch.int32, device=DEV)
    first = torch.empty_like(t0)

    def bufs(rows):
        return [torch.empty(k, dtype=torch.int32, device=DEV) for k in (30, rows, rows, 2)]

    ref, src, dst, info = bufs(1)
    kv_pages_assign(t0, _i32([-1]), _i32([0]), _i32([n]), P, first, ref, src, dst, info)
    for layer in range(2):
        kv8_append(shared, layer, prompt, hq, first, _i32([0]), torch.empty(n, hq * hd, dtype=torch.bfloat16, device=DEV))
    ref, src, dst, info = bufs(3)
    kv_pages_assign(first, _i32([0, 0, 0]), _i32([n] * 3), _i32([1] * 3), P, t1, ref, src, dst, info)
    kv_pages_copy(shared, src, dst)
    assert info.tolist() == [30 - 5, 0] and ref.tolist()[:3] == [3, 3, 1]
    own = torch.arange(9, dtype=torch.int32, device=DEV).view(3, 3)
    for layer in range(2):
        q = torch.empty(3, hq * hd, dtype=torch.bfloat16, device=DEV)
        kv8_append(shared, layer, nxt, hq, t1, _i32([n] * 3), q)
        for i in range(3):
            kv8_append(single, layer, prompt, hq, own[i:i + 1], _i32([0]), torch.empty(n, hq * hd, dtype=torch.bfloat16, device=DEV))
        kv8_append(single, layer, nxt, hq, own, _i32([n] * 3), torch.empty_like(q))
        a, b = torch.empty_like(q), torch.empty_like(q)
        kv8_attention(shared, layer, q, t1, _i32([n] * 3), a, kv8_attention_workspace(shared, 3, hq))
        kv8_attention(single, layer, q, own, _i32([n] * 3), b, kv8_attention_workspace(single, 3, hq))
        assert torch.equal(a, b)
