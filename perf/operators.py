"""Cases of the paged 8-bit KV cache and of speculative decoding, for timing and for comparing outputs.

Four operators, each in a plain form (elementary torch operations in 32 bits) and
as the call a user makes of this package:

  append     rotary positions and 8-bit store of new tokens, and reading the
             touched pages back
  attention  grouped-query attention of one or several new tokens over the cache
  assign     tables of the next step (kept, forked, freed and new pages) and the
             copies of pages that two sequences would write
  compact    used pages moved to the front of the pool
  verify     drafted tokens against the target's probabilities

``listed()`` names the cases, ``draw(rng)`` draws one more from the same ranges,
``prepare`` makes what a program holds before the call, ``run`` is one call and
``exact`` the result from the definition in 64 bits.  Lengths are a function of
the case alone (so ``work`` can count them); values come from the seed.
"""
import math

import torch

own = False

QMAX = {"int8": 127.0, "e4m3": 448.0}
CODE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
ONE = 1 << 38  # fixed-point unit of a probability


# ------------------------------------------------------------------ cases

def listed():
    return [
        # one sequence at the 2048-token context that the decode benchmark uses, Llama-3-8B heads: the latency of a single chat
        dict(name="attention single 2048", op="attention", B=1, T=1, hq=32, hkv=8, hd=128, P=64, kind="int8", lo=2047, hi=2047, ragged=False),
        # a serving batch of sequences of every length up to the 70B benchmark context, small pages
        dict(name="attention batch ragged", op="attention", B=48, T=1, hq=64, hkv=8, hd=128, P=16, kind="e4m3", lo=0, hi=4096, ragged=False),
        # a speculative step: up to four drafts and the token before them
        dict(name="attention drafts", op="attention", B=16, T=5, hq=32, hkv=8, hd=128, P=32, kind="int8", lo=500, hi=8191, ragged=True),
        # few sequences with long documents
        dict(name="attention long", op="attention", B=4, T=1, hq=64, hkv=8, hd=128, P=64, kind="int8", lo=100001, hi=131071, ragged=False),
        # a decode step of a small batch: latency
        dict(name="append decode", op="append", B=3, T=1, hq=32, hkv=8, hd=64, P=16, kind="e4m3", lo=7, hi=1500, ragged=False, read="fp32"),
        # prompts entering the cache
        dict(name="append prompts", op="append", B=4, T=2048, hq=64, hkv=8, hd=128, P=64, kind="int8", lo=0, hi=33, ragged=True, read="bf16"),
        # eight prompts, each sampled eight ways: shared pages, and a copy of the last one for every sample but the first
        dict(name="assign fork", op="assign", rows=8, fork=8, lo=1500, hi=2047, P=64, hkv=8, hd=64, layers=16, kind="int8"),
        # one more token for each of 256 sequences of one shard: table work, hardly a copy
        dict(name="assign step", op="assign", rows=256, fork=1, lo=1, hi=8191, P=16, hkv=1, hd=64, layers=1, kind="e4m3"),
        # a small pool
        dict(name="compact small", op="compact", rows=6, lo=0, hi=300, P=32, hkv=2, hd=64, layers=2, live=0.6, kind="int8"),
        # a fragmented pool of a layer group
        dict(name="compact pool", op="compact", rows=24, lo=100, hi=1400, P=16, hkv=8, hd=128, layers=8, live=0.55, kind="int8"),
        # one sequence, four drafts, the stacks' vocabulary
        dict(name="verify single", op="verify", B=1, T=4, V=128256, draft=True, ragged=False),
        # a batch, up to eight drafts
        dict(name="verify batch", op="verify", B=64, T=8, V=128256, draft=True, ragged=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "append", "assign", "compact", "verify"])
    kind, P, hd = rng.choice(["int8", "e4m3"]), rng.choice([16, 32, 64]), rng.choice([64, 128])
    if op == "attention":
        hq, hkv = rng.choice([(32, 8), (64, 8), (8, 1), (8, 8), (12, 4), (14, 2)])
        hi, most = _log(rng, 1, 131071), 4 * 131071 * 8  # most: key rows of the longest listed case, at eight query rows each
        T = max(1, min(rng.choice([1, 1, 2, 3, 5, 8]), 8 * most // (hi * hq)))
        B = max(1, min(_log(rng, 1, 64), 8 * most // (hi * max(8 * hkv, hq * T))))
        return dict(op=op, B=B, T=T, hq=hq, hkv=hkv, hd=hd, P=P, kind=kind,
                    lo=rng.choice([0, hi // 2, hi]), hi=hi, ragged=rng.random() < 0.5)
    if op == "append":
        hq, hkv = rng.choice([(32, 8), (64, 8), (8, 1), (12, 4)])
        T = _log(rng, 1, 2048)
        B = max(1, min(_log(rng, 1, 64), 4 * 2048 // T))
        return dict(op=op, B=B, T=T, hq=hq, hkv=hkv, hd=hd, P=P, kind=kind, lo=0, hi=_log(rng, 1, 4000),
                    ragged=rng.random() < 0.5, read=rng.choice(["fp32", "bf16"]))
    if op == "assign":
        rows, fork = _log(rng, 1, 64), rng.choice([1, 2, 3, 8])
        hi = _log(rng, 1, max(2, min(8191, 8 * 2047 // rows)))
        return dict(op=op, rows=rows, fork=fork, lo=rng.choice([0, hi // 2]), hi=hi, P=P, hkv=rng.choice([1, 2, 8]), hd=64,
                    layers=rng.choice([1, 4, 16]), kind=kind)
    if op == "compact":
        rows = _log(rng, 1, 24)
        hi = _log(rng, 1, 1400)
        return dict(op=op, rows=rows, lo=rng.choice([0, hi // 2]), hi=hi, P=P, hkv=rng.choice([1, 2, 8]), hd=64,
                    layers=rng.choice([1, 4, 8]), live=rng.uniform(0.2, 1.0), kind=kind)
    return dict(op=op, B=_log(rng, 1, 64), T=rng.choice([1, 2, 4, 7, 8]), V=_log(rng, 1000, 128255) | 1,
                draft=rng.random() < 0.7, ragged=rng.random() < 0.5)


def _spread(lo, hi, n):
    """n lengths over [lo, hi], the longest among them."""
    out = [lo + int((hi - lo) * ((0.6180339887498949 * (i + 1)) % 1.0)) for i in range(n)]
    out[0] = hi
    return out


def _lens(c):
    return _spread(c["lo"], c["hi"], c["B"])


def _news(c):
    """New tokens of each sequence: up to T, an idle sequence among eight or more."""
    T, B = c["T"], c["B"]
    if not c["ragged"]:
        return [T] * B
    out = [T - int(0.6 * T * ((0.7548776662466927 * i) % 1.0)) for i in range(B)]
    if B >= 8:
        out[B - 2] = 0
    return out


def _cdiv(a, b):
    return -(-a // b)


# ----------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _pool(c, layers, pages, g):
    """Codes and scales of a filled pool: values around one, larger in some heads."""
    shape = (layers, 2, pages, c["hkv"], c["P"], c["hd"])
    codes = torch.empty(shape, dtype=CODE[c["kind"]], device="cuda")
    for l in range(layers):
        for kv in range(2):
            x = torch.randn(shape[2:], device="cuda", generator=g) * (QMAX[c["kind"]] / 4.0)
            x = x.clamp_(-QMAX[c["kind"]], QMAX[c["kind"]])
            codes[l, kv] = x.round_().to(torch.int8) if c["kind"] == "int8" else x.to(CODE["e4m3"])
    scales = (4.0 / QMAX[c["kind"]]) * torch.exp(0.3 * torch.randn(shape[:4], device="cuda", generator=g))
    return codes, scales.float().contiguous()


def _table(lens, P, pages, width, g):
    """Rows of pages in random order, -1 past each row's length."""
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    need = torch.tensor([_cdiv(n, P) for n in lens], device="cuda")
    begin = need.cumsum(0) - need
    j = torch.arange(width, device="cuda")
    at = (begin[:, None] + j[None, :]).clamp(max=pages - 1)
    return torch.where(j[None, :] < need[:, None], order[at], torch.full_like(order[at], -1)).contiguous()


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _inputs(c, seed):
    g = _gen(seed)
    op, s = c["op"], {}
    if op in ("attention", "append"):
        lens, news = _lens(c), _news(c)
        ends = [a + b for a, b in zip(lens, news)]
        width = max(1, _cdiv(max(ends), c["P"]))
        pages = sum(_cdiv(n, c["P"]) for n in ends) + 3
        s["codes"], s["scales"] = _pool(c, 1, pages, g)
        s["table"] = _table(ends, c["P"], pages, width, g)
        s["lens"], s["news"] = _ints(lens), _ints(news)
        M = c["B"] * c["T"]
        if op == "attention":
            s["q"] = (2.0 * torch.randn(M, c["hq"] * c["hd"], device="cuda", generator=g)).to(torch.bfloat16)
            s["out"] = torch.empty_like(s["q"])
        else:
            W = (c["hq"] + 2 * c["hkv"]) * c["hd"]
            s["qkv"] = torch.randn(M, W, device="cuda", generator=g).to(torch.bfloat16)
            inv = 500000.0 ** (-torch.arange(0, c["hd"], 2, device="cuda", dtype=torch.float64) / c["hd"])
            ang = torch.arange(max(ends) + 1, device="cuda", dtype=torch.float64)[:, None] * inv
            s["cos"], s["sin"] = ang.cos().float().contiguous(), ang.sin().float().contiguous()
            s["q_out"] = torch.empty(M, c["hq"] * c["hd"], device="cuda", dtype=torch.bfloat16)
            first = [n // c["P"] * c["P"] for n in lens]  # the first touched page's start
            s["first"], s["count"] = _ints(first), _ints([e - f for e, f in zip(ends, first)])
            L = max(1, max(_cdiv(e, c["P"]) * c["P"] - f for e, f in zip(ends, first)))
            dt = torch.float32 if c["read"] == "fp32" else torch.bfloat16
            s["k_out"] = torch.empty(c["B"], c["hkv"], L, c["hd"], device="cuda", dtype=dt)
            s["v_out"] = torch.empty_like(s["k_out"])
    elif op == "assign":
        lens = _spread(c["lo"], c["hi"], c["rows"])
        rows = c["rows"] * c["fork"]
        add = [1 + (i % 3 == 2) for i in range(rows)]
        need = sum(_cdiv(n, c["P"]) for n in lens)
        pages = need + 2 * rows + 5
        s["codes"], s["scales"] = _pool(c, c["layers"], pages, g)
        s["table"] = _table(lens, c["P"], pages, max(1, _cdiv(max(lens) + 2, c["P"])), g)
        parent = [i // c["fork"] for i in range(rows)]
        s["parent"], s["add"] = _ints(parent), _ints(add)
        s["keep"] = _ints([lens[p] for p in parent])
        s["table_out"] = torch.empty(rows, s["table"].shape[1], dtype=torch.int32, device="cuda")
        s["ref"] = torch.empty(pages, dtype=torch.int32, device="cuda")
        s["src"], s["dst"] = (torch.empty(rows, dtype=torch.int32, device="cuda") for _ in range(2))
        s["info"] = torch.empty(2, dtype=torch.int32, device="cuda")
    elif op == "compact":
        lens = _spread(c["lo"], c["hi"], c["rows"])
        need = sum(_cdiv(n, c["P"]) for n in lens)
        pages = max(need, int(need / c["live"])) + 1
        s["codes"], s["scales"] = _pool(c, c["layers"], pages, g)
        s["table"] = _table(lens, c["P"], pages, max(1, _cdiv(max(lens), c["P"])), g)
        s["lens"] = _ints(lens)
        s["table_out"] = torch.empty_like(s["table"])
        s["remap"], s["src"], s["dst"] = (torch.empty(pages, dtype=torch.int32, device="cuda") for _ in range(3))
        s["info"] = torch.empty(2, dtype=torch.int32, device="cuda")
    else:
        B, T, V = c["B"], c["T"], c["V"]
        logits = 2.5 * torch.randn(B, T + 1, V, device="cuda", generator=g)
        d_logits = logits[:, :T] + 0.7 * torch.randn(B, T, V, device="cuda", generator=g)
        s["target"] = torch.softmax(logits, -1)
        noise = -torch.log(-torch.log(torch.rand(B, T, V, device="cuda", generator=g).clamp_(1e-9, 1 - 1e-7)))
        s["drafts"] = (d_logits + noise).argmax(-1).to(torch.int32)  # tokens drawn from the draft's distribution
        s["draft"] = torch.softmax(d_logits, -1) if c["draft"] else None
        s["u"] = torch.rand(B, T + 1, device="cuda", generator=g)
        s["draft_lens"] = _ints(_news(c))
        s["accepted"] = torch.empty(B, dtype=torch.int32, device="cuda")
        s["tokens"] = torch.empty(B, T + 1, dtype=torch.int32, device="cuda")
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own and "codes" in s:
        from wal2026_b200 import kv8

        s["cache"] = kv8.PagedKV8Cache(s["codes"], s["scales"])
        if case["op"] == "attention":
            s["ws"] = kv8.kv8_attention_workspace(s["cache"], case["B"], case["hq"], case["T"])
    return s


def work(c):
    op = c["op"]
    if op in ("attention", "append"):
        lens, news = _lens(c), _news(c)
        row = 2 * c["hkv"] * c["hd"]
        new = sum(news)
        if op == "attention":
            seen = sum(a + b for a, b in zip(lens, news) if b)
            pages = sum(_cdiv(a + b, c["P"]) for a, b in zip(lens, news) if b)
            return {"bytes": seen * row + pages * (8 * c["hkv"] + 4) + 2 * 2 * c["B"] * c["T"] * c["hq"] * c["hd"],
                    "flops": 4 * c["hq"] * c["hd"] * sum(b * a + b * (b + 1) // 2 for a, b in zip(lens, news))}
        size = 4 if c["read"] == "fp32" else 2
        back = sum(a + b - a // c["P"] * c["P"] for a, b in zip(lens, news))
        L = max(1, max(_cdiv(a + b, c["P"]) * c["P"] - a // c["P"] * c["P"] for a, b in zip(lens, news)))
        return {"bytes": 2 * new * (2 * c["hq"] + 2 * c["hkv"]) * c["hd"] + new * row + back * row
                + c["B"] * L * row * size, "flops": 6 * new * (c["hq"] + c["hkv"]) * c["hd"]}
    if op in ("assign", "compact"):
        lens = _spread(c["lo"], c["hi"], c["rows"])
        page = c["layers"] * 2 * c["hkv"] * (c["P"] * c["hd"] + 4)
        if op == "assign":
            copies = sum(c["fork"] - 1 for n in lens if n % c["P"])
            entries = c["fork"] * sum(_cdiv(n, c["P"]) for n in lens)
            return {"bytes": 2 * copies * page + 8 * entries, "flops": entries}
        need = sum(_cdiv(n, c["P"]) for n in lens)
        pages = max(need, int(need / c["live"])) + 1
        return {"bytes": int(2 * need * (pages - need) / pages) * page + 8 * need + 4 * pages, "flops": pages}
    return {"bytes": c["B"] * (2 if c["draft"] else 1) * 4 * c["V"], "flops": 4 * c["B"] * c["V"]}


# ------------------------------------------------------------- plain forms

def _values(codes):
    return codes.float()


def _take(codes, pages):
    """codes[..., pages] along the page axis 0; 8-bit floats by their bytes."""
    return codes.view(torch.uint8)[pages].view(codes.dtype)


def _attention_plain(s):
    c = s["case"]
    B, T, hq, hkv, hd, P = (c[k] for k in ("B", "T", "hq", "hkv", "hd", "P"))
    G = hq // hkv
    lens, news = _lens(c), _news(c)
    out = torch.zeros(B, T, hkv, G, hd, device="cuda")
    q = s["q"].float().view(B, T, hkv, G, hd)
    for b in range(B):
        n = lens[b] + news[b]
        if not news[b]:
            continue
        pages = s["table"][b, :_cdiv(n, P)].long()
        kv = []
        for i in range(2):
            x = _values(_take(s["codes"][0, i], pages)) * s["scales"][0, i, pages][:, :, None, None]
            kv.append(x.transpose(0, 1).reshape(hkv, -1, hd)[:, :n])
        qb = q[b, :news[b]].permute(1, 0, 2, 3).reshape(hkv, -1, hd)  # rows t, g
        x = torch.matmul(qb, kv[0].transpose(1, 2)) * (hd ** -0.5)
        t = torch.arange(news[b], device="cuda").repeat_interleave(G)
        x = x.masked_fill(torch.arange(n, device="cuda")[None, :] > lens[b] + t[:, None], float("-inf"))
        x = torch.exp(x - x.amax(-1, keepdim=True))
        o = torch.matmul(x, kv[1]) / x.sum(-1, keepdim=True)
        out[b, :news[b]] = o.view(hkv, news[b], G, hd).transpose(0, 1)
    return out.view(B * T, hq * hd).to(torch.bfloat16)


def _rotate(x, cos, sin):
    half = x.shape[-1] // 2
    x1, x2 = x[..., :half], x[..., half:]
    return torch.cat([x1 * cos + (-x2) * sin, x2 * cos + x1 * sin], -1)


def _quant(x, kind):
    x = x.clamp(-QMAX[kind], QMAX[kind])
    return x.round() if kind == "int8" else x.to(torch.float8_e4m3fn).float()


def _append_plain(s):
    c = s["case"]
    B, T, hq, hkv, hd, P, kind = (c[k] for k in ("B", "T", "hq", "hkv", "hd", "P", "kind"))
    qkv = s["qkv"].float().view(B, T, hq + 2 * hkv, hd)
    t = torch.arange(T, device="cuda")
    pos = (s["lens"].long()[:, None] + t).clamp(max=s["cos"].shape[0] - 1)
    fresh = t[None, :] < s["news"][:, None]
    cos, sin = s["cos"][pos][:, :, None], s["sin"][pos][:, :, None]
    q = torch.where(fresh[:, :, None, None], _rotate(qkv[:, :, :hq], cos, sin), 0.0)
    new = torch.stack([_rotate(qkv[:, :, hq:hq + hkv], cos, sin), qkv[:, :, hq + hkv:]])  # k, v
    L = s["k_out"].shape[2]
    at = torch.arange(L, device="cuda")[None, :] + s["first"].long()[:, None]  # position of each place of the window
    old = at < s["lens"][:, None]
    mine = ~old & (at < (s["lens"] + s["news"])[:, None])
    live = (old | mine)[:, :, None, None]
    pages = s["table"].long().gather(1, (at // P).clamp(max=s["table"].shape[1] - 1)).clamp(min=0)
    out = []
    for i in range(2):
        x = torch.gather(new[i], 1, (at - s["lens"][:, None]).clamp(0, T - 1)[:, :, None, None].expand(-1, -1, hkv, hd))
        codes = _values(s["codes"][0, i].view(torch.uint8)[pages, :, at % P].view(s["codes"].dtype))  # [B, L, hkv, hd]
        nb = L // P
        a = torch.where(mine[:, :, None, None], x.abs(), 0.0).view(B, nb, P, hkv, hd).amax((2, 4)) / QMAX[kind]
        s0 = s["scales"][0, i][pages].view(B, nb, P, hkv)[:, :, 0]
        s0 = torch.where(old.view(B, nb, P)[:, :, :1], s0, 0.0)
        sc = torch.maximum(s0, a)
        ratio = torch.where(sc > s0, s0 / torch.where(sc > 0, sc, 1.0), 1.0)
        sc, ratio = (v.repeat_interleave(P, 1)[..., None] for v in (sc, ratio))
        was = torch.where(ratio < 1, _quant(codes * ratio, kind), codes)
        now = torch.where(sc > 0, _quant(x / torch.where(sc > 0, sc, 1.0), kind), 0.0)
        val = torch.where(live, torch.where(mine[:, :, None, None], now, was) * sc, 0.0)
        out.append(val.transpose(1, 2).to(s["k_out"].dtype).contiguous())
    return q.reshape(B * T, hq * hd).to(torch.bfloat16), out[0], out[1]


def _move(s, src, dst):
    ok = src >= 0
    a, b = src[ok].long(), dst[ok].long()
    raw = s["codes"].view(torch.uint8)
    raw[:, :, b] = raw[:, :, a]
    s["scales"][:, :, b] = s["scales"][:, :, a]


def _assign_plain(s):
    P = s["case"]["P"]
    pages, (rows, width) = s["ref"].shape[0], s["table_out"].shape
    keep, add = s["keep"].long(), s["add"].long()
    j = torch.arange(width, device="cuda")
    kept = j[None, :] < ((keep + P - 1) // P)[:, None]
    tab = torch.where(kept, s["table"].long()[s["parent"].long()], -1)
    ref = torch.bincount(tab[tab >= 0], minlength=pages)
    writes = (add > 0) & (keep % P != 0)
    last = tab.gather(1, (keep // P).clamp(max=width - 1)[:, None])[:, 0]
    wp = torch.where(writes, last, pages)  # page each row would write, `pages` where none
    nw = torch.bincount(wp, minlength=pages + 1)
    first = torch.full((pages + 1,), rows, device="cuda").scatter_reduce(0, wp, torch.arange(rows, device="cuda"), "amin")
    refx = torch.cat([ref, ref.new_zeros(1)])
    stays = (refx[wp] == 1) | ((refx[wp] == nw[wp]) & (first[wp] == torch.arange(rows, device="cuda")))
    cow = writes & ~stays
    have, want = (keep + P - 1) // P, (keep + add + P - 1) // P
    want = torch.where(add > 0, want, have)
    n = cow.long() + want - have
    begin = n.cumsum(0) - n
    free = (ref == 0).nonzero()[:, 0]
    src, dst = torch.where(cow, last, -1), torch.where(cow, free[begin.clamp(max=free.numel() - 1)], -1)
    fresh = (j[None, :] >= have[:, None]) & (j[None, :] < want[:, None])
    at = begin[:, None] + cow.long()[:, None] + j[None, :] - have[:, None]
    tab = torch.where(fresh, free[at.clamp(0, free.numel() - 1)], tab)
    tab = torch.where(cow[:, None] & (j[None, :] == (keep // P)[:, None]), dst[:, None], tab)
    ref = torch.bincount(tab[tab >= 0], minlength=pages)
    _move(s, src, dst)
    info = torch.stack([(ref == 0).sum(), ref.new_zeros(())])
    return [v.to(torch.int32) for v in (tab, ref, src, dst, info)] + [s["codes"], s["scales"]]


def _compact_plain(s):
    P, pages = s["case"]["P"], s["remap"].shape[0]
    width = s["table"].shape[1]
    kept = torch.arange(width, device="cuda")[None, :] < ((s["lens"].long() + P - 1) // P)[:, None]
    tab = torch.where(kept, s["table"].long(), -1)
    used = torch.bincount(tab[tab >= 0], minlength=pages) > 0
    live = used.sum()
    p = torch.arange(pages, device="cuda")
    movers, holes = (used & (p >= live)).nonzero()[:, 0], (~used & (p < live)).nonzero()[:, 0]
    remap = torch.where(used, p, -1)
    remap[movers] = holes
    src, dst = torch.full_like(p, -1), torch.full_like(p, -1)
    src[:movers.numel()], dst[:movers.numel()] = movers, holes
    tab = torch.where(tab >= 0, remap[tab.clamp(min=0)], -1)
    _move(s, src, dst)
    info = torch.stack([live, (src >= 0).sum()])
    return [v.to(torch.int32) for v in (tab, remap, src, dst, info)] + [s["codes"], s["scales"]]


def _fixed(p):
    return (torch.nan_to_num(p, nan=0.0).clamp(0.0, 1.0) * float(ONE)).round().long()


def _verify_plain(s):
    p, q, x = s["target"], s["draft"], s["drafts"].long()
    B, T = x.shape
    U = (s["u"] * float(1 << 24)).long()
    px = _fixed(p[:, :T].gather(2, x[:, :, None])[:, :, 0])
    qx = _fixed(q.gather(2, x[:, :, None])[:, :, 0]) if q is not None else torch.full_like(px, ONE)
    t = torch.arange(T, device="cuda")
    ok = (U[:, :T] * qx < px * (1 << 24)) & (t[None, :] < s["draft_lens"][:, None])
    a = ok.long().cumprod(1).sum(1)
    b = torch.arange(B, device="cuda")
    w = _fixed(p[b, a])
    first = w
    rejected = a < s["draft_lens"]
    at = a.clamp(max=T - 1)
    if q is not None:
        w = torch.where(rejected[:, None], (w - _fixed(q[b, at])).clamp(min=0), w)
    else:
        w = w.scatter(1, x[b, at][:, None], torch.where(rejected, 0, w[b, x[b, at]])[:, None])
    w = torch.where(w.sum(1, keepdim=True) > 0, w, first)
    run_sum = w.cumsum(1)
    W = run_sum[:, -1]
    R = ((W >> 32) * U[:, T] << 8) + ((W & 0xFFFFFFFF) * U[:, T] >> 24)
    token = torch.where(W > 0, (run_sum <= R[:, None]).sum(1), -1)
    out = torch.where(t[None, :] < a[:, None], x, -1)
    out = torch.cat([out, torch.full_like(a, -1)[:, None]], 1).scatter(1, a[:, None], token[:, None])
    return a.to(torch.int32), out.to(torch.int32)


# -------------------------------------------------------------- one pass

def run(s):
    c = s["case"]
    op = c["op"]
    if not own:
        return {"attention": _attention_plain, "append": _append_plain, "assign": _assign_plain,
                "compact": _compact_plain, "verify": _verify_plain}[op](s)
    from wal2026_b200 import kv8, speculative

    if op == "attention":
        kv8.kv8_attention(s["cache"], 0, s["q"], s["table"], s["lens"], s["out"], s["ws"], new_lens=s["news"])
        return s["out"]
    if op == "append":
        kv8.kv8_append(s["cache"], 0, s["qkv"], c["hq"], s["table"], s["lens"], s["q_out"], cos=s["cos"], sin=s["sin"],
                       new_lens=s["news"])
        kv8.kv8_read(s["cache"], 0, s["table"], s["first"], s["count"], s["k_out"], s["v_out"])
        return s["q_out"], s["k_out"], s["v_out"]
    if op == "assign":
        kv8.kv_pages_assign(s["table"], s["parent"], s["keep"], s["add"], c["P"], s["table_out"], s["ref"], s["src"],
                            s["dst"], s["info"])
        kv8.kv_pages_copy(s["cache"], s["src"], s["dst"])
        return [s["table_out"], s["ref"], s["src"], s["dst"], s["info"], s["codes"], s["scales"]]
    if op == "compact":
        kv8.kv_pages_compact(s["table"], s["lens"], c["P"], s["table_out"], s["remap"], s["src"], s["dst"], s["info"])
        kv8.kv_pages_copy(s["cache"], s["src"], s["dst"])
        return [s["table_out"], s["remap"], s["src"], s["dst"], s["info"], s["codes"], s["scales"]]
    speculative.verify_drafts(s["target"], s["draft"], s["drafts"], s["u"], s["accepted"], s["tokens"],
                              draft_lens=s["draft_lens"])
    return s["accepted"], s["tokens"]


# ------------------------------------------------- definitions in 64 bits

def _exact_attention(c, s):
    B, T, G = c["B"], c["T"], c["hq"] // c["hkv"]
    lens, news, table = _lens(c), _news(c), s["table"].tolist()
    q = s["q"].double().view(B, T, c["hkv"], G, c["hd"])
    out = torch.zeros_like(q)
    for b in range(B):
        n = lens[b] + news[b]
        ids = torch.tensor(table[b][:_cdiv(n, c["P"])], device="cuda")
        for h in range(c["hkv"]):
            k, v = ((s["codes"][0, i, :, h].view(torch.uint8)[ids].view(s["codes"].dtype).float().double()
                     * s["scales"][0, i, :, h].double()[ids][:, None, None]).flatten(0, 1) for i in range(2))
            for t in range(news[b]):
                m = lens[b] + t + 1
                w = torch.softmax(q[b, t, h] @ k[:m].T / math.sqrt(c["hd"]), -1)
                out[b, t, h] = w @ v[:m]
    return out.view(B * T, -1)


def _exact_append(c, s):
    """Block by block."""
    hq, hkv, hd, P, T = c["hq"], c["hkv"], c["hd"], c["P"], c["T"]
    lens, news, table = _lens(c), _news(c), s["table"].tolist()
    x = s["qkv"].double().view(c["B"], T, -1, hd)
    half = hd // 2
    q = torch.zeros(c["B"], T, hq, hd, dtype=torch.float64, device="cuda")
    outs = [torch.zeros(s["k_out"].shape, dtype=torch.float64, device="cuda") for _ in range(2)]

    def code(v):
        v = v.clamp(-QMAX[c["kind"]], QMAX[c["kind"]])
        if c["kind"] == "int8":
            return v.round()
        e = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))).clamp(min=-6)  # spacing 2^(e-3), subnormal below 2^-6
        return torch.round(v * torch.exp2(3 - e)) * torch.exp2(e - 3)

    for b in range(c["B"]):
        if not news[b]:
            if lens[b] % P:
                page = table[b][lens[b] // P]
                for i in range(2):
                    outs[i][b, :, :lens[b] % P] = (s["codes"][0, i, page].float().double() * s["scales"][0, i, page].double()[:, None, None])[:, :lens[b] % P]
            continue
        co, si = (s[k][lens[b]:lens[b] + news[b]].double()[:, None] for k in ("cos", "sin"))

        def turn(y):
            return torch.cat((y[..., :half] * co - y[..., half:] * si, y[..., half:] * co + y[..., :half] * si), -1)

        y = x[b, :news[b]]
        q[b, :news[b]] = turn(y[:, :hq])
        for i, new in enumerate((turn(y[:, hq:hq + hkv]), y[:, hq + hkv:])):
            for j in range(lens[b] // P, _cdiv(lens[b] + news[b], P)):
                lo, hi = max(lens[b], j * P), min(lens[b] + news[b], (j + 1) * P)
                had = lo - j * P
                z = new[lo - lens[b]:hi - lens[b]].transpose(0, 1)  # [hkv, tokens, hd]
                page = table[b][j]
                old = s["scales"][0, i, page].double() if had else torch.zeros(hkv, dtype=torch.float64, device="cuda")
                sc = torch.maximum(old, z.abs().amax((1, 2)) / QMAX[c["kind"]])[:, None, None]
                before = s["codes"][0, i, page, :, :had].float().double()
                r = old[:, None, None] / sc
                before = torch.where(r < 1, code(before * r), before)
                o = j * P - lens[b] // P * P
                outs[i][b, :, o:o + had] = before * sc
                outs[i][b, :, o + had:o + hi - j * P] = code(z / sc) * sc
    return q.view(c["B"] * T, -1), outs[0], outs[1]


def _exact_assign(c, s):
    P, pages = c["P"], s["ref"].shape[0]
    table, parent, keep, add = (s[k].tolist() for k in ("table", "parent", "keep", "add"))
    rows = [table[p][:_cdiv(k, P)] for p, k in zip(parent, keep)]
    users = {}
    for r, row in enumerate(rows):
        for j, page in enumerate(row):
            users.setdefault(page, []).append((r, add[r] > 0 and keep[r] % P != 0 and j == len(row) - 1))
    free = iter([p for p in range(pages) if p not in users])
    src, dst = [-1] * len(rows), [-1] * len(rows)
    out = [list(row) for row in rows]
    for r, row in enumerate(out):
        if add[r] > 0 and keep[r] % P:
            mine = users[row[-1]]
            if len(mine) > 1 and not (all(w for _, w in mine) and mine[0][0] == r):
                src[r], dst[r] = row[-1], next(free)
                row[-1] = dst[r]
        while len(row) * P < keep[r] + add[r]:
            row.append(next(free))
    ref = [0] * pages
    for row in out:
        for page in row:
            ref[page] += 1
    width = s["table_out"].shape[1]
    out = [row + [-1] * (width - len(row)) for row in out]
    return [torch.tensor(v, dtype=torch.int32) for v in (out, ref, src, dst, [ref.count(0), 0])] + [None, None]


def _exact_compact(c, s):
    P, pages = c["P"], s["remap"].shape[0]
    table, lens = s["table"].tolist(), s["lens"].tolist()
    used = sorted({p for row, n in zip(table, lens) for p in row[:_cdiv(n, P)]})
    live = len(used)
    there = set(used)
    holes = [p for p in range(live) if p not in there]
    moves = list(zip([p for p in used if p >= live], holes))
    new = {p: p for p in used} | dict(moves)
    out = [[new[p] if j < _cdiv(n, P) else -1 for j, p in enumerate(row)] for row, n in zip(table, lens)]
    pad = [-1] * (pages - len(moves))
    cols = (out, [new.get(p, -1) for p in range(pages)], [m[0] for m in moves] + pad, [m[1] for m in moves] + pad, [live, len(moves)])
    return [torch.tensor(v, dtype=torch.int32) for v in cols] + [None, None]


def _exact_verify(c, s):
    B, T = c["B"], c["T"]
    accepted, tokens = [], []
    x, lens = s["drafts"].tolist(), s["draft_lens"].tolist()
    u = (s["u"].double() * (1 << 24)).floor().long().tolist()

    def units(p):
        return (p.double().clamp(0, 1) * ONE).round().long().cpu()

    for b in range(B):
        a = 0
        while a < lens[b]:
            qx = int(units(s["draft"][b, a, x[b][a]])) if s["draft"] is not None else ONE
            if u[b][a] * qx >= int(units(s["target"][b, a, x[b][a]])) << 24:
                break
            a += 1
        w = units(s["target"][b, a])
        if a < lens[b]:
            r = w.clone()
            if s["draft"] is not None:
                r = (r - units(s["draft"][b, a])).clamp(min=0)
            else:
                r[x[b][a]] = 0
            w = r if int(r.sum()) else w
        total = int(w.sum())
        place = int(torch.searchsorted(w.cumsum(0), (total * u[b][T]) >> 24, right=True)) if total else -1
        accepted.append(a)
        tokens.append(x[b][:a] + [place] + [-1] * (T - a))
    return torch.tensor(accepted, dtype=torch.int32), torch.tensor(tokens, dtype=torch.int32)


def exact(case, seed):
    s = _inputs(case, seed)
    return {"attention": _exact_attention, "append": _exact_append, "assign": _exact_assign, "compact": _exact_compact,
            "verify": _exact_verify}[case["op"]](case, s)
