"""Cases of shared-prefix attention, logit rules and 4-bit linears, for timing and for comparing outputs.

Four operators of a decoding step that takes several samples of long prompts,
each in a plain form (elementary torch operations in 32 bits) and as the call a
user makes of this package:

  groups     which rows of a page table share their first pages, and how far
  shared     grouped-query attention over the paged 8-bit cache, what a group
             of rows shares read once for all of them
  rules      penalties for repeated tokens, biases, grammar masks and the
             temperature on logits, and their softmax
  int4       y = x W^T with 4-bit weights and a scale (and a zero point) per group

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
FLOAT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------ cases

def listed():
    return [
        # four samples of one prompt at the 2048-token context of the decode benchmark, Llama-3-8B heads: latency
        dict(name="shared samples", op="shared", prompts=1, fork=4, alone=0, T=1, hq=32, hkv=8, hd=128, P=64, kind="int8", lo=2000, hi=2000, tail=200, least=256),
        # eight prompts with eight samples each and a few requests of their own, small pages, the 70B heads
        dict(name="shared prompts", op="shared", prompts=8, fork=8, alone=5, T=1, hq=64, hkv=8, hd=128, P=16, kind="e4m3", lo=1000, hi=4096, tail=600, least=256),
        # a speculative step of sixteen samples: up to four drafts and the token before them
        dict(name="shared drafts", op="shared", prompts=1, fork=16, alone=0, T=5, hq=32, hkv=8, hd=128, P=32, kind="int8", lo=8200, hi=8200, tail=300, least=512),
        # many questions about one long document
        dict(name="shared document", op="shared", prompts=1, fork=64, alone=0, T=1, hq=64, hkv=8, hd=128, P=64, kind="int8", lo=65700, hi=65700, tail=900, least=1024),
        # the groups of a small batch
        dict(name="groups small", op="groups", prompts=2, fork=3, alone=2, P=64, lo=500, hi=2000, tail=100, least=256),
        # 32 prompts of the 70B benchmark context, eight samples each, small pages
        dict(name="groups batch", op="groups", prompts=32, fork=8, alone=40, P=16, lo=300, hi=8100, tail=600, least=128),
        # one sequence, the stacks' vocabulary: every penalty, no mask
        dict(name="rules single", op="rules", B=1, T=1, V=128256, text=2048, bias=40, mask=False, penalties=True, dtype="bf16"),
        # a grammar: masks and biases of a speculative step, no penalties
        dict(name="rules grammar", op="rules", B=16, T=5, V=128256, text=300, bias=300, mask=True, penalties=False, dtype="fp32"),
        # a batch with up to eight drafts, all rules at once
        dict(name="rules batch", op="rules", B=64, T=9, V=128256, text=4096, bias=16, mask=True, penalties=True, dtype="bf16"),
        # an attention output projection of the 8B stack for one token: latency
        dict(name="int4 o", op="int4", M=1, N=4096, K=4096, group=128, zeros=False, x="bf16", y="bf16"),
        # a down projection for a batch, zero points, partial sums in fp32 as row-parallel layers leave them
        dict(name="int4 down", op="int4", M=16, N=4096, K=14336, group=64, zeros=True, x="bf16", y="fp32"),
        # the vocabulary projection of the 8B stack for a speculative step
        dict(name="int4 head", op="int4", M=5, N=128256, K=4096, group=128, zeros=False, x="bf16", y="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["shared", "shared", "groups", "rules", "rules", "int4", "int4"])
    kind, P, hd = rng.choice(["int8", "e4m3"]), rng.choice([16, 32, 64]), rng.choice([64, 128])
    if op == "shared":
        hq, hkv = rng.choice([(32, 8), (64, 8), (8, 1), (8, 8), (12, 4), (14, 2)])
        hi = _log(rng, 64, 65700)
        T = rng.choice([1, 1, 2, 3, 5])
        rows = max(1, min(_log(rng, 1, 64), 64 * 64 * 65700 // (4 * hi * hq * T)))
        fork = max(1, min(_log(rng, 1, 64), rows))
        return dict(op=op, prompts=max(1, rows // fork), fork=fork, alone=rng.choice([0, 0, 1, 3]), T=T, hq=hq, hkv=hkv,
                    hd=hd, P=P, kind=kind, lo=rng.choice([1, hi // 2 + 1, hi]), hi=hi, tail=_log(rng, 1, 900),
                    least=rng.choice([64, 128, 256, 1024]))
    if op == "groups":
        hi = _log(rng, 320, 8100)
        return dict(op=op, prompts=_log(rng, 2, 32), fork=rng.choice([2, 3, 8]), alone=rng.choice([3, 17, 40]), P=P,
                    lo=rng.choice([1, hi // 2, hi]), hi=hi, tail=_log(rng, 1, 600), least=rng.choice([32, 100, 128, 256]))
    if op == "rules":
        return dict(op=op, B=_log(rng, 1, 64), T=rng.choice([1, 1, 2, 5, 9]), V=_log(rng, 1000, 128255) | 1,
                    text=_log(rng, 1, 4096), bias=rng.choice([0, 1, 7, 300]), mask=rng.random() < 0.5,
                    penalties=rng.random() < 0.7, dtype=rng.choice(["bf16", "fp16", "fp32"]))
    group = rng.choice([32, 64, 128])
    N = _log(rng, 40, 128256)
    K = max(1, min(14336, 4096 * 128256 // N, _log(rng, 128, 14336)) // group) * group
    return dict(op=op, M=rng.choice([1, 1, 2, 3, 5, 8, 13, 16, 24, 32, 50]), N=N, K=K, group=group, zeros=rng.random() < 0.5,
                x=rng.choice(["bf16", "fp16"]), y=rng.choice(["bf16", "fp16", "fp32"]))


def _cdiv(a, b):
    return -(-a // b)


def _spread(lo, hi, n):
    """n lengths over [lo, hi], the longest first."""
    out = [lo + int((hi - lo) * ((0.6180339887498949 * (i + 1)) % 1.0)) for i in range(n)]
    out[0] = hi
    return out


def _rows(c):
    """(prompt or -1, prompt length, length) of each row: a group's rows are not neighbours, as requests come and go."""
    lens = _spread(c["lo"], c["hi"], c["prompts"])
    rows = [(p, lens[p]) for _ in range(c["fork"]) for p in range(c["prompts"])]
    own_len = _spread(c["lo"], c["hi"], max(1, c["alone"]))
    for i in range(c["alone"]):
        rows.insert((3 * i + 1) % (len(rows) + 1), (-1, own_len[i]))
    return [(p, n, n + int(c["tail"] * ((0.7548776662466927 * i) % 1.0))) for i, (p, n) in enumerate(rows)]


def _news(c):
    """New tokens of each row: up to T, an idle row among eight or more."""
    rows = len(_rows(c))
    out = [c["T"] - int(0.6 * c["T"] * ((0.5698402909980532 * i) % 1.0)) for i in range(rows)]
    if rows >= 8:
        out[rows - 2] = 0
    return out


def _groups(c):
    """(members, shared positions) of each group, from how the rows were made."""
    by = {}
    for b, (p, n, length) in enumerate(_rows(c)):
        if p >= 0 and n // c["P"] * c["P"] >= c["least"]:
            by.setdefault(p, []).append((b, n))
    out = []
    for p, members in by.items():
        shared = members[0][1] // c["P"] * c["P"] // 32 * 32
        if len(members) > 1 and shared >= c["least"]:
            out.append(([b for b, _ in members], shared))
    return sorted(out)


# ----------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _pool(c, pages, g):
    """Codes and scales of a filled pool: values around one, larger in some pages."""
    shape = (1, 2, pages, c["hkv"], c["P"], c["hd"])
    codes = torch.empty(shape, dtype=CODE[c["kind"]], device="cuda")
    for kv in range(2):
        x = torch.randn(shape[2:], device="cuda", generator=g) * (QMAX[c["kind"]] / 4.0)
        x = x.clamp_(-QMAX[c["kind"]], QMAX[c["kind"]])
        codes[0, kv] = x.round_().to(torch.int8) if c["kind"] == "int8" else x.to(CODE["e4m3"])
    scales = (4.0 / QMAX[c["kind"]]) * torch.exp(0.3 * torch.randn(shape[:4], device="cuda", generator=g))
    return codes, scales.float().contiguous()


def _pages(c, extra):
    """Pages of every row as numbers 0 .. n - 1, and n: a prompt's whole pages are common, the rest is the row's own."""
    first, n, out = {}, 0, []
    for p, prompt, length in _rows(c):
        common = prompt // c["P"] if p >= 0 else 0
        if common and p not in first:
            first[p] = list(range(n, n + common))
            n += common
        mine = _cdiv(length + extra, c["P"]) - common
        out.append((first[p] if common else []) + list(range(n, n + mine)))
        n += mine
    return out, n


def _table(c, extra, spare, seed):
    """int32 [rows, width] on the GPU with the pages in random order, -1 past each row's; and how many pages there are."""
    rows, n = _pages(c, extra)
    width = max(len(r) for r in rows)
    flat = torch.tensor([r + [-1] * (width - len(r)) for r in rows], device="cuda")
    order = torch.randperm(n + spare, device="cuda", generator=_gen(seed + 77))
    return torch.where(flat >= 0, order[flat.clamp(min=0)], flat).to(torch.int32).contiguous(), n + spare


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _inputs(c, seed):
    g = _gen(seed)
    op, s = c["op"], {}
    if op in ("shared", "groups"):
        lens = [r[2] for r in _rows(c)]
        s["table"], pages = _table(c, c.get("T", 1), 3, seed)
        s["lens"] = _ints(lens)
        if op == "groups":  # rows in the order of their requests
            order = torch.randperm(len(lens), device="cuda", generator=g)
            s["table"], s["lens"] = s["table"][order].contiguous(), s["lens"][order].contiguous()
        s["groups"] = torch.empty(4, len(lens), dtype=torch.int32, device="cuda")
        if op == "shared":
            s["codes"], s["scales"] = _pool(c, pages, g)
            s["news"] = _ints(_news(c))
            s["q"] = (2.0 * torch.randn(len(lens) * c["T"], c["hq"] * c["hd"], device="cuda", generator=g)).to(torch.bfloat16)
            s["out"] = torch.empty_like(s["q"])
    elif op == "rules":
        B, T, V = c["B"], c["T"], c["V"]
        s["logits"] = (3.0 * torch.randn(B, T, V, device="cuda", generator=g)).to(FLOAT[c["dtype"]])
        s["out"] = torch.empty(B, T, V, device="cuda")
        # a text repeats itself: tokens of a few topics, frequent ones more often
        u = torch.rand(B, c["text"] + T, device="cuda", generator=g)
        s["text"] = (V * u ** 4).long().clamp(max=V - 1).to(torch.int32).contiguous()
        lens = _spread(c["text"] // 3, c["text"], B)
        s["lens"], s["prompts"] = _ints(lens), _ints([n // 2 for n in lens])
        s["temperature"] = 0.6 + 0.6 * torch.rand(B, device="cuda", generator=g)
        s["repetition"] = s["presence"] = s["frequency"] = s["bias_ids"] = s["bias"] = s["mask"] = None
        if c["penalties"]:
            s["repetition"] = 1.0 + 0.3 * torch.rand(B, device="cuda", generator=g)
            s["presence"] = 0.5 * torch.rand(B, device="cuda", generator=g)
            s["frequency"] = 0.2 * torch.rand(B, device="cuda", generator=g)
        if c["bias"]:
            ids = torch.stack([torch.randperm(V, device="cuda", generator=g)[:c["bias"]] for _ in range(B)])
            s["bias_ids"] = ids.to(torch.int32).contiguous()
            s["bias"] = 4.0 * torch.randn(B, c["bias"], device="cuda", generator=g)
        if c["mask"]:
            # a grammar allows a sixteenth of the tokens: words of 32 tokens, bit i of word w is token 32 w + i
            words = torch.randint(-2 ** 31, 2 ** 31, (4, B, T, _cdiv(V, 32)), device="cuda", generator=g)
            s["mask"] = (words[0] & words[1] & words[2] & words[3]).to(torch.int32)
    else:
        M, N, K, group = c["M"], c["N"], c["K"], c["group"]
        s["codes"] = torch.randint(0, 16, (N, K), device="cuda", generator=g, dtype=torch.uint8)
        s["scales"] = (0.004 * torch.exp(0.3 * torch.randn(N, K // group, device="cuda", generator=g))).to(torch.float16)
        s["zeros"] = torch.randint(4, 12, (N, K // group), device="cuda", generator=g, dtype=torch.uint8) if c["zeros"] else None
        s["x"] = torch.randn(M, K, device="cuda", generator=g).to(FLOAT[c["x"]])
        s["y"] = torch.empty(M, N, dtype=FLOAT[c["y"]], device="cuda")
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own and case["op"] == "shared":
        from wal2026_b200 import kv8

        s["cache"] = kv8.PagedKV8Cache(s["codes"], s["scales"])
        s["ws"] = kv8.kv8_attention_shared_workspace(s["cache"], s["table"].shape[0], case["hq"], case["T"])
        kv8.kv_pages_groups(s["table"], s["lens"], case["P"], s["groups"], least=case["least"])  # once for all layers of a step
    if own and case["op"] == "int4":
        from wal2026_b200.int4 import Int4Linear

        s["layer"] = Int4Linear(s["codes"], s["scales"], s["zeros"])
        s["codes"] = s["scales"] = s["zeros"] = None
    return s


def work(c):
    op = c["op"]
    if op == "rules":
        n = c["B"] * c["T"] * c["V"]
        text = 4 * sum(_spread(c["text"] // 3, c["text"], c["B"])) if c["penalties"] else 0
        size = 4 if c["dtype"] == "fp32" else 2
        return {"bytes": n * (size + 4) + (n // 8 if c["mask"] else 0) + 8 * c["B"] * c["bias"] + text, "flops": 4 * n}
    if op == "int4":
        M, N, K, groups = c["M"], c["N"], c["K"], c["K"] // c["group"]
        return {"bytes": N * K // 2 + N * groups * (3 if c["zeros"] else 2) + 2 * M * K + M * N * (4 if c["y"] == "fp32" else 2),
                "flops": 2 * M * N * K}
    rows, groups = _rows(c), _groups(c)
    if op == "groups":
        # every grouped row's common pages and the page that decides, and the lengths
        entries = sum(len(m) * (s // c["P"]) for m, s in groups) + len(rows)
        return {"bytes": 4 * entries + 4 * len(rows) + 16 * len(rows), "flops": entries}
    news = _news(c)
    row = 2 * c["hkv"] * c["hd"]
    shared = {b: s for members, s in groups for b in members}
    seen = sum(s for members, s in groups if any(news[b] for b in members))
    seen += sum(r[2] + n - shared.get(b, 0) for b, (r, n) in enumerate(zip(rows, news)) if n)
    return {"bytes": seen * row + _cdiv(seen, c["P"]) * (8 * c["hkv"] + 4) + 4 * len(rows) * c["T"] * c["hq"] * c["hd"],
            "flops": 4 * c["hq"] * c["hd"] * sum(n * r[2] + n * (n + 1) // 2 for r, n in zip(rows, news))}


# ------------------------------------------------------------- plain forms

def _values(s, pages):
    """K and V of pages, fp32 [hkv, positions, hd] each."""
    out = []
    for i in range(2):
        codes = s["codes"][0, i].view(torch.uint8)[pages].view(s["codes"].dtype).float()
        x = codes * s["scales"][0, i, pages][:, :, None, None]
        out.append(x.transpose(0, 1).reshape(x.shape[1], -1, x.shape[3]))
    return out


def _part(q, k, v, seen):
    """(maximum, sum, weighted sum) of rows q [hkv, rows, hd] over positions; seen [rows, positions] or None."""
    x = torch.matmul(q, k.transpose(1, 2)) * (q.shape[-1] ** -0.5)
    if seen is not None:
        x = x.masked_fill(~seen, float("-inf"))
    m = x.amax(-1, keepdim=True)
    x = torch.exp(x - m)
    return m, x.sum(-1, keepdim=True), torch.matmul(x, v)


def _shared_plain(s):
    c = s["case"]
    T, hq, hkv, hd, P = (c[k] for k in ("T", "hq", "hkv", "hd", "P"))
    G = hq // hkv
    rows, news = _rows(c), _news(c)
    B = len(rows)
    q = s["q"].float().view(B, T, hkv, G, hd)
    first, start = {}, {}
    for members, n in _groups(c):
        k, v = _values(s, s["table"][members[0], :_cdiv(n, P)].long())
        x = q[torch.tensor(members, device="cuda")].permute(2, 0, 1, 3, 4).reshape(hkv, -1, hd)  # rows member, t, g
        parts = _part(x, k[:, :n], v[:, :n], None)
        for i, b in enumerate(members):
            first[b] = [y.view(hkv, len(members), T * G, -1)[:, i] for y in parts]
            start[b] = n
    out = torch.zeros(B, T, hkv, G, hd, device="cuda")
    for b in range(B):
        if not news[b]:
            continue
        n0, n = start.get(b, 0), rows[b][2] + news[b]
        k, v = _values(s, s["table"][b, n0 // P:_cdiv(n, P)].long())
        lead = n0 % P
        k, v = k[:, lead:lead + n - n0], v[:, lead:lead + n - n0]
        t = torch.arange(T, device="cuda").repeat_interleave(G)
        seen = torch.arange(n0, n, device="cuda")[None, :] <= rows[b][2] + t[:, None]
        m, l, o = _part(q[b].permute(1, 0, 2, 3).reshape(hkv, T * G, hd), k, v, seen)
        if b in first:
            m1, l1, o1 = first[b]
            top = torch.maximum(m, m1)
            a, a1 = torch.exp(m - top), torch.exp(m1 - top)
            l, o = l * a + l1 * a1, o * a + o1 * a1
        out[b, :news[b]] = (o / l).view(hkv, T, G, hd).transpose(0, 1)[:news[b]]
    return out.view(B * T, hq * hd).to(torch.bfloat16)


def _groups_plain(s):
    c, table, lens = s["case"], s["table"].long(), s["lens"].long()
    B, width = table.shape
    P, least = c["P"], c["least"]
    full = torch.minimum(lens.clamp(min=0), torch.full_like(lens, width * P - 1)) // P
    at = _cdiv(least, P) - 1
    key = table[:, at] if at < width else torch.full_like(lens, -1)
    b = torch.arange(B, device="cuda")
    able = (full * P // 32 * 32 >= least) & (key >= 0)
    same = able[:, None] & able[None, :] & (key[:, None] == key[None, :])
    leader = torch.where(able, torch.where(same, b[None, :], B).amin(1), b)
    equal = (table == table[leader]) & (torch.arange(width, device="cuda")[None, :] < torch.minimum(full, full[leader])[:, None])
    common = equal.long().cumprod(1).sum(1)
    least_common = torch.full_like(common, width).scatter_reduce(0, leader, common, "amin")
    size = torch.bincount(leader, minlength=B)
    shared = least_common[leader] * P // 32 * 32
    grouped = able & (size[leader] > 1) & (shared >= least)
    shared = torch.where(grouped, shared, 0)
    order = torch.sort(torch.where(grouped, leader * B + b, B * B + b)).indices
    count = grouped.sum()
    order = torch.where(b < count, order, -1)
    heads = torch.where(grouped & (leader == b), size, 0)  # by lowest member
    rank = torch.sort(torch.where(heads > 0, b, B + b)).indices
    sizes = heads[rank]
    begin = torch.where(sizes > 0, sizes.cumsum(0) - sizes, 0)
    return torch.stack([order, begin, sizes, shared]).to(torch.int32)


def _rules_plain(s):
    c = s["case"]
    B, T, V = c["B"], c["T"], c["V"]
    x = s["logits"].float()
    if c["penalties"]:
        # text up to and with the row's own token; the first prompt tokens count as seen only
        j = torch.arange(s["text"].shape[1], device="cuda")
        upto = s["lens"].long()[:, None] + torch.arange(T, device="cuda")  # [B, T]
        gen = torch.zeros(B, T, V, device="cuda")
        old = torch.zeros(B, V, device="cuda")
        prompt = j[None, :] < s["prompts"][:, None]
        old.scatter_add_(1, s["text"].long(), prompt.float())
        for t in range(T):
            w = (~prompt & (j[None, :] <= upto[:, t, None])).float()
            gen[:, t].scatter_add_(1, s["text"].long(), w)
        seen = (gen > 0) | (old > 0)[:, None]
        r = s["repetition"][:, None, None]
        x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
        x = x - s["frequency"][:, None, None] * gen
        x = x - s["presence"][:, None, None] * (gen > 0)
    if c["bias"]:
        x = x.scatter_add(2, s["bias_ids"].long()[:, None].expand(B, T, -1), s["bias"][:, None].expand(B, T, -1))
    if c["mask"]:
        bit = torch.arange(32, device="cuda")
        allowed = ((s["mask"][..., None] >> bit) & 1).view(B, T, -1)[..., :V]
        x = x.masked_fill(allowed == 0, float("-inf"))
    x = x / s["temperature"][:, None, None]
    x = torch.exp(x - x.amax(-1, keepdim=True))
    return x / x.sum(-1, keepdim=True)


def _int4_plain(s):
    c = s["case"]
    N, K, group = c["N"], c["K"], c["group"]
    out = []
    for i in range(0, N, 16384):
        q = s["codes"][i:i + 16384].view(-1, K // group, group).float()
        z = s["zeros"][i:i + 16384].float()[..., None] if s["zeros"] is not None else 8.0
        w = (q - z) * s["scales"][i:i + 16384].float()[..., None]
        out.append(torch.matmul(s["x"].float(), w.view(-1, K).t()))
    return torch.cat(out, 1).to(s["y"].dtype)


# -------------------------------------------------------------- one pass

def run(s):
    c = s["case"]
    op = c["op"]
    if not own:
        return {"shared": _shared_plain, "groups": _groups_plain, "rules": _rules_plain, "int4": _int4_plain}[op](s)
    if op == "shared":
        from wal2026_b200 import kv8

        kv8.kv8_attention_shared(s["cache"], 0, s["q"], s["table"], s["lens"], s["groups"], s["out"], s["ws"],
                                 new_lens=s["news"])
        return s["out"]
    if op == "groups":
        from wal2026_b200 import kv8

        kv8.kv_pages_groups(s["table"], s["lens"], c["P"], s["groups"], least=c["least"])
        return s["groups"]
    if op == "rules":
        from wal2026_b200 import logits

        logits.logit_rules(s["logits"], s["out"], text=s["text"], lens=s["lens"], prompt_lens=s["prompts"],
                           repetition=s["repetition"], presence=s["presence"], frequency=s["frequency"],
                           bias_ids=s["bias_ids"], bias=s["bias"], mask=s["mask"], temperature=s["temperature"])
        return s["out"]
    s["layer"].gemv_into(s["x"], s["y"])
    return s["y"]


# ------------------------------------------------- definitions in 64 bits

def _exact_shared(c, s):
    """Row by row over all of its positions, as if nothing were shared."""
    rows, news, table = _rows(c), _news(c), s["table"].tolist()
    T, G, hkv, hd, P = c["T"], c["hq"] // c["hkv"], c["hkv"], c["hd"], c["P"]
    q = s["q"].double().view(len(rows), T, hkv, G, hd)
    out = torch.zeros_like(q)
    for b, (_, _, length) in enumerate(rows):
        if not news[b]:
            continue
        ids = torch.tensor(table[b][:_cdiv(length + news[b], P)], device="cuda")
        for h in range(hkv):
            k, v = ((s["codes"][0, i, :, h].view(torch.uint8)[ids].view(s["codes"].dtype).float().double()
                     * s["scales"][0, i, :, h].double()[ids][:, None, None]).flatten(0, 1) for i in range(2))
            for t in range(news[b]):
                m = length + t + 1
                out[b, t, h] = torch.softmax(q[b, t, h] @ k[:m].T / math.sqrt(hd), -1) @ v[:m]
    return out.view(len(rows) * T, -1)


def _exact_groups(c, s):
    table, lens = s["table"].tolist(), s["lens"].tolist()
    B, width, P, least = len(lens), len(table[0]), c["P"], c["least"]
    at = _cdiv(least, P) - 1
    by = {}
    for b in range(B):
        full = min(max(lens[b], 0), width * P - 1) // P
        if full * P // 32 * 32 >= least and table[b][at] >= 0:
            by.setdefault(table[b][at], []).append((b, full))
    order, begin, sizes, shared = [], [], [], [0] * B
    for members in sorted(by.values()):
        b0, n = members[0]
        for b, full in members:
            k = 0
            while k < min(full, n) and table[b][k] == table[b0][k]:
                k += 1
            n = k
        positions = n * P // 32 * 32
        if len(members) < 2 or positions < least:
            continue
        begin.append(len(order))
        sizes.append(len(members))
        for b, _ in members:
            order.append(b)
            shared[b] = positions
    fill = B - len(sizes)
    return torch.tensor([order + [-1] * (B - len(order)), begin + [0] * fill, sizes + [0] * fill, shared], dtype=torch.int32)


def _exact_rules(c, s):
    """A row at a time; counts by counting."""
    B, T, V = c["B"], c["T"], c["V"]
    out = torch.empty(B, T, V, dtype=torch.float64, device="cuda")
    text, lens, prompts = s["text"].tolist(), s["lens"].tolist(), s["prompts"].tolist()
    for b in range(B):
        for t in range(T):
            x = s["logits"][b, t].double()
            if c["penalties"]:
                upto = lens[b] + t + 1
                before = torch.bincount(torch.tensor(text[b][:upto], device="cuda"), minlength=V)
                made = torch.bincount(torch.tensor(text[b][prompts[b]:upto], device="cuda", dtype=torch.long), minlength=V)
                r, f, p = (float(s[k][b]) for k in ("repetition", "frequency", "presence"))
                x = torch.where(before > 0, torch.where(x > 0, x / r, x * r), x) - f * made - p * (made > 0)
            if c["bias"]:
                x = x.index_add(0, s["bias_ids"][b].long(), s["bias"][b].double())
            if c["mask"]:
                words = s["mask"][b, t].long() & 0xFFFFFFFF
                v = torch.arange(V, device="cuda")
                x = torch.where((words[v // 32] >> (v % 32)) & 1 == 1, x, float("-inf"))
            out[b, t] = torch.softmax(x / float(s["temperature"][b]), -1)
    return out


def _exact_int4(c, s):
    out = []
    for i in range(0, c["N"], 8192):
        w = s["codes"][i:i + 8192].double()
        w -= 8.0 if s["zeros"] is None else s["zeros"][i:i + 8192].double().repeat_interleave(c["group"], 1)
        w *= s["scales"][i:i + 8192].double().repeat_interleave(c["group"], 1)
        out.append(s["x"].double() @ w.T)
    return torch.cat(out, 1)


def exact(case, seed):
    s = _inputs(case, seed)
    return {"shared": _exact_shared, "groups": _exact_groups, "rules": _exact_rules, "int4": _exact_int4}[case["op"]](case, s)
