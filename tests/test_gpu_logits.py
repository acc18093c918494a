"""Rules on logits on the GPU against their definition in 64 bits.

Tolerance.  Each of up to five steps (x / repetition or x * repetition, frequency,
presence, bias, x / temperature) rounds to fp32, and the difference to the
maximum once more: with A the largest magnitude that occurs, an exponent is off
by at most 8 * 2^-24 * A, and its maximum by as much; exp is good to 2 units
(2^-22), the sum of V terms in any order to (log2(1024) + V / 512) roundings and the
factors to three.  Probabilities are therefore compared relative to
    16 * 2^-24 * A + (V / 512 + 24) * 2^-23,
below fp32's smallest normal number absolutely.  Logits are compared with 8 * 2^-24 * A, and
a step that leaves fp32's range gives an infinity in either.  A is taken for each row.
"""
from __future__ import annotations

import pytest
import torch

from wal2026_b200.logits import logit_rules, pack_mask

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _f32(v):
    return torch.tensor(v, dtype=F32, device=DEV)


def _reference(logits, softmax=True, text=None, lens=None, prompt_lens=None, new_lens=None, repetition=None, presence=None,
               frequency=None, bias_ids=None, bias=None, allowed=None, temperature=None):
    """(out, largest magnitude met in each row) in float64."""
    B, T, V = logits.shape
    out = torch.zeros(B, T, V, dtype=torch.float64, device=DEV)
    mosts = torch.ones(B, T, 1, dtype=torch.float64, device=DEV)
    for b in range(B):
        for t in range(T):
            if new_lens is not None and t >= int(new_lens[b]):
                continue
            x = logits[b, t].double()

            def see(x):
                x = torch.where(x.float().isinf(), x.float().double(), x)  # past fp32's largest number
                f = x[x.isfinite()]
                if f.numel():
                    mosts[b, t] = torch.maximum(mosts[b, t], f.abs().max())
                return x

            x = see(x)
            if repetition is not None or presence is not None or frequency is not None:
                upto = max(0, min(int(lens[b]) + t + 1, text.shape[1]))
                p0 = 0 if prompt_lens is None else max(0, int(prompt_lens[b]))
                toks = [v for v in text[b, :upto].tolist()]
                made, seen = torch.zeros(V, dtype=torch.float64), torch.zeros(V, dtype=torch.bool)
                for j, v in enumerate(toks):
                    if 0 <= v < V:
                        seen[v] = True
                        made[v] += j >= p0
                made, seen = made.to(DEV), seen.to(DEV)
                r = 1.0 if repetition is None else float(repetition[b])
                x = see(torch.where(seen, torch.where(x > 0, x / r, x * r), x))
                x = x - (0.0 if frequency is None else float(frequency[b])) * made
                x = x - (0.0 if presence is None else float(presence[b])) * (made > 0)
                x = see(x)
            if bias is not None:
                for i, v in enumerate(bias_ids[b].tolist()):
                    if 0 <= v < V:
                        x[v] = x[v] + float(bias[b, i])
                x = see(x)
            if allowed is not None:
                x = torch.where(allowed[b, t], x, float("-inf"))
            x = torch.where(x.isnan(), float("-inf"), x)
            temp = 1.0 if temperature is None else float(temperature[b])
            if temp > 0:
                x = x / temp
                x = torch.where(x.isnan(), float("-inf"), x)
                x = see(x)
            if not softmax:
                out[b, t] = x
                continue
            top = x.max()
            if top == float("-inf"):
                continue
            if not temp > 0:
                out[b, t, int((x == top).nonzero()[0])] = 1.0
                continue
            e = torch.where(x == top, 1.0, torch.exp(x - top))
            out[b, t] = e / e.sum()
    return out, mosts


def _check(logits, allowed=None, softmax=True, **rules):
    B, T, V = logits.shape
    out = torch.full((B, T, V), float("nan"), device=DEV)
    mask = None if allowed is None else pack_mask(allowed)
    logit_rules(logits, out, mask=mask, softmax=softmax, **rules)
    want, most = _reference(logits, softmax, allowed=allowed, **rules)
    if softmax:
        tol = want * (16 * 2.0 ** -24 * most + (V / 512 + 24) * 2.0 ** -23) + 2.0 ** -126
        bad = ~((out.double() - want).abs() <= tol)
    else:
        bad = ~((out.double() == want) | ((out.double() - want).abs() <= 8 * 2.0 ** -24 * most))
    assert not bool(bad.any()), (int(bad.sum()), float((out.double() - want).abs().max()))
    again = torch.empty_like(out)
    logit_rules(logits, again, mask=mask, softmax=softmax, **rules)
    assert torch.equal(out, again)
    return out


def _inputs(B, T, V, L, nb, dtype, seed):
    g = _gen(seed)
    logits = (4 * torch.randn(B, T, V, device=DEV, generator=g)).to(dtype)
    text = torch.randint(0, max(1, V // 3), (B, L), device=DEV, generator=g, dtype=torch.int32)
    lens = _i32([max(0, L - T - 3 * b) for b in range(B)])
    rules = dict(text=text, lens=lens, prompt_lens=_i32([int(n) // 2 for n in lens]),
                 repetition=1 + torch.rand(B, device=DEV, generator=g), presence=torch.rand(B, device=DEV, generator=g),
                 frequency=0.3 * torch.rand(B, device=DEV, generator=g), temperature=0.5 + torch.rand(B, device=DEV, generator=g),
                 bias_ids=torch.randint(0, V, (B, nb), device=DEV, generator=g, dtype=torch.int32),
                 bias=3 * torch.randn(B, nb, device=DEV, generator=g))
    allowed = torch.rand(B, T, V, device=DEV, generator=g) < 0.3
    return logits, rules, allowed


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("B,T,V,L", [(1, 1, 1, 1), (2, 3, 31, 9), (3, 1, 1000, 300), (1, 5, 2049, 64), (2, 2, 4097, 1000),
                                     (1, 1, 16387, 40), (2, 1, 32000, 5000), (1, 2, 128256, 700)])
def test_all_rules_together(dtype, B, T, V, L):
    logits, rules, allowed = _inputs(B, T, V, L, 5, dtype, V + T)
    _check(logits, allowed, **rules)
    _check(logits, allowed, softmax=False, **rules)


@pytest.mark.parametrize("names", [(), ("repetition",), ("presence",), ("frequency",), ("temperature",), ("bias_ids", "bias"),
                                   ("mask",), ("repetition", "mask"), ("presence", "frequency", "temperature")])
@pytest.mark.parametrize("V", [777, 20480])
def test_each_rule_alone(names, V):
    logits, rules, allowed = _inputs(2, 2, V, 200, 9, BF, V)
    keep = {k: v for k, v in rules.items() if k in names}
    if any(k in names for k in ("repetition", "presence", "frequency")):
        keep.update(text=rules["text"], lens=rules["lens"])
    _check(logits, allowed if "mask" in names else None, **keep)


def test_rows_with_nothing_left_and_values_that_are_not_finite():
    inf, nan = float("inf"), float("nan")
    B, T, V = 6, 2, 5000
    logits, rules, allowed = _inputs(B, T, V, 50, 4, F32, 3)
    allowed[0] = False                                   # an empty row
    logits[1, 0] = -inf                                  # nothing to choose from
    logits[1, 1] = torch.finfo(F32).min                  # masks made of the type's lowest value
    logits[1, 1, 77] = 0.0
    logits[2, :, ::2] = nan                              # left out
    logits[2, 0, 1], allowed[2, 0, 1] = nan, False       # in a masked place
    logits[3, 0, 4096], allowed[3, 0, 4096] = inf, False
    logits[3, 1, 9], logits[3, 1, 4999] = inf, inf       # these two share it
    allowed[3, 1, 9] = allowed[3, 1, 4999] = True
    logits[4] = nan
    rules["bias"][5, 0] = -inf                           # a banned token
    rules["text"][3] = 0                                 # away from the infinite ones
    out = _check(logits, allowed, **rules)
    assert float(out[0].abs().sum()) == 0.0 and float(out[4].abs().sum()) == 0.0
    assert out[3, 1, 9] == 0.5 and out[3, 1, 4999] == 0.5
    _check(logits, allowed, softmax=False, **rules)
    low = torch.full((1, 1, 300), torch.finfo(F32).min, device=DEV)
    assert bool(((_check(low) - 1 / 300).abs() < 1e-8).all())


@pytest.mark.parametrize("V", [5, 4000, 30001])
def test_greedy_takes_the_first_of_the_largest(V):
    logits, rules, allowed = _inputs(5, 2, V, 20, 2, BF, V)
    logits[0] = 1.0
    logits[1, :, V // 2:] = 9.0
    allowed[1, :, V // 2] = False
    allowed[2] = False
    temp = _f32([0.0, 0.0, 0.0, -1.0, float("nan")])
    out = _check(logits, allowed, temperature=temp)
    assert torch.equal(out.sum(-1), allowed.any(-1).float())  # one each, none where nothing is allowed
    _check(logits, allowed, temperature=temp, softmax=False)


def test_texts_of_no_and_of_wrong_tokens():
    B, T, V = 4, 3, 700
    logits, rules, _ = _inputs(B, T, V, 40, 6, BF, 12)
    rules["text"][0, :5] = _i32([-1, V, 2 ** 31 - 1, -2 ** 31, 3])
    rules["lens"] = _i32([0, -5, 1000, 39])              # the new token alone, a negative one, past the text
    rules["prompt_lens"] = _i32([0, 3, -7, 100])
    rules["bias_ids"][1] = _i32([-1, V, 5, 5, 5, 2 ** 31 - 1])  # unused places, and the same token three times
    _check(logits, **rules)
    _check(logits, **(rules | dict(prompt_lens=None)))
    empty = rules | dict(text=rules["text"][:, :0])
    _check(logits, **empty)
    _check(logits, **(rules | dict(bias_ids=rules["bias_ids"][:, :0].contiguous(), bias=rules["bias"][:, :0].contiguous())))


def test_padding_rows_strides_and_shared_masks():
    B, T, V = 3, 4, 1001
    logits, rules, allowed = _inputs(B, T, V, 60, 3, BF, 5)
    news = _i32([4, 0, 2])
    wide = torch.zeros(B, T + 1, V + 7, dtype=BF, device=DEV)
    wide[:, 1:, 3:3 + V] = logits
    out = torch.full((B, T + 2, V + 9), 7.0, device=DEV)
    text = torch.full((B, 90), 5, dtype=torch.int32, device=DEV)
    text[:, :60] = rules["text"]
    mask = pack_mask(allowed[:, :1]).expand(B, T, -1)
    rules = rules | dict(text=text[:, :60], new_lens=news)
    view = out[:, 2:, 5:5 + V]
    logit_rules(wide[:, 1:, 3:3 + V], view, mask=mask, **rules)
    want, most = _reference(logits, allowed=allowed[:, :1].expand(B, T, V), **rules)
    assert bool(((view.double() - want).abs() <= want * (16 * 2.0 ** -24 * most + 26 * 2.0 ** -23) + 2.0 ** -126).all())
    assert float(view[1].abs().sum()) == 0.0 and float(view[2, 2:].abs().sum()) == 0.0
    out[:, 2:, 5:5 + V] = 7.0
    assert bool((out == 7.0).all())  # nothing else was written


@pytest.mark.parametrize("T,keep", [(2, (1,)), (3, (2, 1, 3, 0)), (5, (1, 3))])
def test_skipped_rows_between_rows_of_several_ctas(T, keep):
    # more rows than clusters of CTAs run at a time, so that a cluster goes from one sequence's rows to the next one's
    B, V = 150, 33000
    logits = torch.randn(B, T, V, device=DEV, generator=_gen(T))
    scale = torch.arange(1, B + 1, device=DEV).view(B, 1, 1) / 20.0  # maxima and sums differ from row to row
    logits = (logits * scale).contiguous()
    news = _i32([keep[b % len(keep)] for b in range(B)])
    live = (torch.arange(T, device=DEV) < news[:, None]).unsqueeze(-1)
    want = torch.softmax(logits.double(), -1) * live
    most = logits.abs().amax(-1, keepdim=True).double()
    bound = want * (16 * 2.0 ** -24 * most + (V / 512 + 24) * 2.0 ** -23) + 2.0 ** -126
    for _ in range(5):
        out = torch.full((B, T, V), 7.0, device=DEV)
        logit_rules(logits, out, new_lens=news)
        assert bool(((out.double() - want).abs() <= bound).all())


def test_the_largest_vocabulary_and_as_many_biases_as_are_allowed():
    V = 393216
    g = _gen(1)
    logits = torch.randn(1, 1, V, device=DEV, generator=g)
    ids = torch.randint(0, 500, (1, 1024), device=DEV, generator=g, dtype=torch.int32)  # many are equal
    _check(logits, bias_ids=ids, bias=0.01 * torch.randn(1, 1024, device=DEV, generator=g), temperature=_f32([0.9]))


def test_a_draft_sees_the_drafts_before_it():
    V, T = 64, 3
    logits = torch.zeros(1, T, V, device=DEV)
    text = _i32([[9, 9, 3, 4, 5]])
    out = _check(logits, softmax=False, text=text, lens=_i32([2]), prompt_lens=_i32([1]), frequency=_f32([1.0]))
    assert out[0, 0, 9] == -1 and out[0, 0, 3] == -1 and out[0, 0, 4] == 0
    assert out[0, 2, 3] == -1 and out[0, 2, 4] == -1 and out[0, 2, 5] == -1


def test_on_another_stream_and_captured():
    logits, rules, allowed = _inputs(2, 2, 3001, 80, 3, BF, 9)
    mask, out = pack_mask(allowed), torch.empty(2, 2, 3001, device=DEV)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        logit_rules(logits, out, mask=mask, **rules)
    s.synchronize()
    want = _check(logits, allowed, **rules)
    assert torch.equal(out, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logit_rules(logits, out, mask=mask, **rules)
    rules["lens"].sub_(10)
    logits.neg_()
    graph.replay()
    assert torch.equal(out, _check(logits, allowed, **rules))


def test_refusals():
    logits, rules, allowed = _inputs(2, 2, 100, 30, 3, BF, 2)
    out, mask = torch.empty(2, 2, 100, device=DEV), pack_mask(allowed)
    ok = rules | dict(mask=mask)
    logit_rules(logits, out, **ok)
    for change in (dict(text=None), dict(lens=None), dict(text=rules["text"].long()), dict(text=rules["text"][:1]),
                   dict(lens=rules["lens"].long()), dict(bias=None), dict(bias=rules["bias"][:, :2]), dict(mask=mask[:, :1]),
                   dict(mask=mask.long()), dict(temperature=rules["temperature"].double()), dict(repetition=_f32([1.0])),
                   dict(mask=mask.cpu()), dict(new_lens=rules["lens"][:1])):
        with pytest.raises(ValueError):
            logit_rules(logits, out, **(ok | change))
    for bad in ((logits[0], out[0]), (logits.double(), out), (logits, out.to(BF)), (logits, out[:, :1]), (logits.cpu(), out.cpu()),
                (logits.transpose(1, 2), out.transpose(1, 2)), (logits[:0], out[:0]), (logits, out[:1].expand(2, 2, 100))):
        with pytest.raises(ValueError):
            logit_rules(*bad)
    with pytest.raises(ValueError):
        logit_rules(torch.zeros(1, 1, 393217, device=DEV), torch.zeros(1, 1, 393217, device=DEV))
