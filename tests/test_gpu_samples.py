"""Several samples of prompts on the GPU: shared prefixes, rules on logits and the 4-bit head in one decoding loop.

The attention of a shared step and of a plain one are each within 2^-8 of a value
and (2^-11 + 2^-13) of the weighted mean of |v| of the exact one, so they differ by
twice that; it is compared layer by layer on the step's own queries and cache.
What the rules and the verification make of given logits is compared for
equality.
"""
from __future__ import annotations

import pytest
import torch

from wal2026_b200.int4 import Int4Linear
from wal2026_b200.kv8 import kv8_attention, kv8_attention_workspace
from wal2026_b200.llama import LlamaShape, dense_llama, int4_llama, rvq_llama, time_decode
from wal2026_b200.logits import LogitRules, logit_rules, pack_mask
from wal2026_b200.paged_decode import PagedDecoder
from wal2026_b200.speculative import verify_drafts

pytestmark = pytest.mark.gpu
DEV = "cuda"
SHAPE = LlamaShape(layers=2, hidden=1024, mlp=2048, heads=8, kv_heads=2, vocab=1500)


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _tokens(rows, n, seed=1):
    return torch.randint(0, SHAPE.vocab, (rows, n), device=DEV, generator=_gen(seed))


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _decoder(stack, **kw):
    """Two prompts in rows 0 and 1, forked to rows 0 .. 6; row 7 empty."""
    dec = PagedDecoder(stack, rows=8, max_len=512, page_size=16, **kw)
    lens = _i32([300, 170, 0, 0, 0, 0, 0, 0])
    dec.step(_tokens(8, 300), lens)
    dec.advance(lens)
    dec.fork([0, 1, 0, 1, 0, 0, 1, -1])
    return dec


def _compare_attention(dec, T, news):
    """The last layer's attention of the last step against the plain attention on the same queries and cache."""
    bufs, cache = dec._buffers(T), dec.cache
    plain = torch.empty_like(bufs.attn)
    hq = dec.stack.layers[0].hq
    kv8_attention(cache, cache.layers - 1, bufs.q, dec.table, dec.lens, plain, kv8_attention_workspace(cache, dec.rows, hq, T), new_lens=news)
    most = float(cache.codes[-1, 1].float().abs().amax() * cache.scales[-1, 1].amax())
    off = (bufs.attn.float() - plain.float()).abs()
    assert bool((off <= 2 * (2.0 ** -8 * plain.float().abs() + (2.0 ** -11 + 2.0 ** -13) * most)).all())
    assert bool(plain.any())


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
def test_forked_rows_share_their_prompts(dtype):
    stack = rvq_llama(SHAPE, seed=3)
    dec = _decoder(stack, dtype=dtype, share=64)
    news = _i32([3, 3, 1, 2, 0, 3, 3, 2])
    for seed in range(3):
        dec.step(_tokens(8, 3, 10 + seed), news)
        assert dec.groups[2].tolist()[:3] == [4, 3, 0] and dec.groups[3].tolist() == [288, 160, 288, 160, 288, 288, 160, 0]
        _compare_attention(dec, 3, news)
        dec.advance(news)
    dec.compact()
    dec.step(_tokens(8, 1, 20))
    _compare_attention(dec, 1, None)
    dec.fork([0, -1, 0, -1, 1, 7, -1, 3])  # other groups: 0 with 2; 1 and 3 went to rows 4 and 7
    dec.step(_tokens(8, 1, 21))
    assert sorted(r for r in dec.groups[0].tolist() if r >= 0) == [0, 2, 4, 7]
    _compare_attention(dec, 1, None)


def test_a_decoder_without_groups_gives_the_same_bits():
    stack = rvq_llama(SHAPE, seed=3)
    a, b = (PagedDecoder(stack, rows=3, max_len=128, page_size=16, share=s) for s in (None, 32))
    tokens = _tokens(3, 60)
    assert torch.equal(a.step(tokens), b.step(tokens))


def test_a_captured_step_follows_the_groups():
    stack = rvq_llama(SHAPE, seed=5)
    dec = _decoder(stack, share=64)
    tokens = _tokens(8, 1, 4)
    dec.step(tokens)  # warm up; nothing is kept
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits = dec.step(tokens)
        dec.advance()
    for seed in range(3):
        tokens.copy_(_tokens(8, 1, 30 + seed))
        if seed == 2:
            dec.fork([1, 1, 2, 3, 4, 5, 6, 7])
        graph.replay()
        dec.lens.sub_(1)  # as the step saw them
        _compare_attention(dec, 1, None)
        again = dec.step(tokens)
        assert torch.equal(logits, again)
        dec.advance()


def _target(logits, texts, T, rules, prompts):
    """What the rules make of logits, the text of each row written out by hand."""
    B, n, V = logits.shape
    longest = max(len(t) for t in texts)
    text = torch.full((B, longest), -1, dtype=torch.int32, device=DEV)
    for b, t in enumerate(texts):
        text[b, :len(t)] = _i32(t)
    out = torch.empty(B, n, V, device=DEV)
    logit_rules(logits, out, text=text, lens=_i32([len(t) - n for t in texts]), prompt_lens=_i32(prompts),
                repetition=rules.repetition, presence=rules.presence, frequency=rules.frequency, bias_ids=rules.bias_ids,
                bias=rules.bias, mask=rules.mask.expand(B, n, -1), temperature=rules.temperature)
    return out


def test_speculation_under_rules_follows_the_rows_texts():
    stack = rvq_llama(SHAPE, seed=7)
    dec = _decoder(stack, share=64, text=True)
    prompts = _tokens(8, 300)
    source = [0, 1, 0, 1, 0, 0, 1]
    texts = [prompts[s, :[300, 170][s]].tolist() for s in source] + [[]]
    dec.prompt_lens.copy_(_i32([len(t) for t in texts]))
    g = _gen(8)
    allowed = torch.rand(8, 1, SHAPE.vocab, device=DEV, generator=g) < 0.5
    rules = LogitRules(repetition=1 + torch.rand(8, device=DEV, generator=g), presence=torch.rand(8, device=DEV, generator=g),
                       frequency=torch.rand(8, device=DEV, generator=g), bias_ids=torch.randint(0, SHAPE.vocab, (8, 6), device=DEV, generator=g, dtype=torch.int32),
                       bias=torch.randn(8, 6, device=DEV, generator=g), mask=pack_mask(allowed),
                       temperature=0.5 + torch.rand(8, device=DEV, generator=g))
    starts = [len(t) for t in texts]
    last = _tokens(8, 1, 50)[:, 0].int()
    for step in range(4):
        drafts = _tokens(8, 2, 60 + step).int()
        u = torch.rand(8, 3, device=DEV, generator=g)
        before = dec.lens.clone()
        logits = dec.step(torch.cat([last[:, None], drafts], 1))  # the same step, kept by none
        full = [t + [int(last[b])] + drafts[b].tolist() for b, t in enumerate(texts)]
        target = _target(logits, full, 2, rules, starts)
        want_a, want_t = _i32([0] * 8), torch.empty(8, 3, dtype=torch.int32, device=DEV)
        verify_drafts(target, None, drafts, u, want_a, want_t)
        accepted, tokens = dec.speculate(drafts, u, last=last, rules=rules)
        assert torch.equal(accepted, want_a) and torch.equal(tokens, want_t)
        assert torch.equal(dec.lens, before + accepted + 1)
        for b in range(8):
            a = int(accepted[b])
            texts[b] += [int(last[b])] + drafts[b, :a].tolist()
            assert dec.text[b, :len(texts[b])].tolist() == texts[b]
            token = int(tokens[b, a])
            assert token == -1 or bool(allowed[b, 0, token])
        last = tokens.gather(1, accepted.view(8, 1).long()).view(8).clamp(min=0).contiguous()
        if step == 1:
            dec.fork([3, 1, 2, 3, 4, 0, 6, -1])
            order = [3, 1, 2, 3, 4, 0, 6]
            texts, starts = [list(texts[i]) for i in order] + [[]], [starts[i] for i in order] + [0]
            last = last[torch.tensor(order + [7], device=DEV)].contiguous()
            assert dec.prompt_lens.tolist() == starts


def test_rules_without_penalties_and_temperature_zero():
    stack = rvq_llama(SHAPE, seed=9)
    dec = PagedDecoder(stack, rows=2, max_len=64, page_size=16)
    tokens = _tokens(2, 3)
    last, drafts, u = tokens[:, 0].int(), tokens[:, 1:].int().contiguous(), torch.rand(2, 3, device=DEV, generator=_gen(1))
    logits = dec.step(tokens)
    best = logits.float().argmax(-1)
    accepted, out = dec.speculate(drafts, u, last=last, temperature=0.0, rules=LogitRules())
    a = accepted.tolist()
    assert [int(out[b, a[b]]) for b in range(2)] == [int(best[b, a[b]]) for b in range(2)]
    with pytest.raises(ValueError):
        dec.speculate(drafts, u, last=last, rules=LogitRules(presence=torch.ones(2, device=DEV)))


def test_a_step_without_room_keeps_the_text():
    stack = rvq_llama(SHAPE, seed=9)
    dec = PagedDecoder(stack, rows=2, max_len=32, page_size=16, text=True, share=16)
    dec.step(_tokens(2, 30))
    dec.advance(_i32([30, 30]))
    text = dec.text.clone()
    dec.step(_tokens(2, 3, 5), _i32([3, 1]))  # row 0 has two places left
    dec.advance(_i32([3, 1]))
    assert dec.lens.tolist() == [30, 30] and torch.equal(dec.text, text) and dec.missing.item() > 0
    dec.step(_tokens(2, 2, 6))
    assert dec.text[:, 30:].tolist() == _tokens(2, 2, 6).tolist()


@pytest.mark.parametrize("zero_points", [False, True])
def test_quantized_head_computes_the_logits_of_its_weight(zero_points):
    stack = rvq_llama(SHAPE, seed=2)
    dec = PagedDecoder(stack, rows=3, max_len=64, page_size=16)
    tokens = _tokens(3, 40)
    dense = dec.step(tokens).float()
    stack.quantize_head(64, zero_points=zero_points)
    x = dec._buffers(40).x
    want = (x.double() @ stack.head.reconstruct_weight(torch.float32).double().T).view(3, 40, -1)
    mag = (x.double().abs() @ stack.head.reconstruct_weight(torch.float32).double().abs().T).view(3, 40, -1)
    got = dec.step(tokens)
    assert bool(((got.double() - want).abs() <= 1.01 * 2.0 ** -8 * want.abs() + mag * 2.0 ** -12).all())
    assert float((got.float() - dense).std()) < 0.2 * float(dense.std())  # 4 bits of a Gaussian: a tenth of its spread
    stack.head = None
    assert torch.equal(dec.step(tokens).float(), dense)


def test_int4_stack_steps():
    a, b = int4_llama(SHAPE, seed=4), dense_llama(SHAPE, seed=4)
    assert isinstance(a.layers[0].qkv, Int4Linear) and a.linear_bytes() < 0.3 * b.linear_bytes()
    a.quantize_head()
    assert a.linear_bytes() < 0.3 * b.linear_bytes()
    tokens = _tokens(2, 1)[:, 0]
    cos, sin = a.rope_tables(0)
    a.allocate_cache(2, 4, fill_random=False)
    plain = a.decode_step(tokens, 0, cos, sin).float()
    fused = a.decode_step_fused(tokens, 0, cos, sin).float()
    # the fused step keeps fp32 sums of o and down where the plain one rounds to bf16: a few roundings of 2^-8 per layer
    assert float((plain - fused).abs().max()) <= 0.1 * float(plain.std())
    dec = PagedDecoder(a, rows=2, max_len=64, page_size=16)
    assert bool(dec.step(_tokens(2, 40)).isfinite().all())
    assert time_decode(a, 2, 8, steps=2)["ms_per_step"] > 0
