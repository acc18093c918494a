"""The paged 8-bit decoding path of a Llama-shaped stack, on the GPU.

Against the dense bf16 cache the logits may differ by the cache's own rounding:
a code is off by at most half a step (int8: amax / 254, about 2% of a value's
spread), so logits of a four-layer stack stay within a few percent of their
spread; the bound below is 10%.  Everything that does not change the numbers
(how tokens are split into steps, forking, compaction, drafts) is held to much
less: the same codes, so differences of bf16 rounding only.
"""
from __future__ import annotations

import pytest
import torch

from wal2026_b200.llama import LlamaShape, dense_llama, rvq_llama
from wal2026_b200.paged_decode import PagedDecoder, main

pytestmark = pytest.mark.gpu
DEV = "cuda"
SHAPE = LlamaShape(layers=4, hidden=1024, mlp=2048, heads=8, kv_heads=2, vocab=1500)


def _tokens(rows, n, seed=1):
    return torch.randint(0, SHAPE.vocab, (rows, n), device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed))


def _dense_logits(stack, tokens):
    """[rows, n, vocab] by the stack's own decode step over a dense cache."""
    rows, n = tokens.shape
    stack.allocate_cache(rows, n, fill_random=False)
    out = []
    for pos in range(n):
        cos, sin = stack.rope_tables(pos)
        out.append(stack.decode_step(tokens[:, pos], pos, cos, sin).float())
    return torch.stack(out, 1)


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("make", [rvq_llama, dense_llama])
def test_logits_follow_the_dense_cache(make, dtype):
    stack = make(SHAPE, seed=2)
    tokens = _tokens(3, 50)
    want = _dense_logits(stack, tokens)
    dec = PagedDecoder(stack, rows=3, max_len=64, page_size=16, dtype=dtype)
    got = dec.step(tokens).float()  # all at once: a prompt
    scale = float(want.std())
    assert float((got - want).square().mean().sqrt()) <= 0.1 * scale
    one = PagedDecoder(stack, rows=3, max_len=64, page_size=16, dtype=dtype)
    for pos in range(50):
        last = one.step(tokens[:, pos:pos + 1]).float()
        one.advance()
    assert float((last[:, 0] - want[:, -1]).square().mean().sqrt()) <= 0.1 * scale


def test_prompts_of_gemm_size_and_their_remainder():
    stack = rvq_llama(SHAPE, seed=4)
    tokens = _tokens(2, 150)
    want = _dense_logits(stack, tokens)
    dec = PagedDecoder(stack, rows=2, max_len=160)
    a = dec.step(tokens[:, :100]).float()  # 200 rows: the prefill GEMM
    dec.advance(torch.tensor([100, 100], dtype=torch.int32, device=DEV))
    b = dec.step(tokens[:, 100:]).float()
    got = torch.cat([a, b], 1)
    assert float((got - want).square().mean().sqrt()) <= 0.1 * float(want.std())


def test_ragged_rows_equal_rows_alone():
    stack = rvq_llama(SHAPE, seed=5)
    tokens, lens = _tokens(3, 40), [40, 7, 0]
    dec = PagedDecoder(stack, rows=3, max_len=64, page_size=32)
    news = torch.tensor(lens, dtype=torch.int32, device=DEV)
    dec.step(tokens, news)
    dec.advance(news)
    nxt = _tokens(3, 1, 9)
    got = dec.step(nxt).float()
    for b, n in enumerate(lens):
        alone = PagedDecoder(stack, rows=1, max_len=64, page_size=32)
        if n:
            alone.step(tokens[b:b + 1, :n])
            alone.advance(torch.tensor([n], dtype=torch.int32, device=DEV))
        ref = alone.step(nxt[b:b + 1]).float()
        assert float((got[b] - ref[0]).abs().max()) <= 0.05 * float(ref.std())


def test_greedy_drafts_are_kept_and_wrong_ones_cut():
    stack = rvq_llama(SHAPE, seed=6)
    prompt = _tokens(2, 20)
    n = torch.tensor([20, 20], dtype=torch.int32, device=DEV)
    plain = PagedDecoder(stack, rows=2, max_len=64, page_size=16)
    logits = plain.step(prompt)
    plain.advance(n)
    seq, gaps = [logits[:, -1].argmax(-1)], []
    for _ in range(6):
        logits = plain.step(seq[-1].view(2, 1)).float()
        plain.advance()
        top = logits[:, 0].topk(2).values
        gaps.append(float((top[:, 0] - top[:, 1]).min() / logits.std()))
        seq.append(logits[:, 0].argmax(-1))
    greedy = torch.stack(seq, 1).to(torch.int32)  # [2, 7]
    if min(gaps) < 0.02:
        pytest.skip("two tokens are nearly as likely: greedy decoding is not defined to that precision")
    for cut in (6, 2, 0):
        dec = PagedDecoder(stack, rows=2, max_len=64, page_size=16)
        dec.step(prompt)
        dec.advance(n)
        drafts = greedy[:, 1:].clone()
        if cut < 6:
            drafts[:, cut] = (drafts[:, cut] + 1) % SHAPE.vocab
        accepted, out = dec.speculate(drafts, torch.rand(2, 7, device=DEV), last=greedy[:, 0].contiguous(), temperature=0.0)
        assert accepted.tolist() == [cut, cut]
        assert torch.equal(out[:, :cut], greedy[:, 1:1 + cut])
        assert dec.lens.tolist() == [21 + cut] * 2
        if cut < 6:
            assert torch.equal(out[:, cut], greedy[:, 1 + cut])  # the token that greedy decoding takes instead
            # and decoding goes on from there as if nothing had been drafted
            nxt = dec.step(out[:, cut].view(2, 1)).float()[:, 0].argmax(-1)
            if cut + 2 < 7:
                assert torch.equal(nxt.to(torch.int32), greedy[:, cut + 2])


def test_forks_share_pages_and_go_their_own_way():
    stack = rvq_llama(SHAPE, seed=7)
    prompt = _tokens(1, 40).expand(3, 40).contiguous()
    dec = PagedDecoder(stack, rows=3, max_len=96, num_pages=12, page_size=16)
    news = torch.tensor([40, 0, 0], dtype=torch.int32, device=DEV)
    dec.step(prompt, news)
    dec.advance(news)
    dec.fork([0, 0, 0])
    assert dec.info.tolist() == [12 - 3, 0] and dec.lens.tolist() == [40] * 3
    branch = _tokens(3, 1, 11)
    got = dec.step(branch).float()
    assert dec.info.tolist() == [12 - 5, 0]  # two of the three copied the last page
    assert len({row[2] for row in dec.table.tolist()}) == 3
    dec.advance()
    for b in range(3):
        alone = PagedDecoder(stack, rows=1, max_len=96, page_size=16)
        alone.step(prompt[:1])
        alone.advance(torch.tensor([40], dtype=torch.int32, device=DEV))
        ref = alone.step(branch[b:b + 1]).float()
        assert float((got[b] - ref[0]).abs().max()) <= 0.05 * float(ref.std())
    before = dec.step(branch).float()
    dec.fork([2, -1, 2])
    dec.compact()
    assert dec.info[0] == 3 and dec.lens.tolist() == [41, 0, 41]
    after = dec.step(branch[2:].expand(3, 1).contiguous()).float()
    assert torch.equal(after[0], after[2])
    assert float((after[0] - before[2]).abs().max()) <= 0.05 * float(before[2].std())


def test_a_step_in_a_graph():
    stack = rvq_llama(SHAPE, seed=8)
    tokens = _tokens(2, 12)
    eager, graphed = (PagedDecoder(stack, rows=2, max_len=32, page_size=16) for _ in range(2))
    fed = tokens[:, :1].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graphed.step(fed)  # buffers of this step size
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        logits = graphed.step(fed)
        graphed.advance()
    graphed.lens.zero_()
    graphed.table.fill_(-1)
    for pos in range(12):
        fed.copy_(tokens[:, pos:pos + 1])
        g.replay()
        want = eager.step(tokens[:, pos:pos + 1])
        eager.advance()
        assert torch.equal(logits, want), pos
    assert graphed.lens.tolist() == [12, 12]


def test_refusals():
    stack = rvq_llama(SHAPE, seed=8)
    dec = PagedDecoder(stack, rows=2, max_len=32, page_size=16)
    with pytest.raises(ValueError, match="rows"):
        dec.step(_tokens(3, 1))
    with pytest.raises(ValueError, match="parents"):
        dec.fork([0])
    with pytest.raises(ValueError, match="parents"):
        dec.fork([0, 2])
    with pytest.raises(ValueError, match="positive"):
        PagedDecoder(stack, rows=0, max_len=32)


def test_the_example_runs(capsys):
    main()
    assert "pages used" in capsys.readouterr().out


def test_idle_rows_of_a_speculative_step():
    # draft_lens -1: nothing stored, reserved or drawn; the other rows as if they were alone
    stack = rvq_llama(SHAPE, seed=9)
    prompt, lens = _tokens(3, 20), torch.tensor([20, 16, 0], dtype=torch.int32, device=DEV)
    last, drafts = _tokens(3, 1, 2).int().view(3), _tokens(3, 3, 3).int()
    u = torch.rand(3, 4, device=DEV, generator=torch.Generator(device=DEV).manual_seed(4))
    both = []
    for idle in (True, False):
        dec = PagedDecoder(stack, rows=3, max_len=64, page_size=16)
        dec.step(prompt, lens)
        dec.advance(lens)
        dl = torch.tensor([3, -1 if idle else 0, -1 if idle else 2], dtype=torch.int32, device=DEV)
        table = dec.table.clone()
        accepted, out = dec.speculate(drafts, u, last=last, draft_lens=dl)
        both.append((accepted, out))
        if idle:
            assert accepted.tolist()[1:] == [0, 0] and bool((out[1:] == -1).all())
            assert dec.lens.tolist()[1:] == [16, 0] and torch.equal(dec.table[1:], table[1:])
        else:
            assert dec.lens.tolist()[1] == 17 and bool((out[1:, 0] >= 0).all())
    assert torch.equal(both[0][0][0], both[1][0][0]) and torch.equal(both[0][1][0], both[1][1][0])
