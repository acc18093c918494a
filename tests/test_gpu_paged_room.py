"""``PagedDecoder`` when pages run out: a step that finds no room changes nothing and can be repeated.

A decoder whose pool ran out and was given room, and one whose pool was large
all along, hold the same codes in other pages: their logits are equal bit for bit.
"""
from __future__ import annotations

import pytest
import torch

from wal2026_b200.llama import LlamaShape, rvq_llama
from wal2026_b200.paged_decode import PagedDecoder

pytestmark = pytest.mark.gpu
DEV = "cuda"
SHAPE = LlamaShape(layers=2, hidden=512, mlp=1024, heads=8, kv_heads=2, vocab=700)


@pytest.fixture(scope="module")
def stack():
    return rvq_llama(SHAPE, seed=5)


def _tokens(rows, n, seed=1):
    return torch.randint(0, SHAPE.vocab, (rows, n), device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed))


def _i32(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _two_forks_and_a_third(stack, num_pages):
    """Rows 0 and 1 share 20 tokens in two pages of 16, row 2 has 20 of its own."""
    dec = PagedDecoder(stack, rows=3, max_len=64, num_pages=num_pages, page_size=16)
    news = _i32(20, 0, 20)
    dec.step(_tokens(3, 20), news)
    dec.advance(news)
    dec.fork([0, 0, 2])
    return dec


def test_a_shared_page_survives_a_step_without_room(stack):
    small, large = (_two_forks_and_a_third(stack, n) for n in (4, 20))
    table = small.table.clone()
    fed = _tokens(3, 1, 7)
    for tries in (1, 2):  # row 1 wants a copy of the page it shares and row 0 is left its own: one page short
        small.step(fed)
        assert small.info.tolist() == [0, 1] and int(small.missing) == tries
        small.advance()
        assert torch.equal(small.table, table) and small.lens.tolist() == [20, 20, 20]
    for dec in (small, large):
        dec.fork([0, 1, -1])
    news = _i32(1, 1, 0)
    got, want = (dec.step(fed, news) for dec in (small, large))
    assert torch.equal(got[:2], want[:2]) and small.info.tolist()[1] == 0 and int(large.missing) == 0
    for dec in (small, large):
        dec.advance(news)
        assert dec.lens.tolist() == [21, 21, 0]
    again = _tokens(3, 1, 8)
    got, want = (dec.step(again, news) for dec in (small, large))
    assert torch.equal(got[:2], want[:2])


def test_speculation_without_room_keeps_nothing(stack):
    small, large = (_two_forks_and_a_third(stack, n) for n in (4, 20))
    table = small.table.clone()
    last, drafts = _tokens(3, 1, 3).int().view(3), _tokens(3, 4, 4).int()
    u = torch.rand(3, 5, device=DEV, generator=torch.Generator(device=DEV).manual_seed(2))
    accepted, out = small.speculate(drafts, u, last=last)
    assert accepted.tolist() == [0, 0, 0] and bool((out == -1).all())
    assert torch.equal(small.table, table) and small.lens.tolist() == [20, 20, 20] and int(small.missing) > 0
    small.fork([0, -1, -1])
    large.fork([0, -1, -1])
    news = _i32(1, 0, 0)
    got, want = (dec.step(last.view(3, 1), news) for dec in (small, large))
    assert torch.equal(got[0], want[0])


def test_a_row_that_is_full(stack):
    dec = PagedDecoder(stack, rows=2, max_len=32, page_size=16)
    news = _i32(32, 5)
    dec.step(_tokens(2, 32), news)
    dec.advance(news)
    table = dec.table.clone()
    dec.step(_tokens(2, 1, 2))
    dec.advance()
    assert dec.info.tolist()[1] == 1 and dec.lens.tolist() == [32, 5] and torch.equal(dec.table, table)
    only = _i32(0, 1)
    dec.step(_tokens(2, 1, 2), only)  # the other row goes on
    dec.advance(only)
    assert dec.info.tolist()[1] == 0 and dec.lens.tolist() == [32, 6]


def test_a_graph_stops_at_the_end_of_the_pool(stack):
    dec = PagedDecoder(stack, rows=1, max_len=64, num_pages=2, page_size=16)
    fed = _tokens(1, 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        dec.step(fed)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        dec.step(fed)
        dec.advance()
    for _ in range(36):
        g.replay()
    assert dec.lens.tolist() == [32] and int(dec.missing) == 4
    assert sorted(dec.table.tolist()[0]) == [-1, -1, 0, 1]


def test_the_last_page_of_a_row_is_whole(stack):
    # max_len inside a page: positions to the page's end have a place, so they have their rotation too
    tokens, news = _tokens(1, 30), _i32(30)
    short, long = (PagedDecoder(stack, rows=1, max_len=n, page_size=16) for n in (20, 64))
    got, want = (dec.step(tokens) for dec in (short, long))
    assert torch.equal(got, want)
    for dec in (short, long):
        dec.advance(news)
    fed = _tokens(1, 2, 6)
    assert torch.equal(short.step(fed), long.step(fed)) and short.info.tolist()[1] == 0
    short.step(_tokens(1, 3, 6))  # past the page: no room
    assert short.info.tolist()[1] == 1


def test_steps_of_many_sizes_hold_one_set_of_buffers(stack):
    def held(sizes):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        dec = PagedDecoder(stack, rows=2, max_len=64, page_size=16)
        logits = [dec.step(_tokens(2, n)) for n in sizes]
        last = logits[-1].clone()
        del logits
        return torch.cuda.memory_allocated() - before, last, dec

    held([64])  # what a first call keeps for good
    one, want, _ = held([64])
    many, got, dec = held([*range(1, 65), 3, 64])
    assert many <= one + (1 << 16) and torch.equal(got, want)
    small, ref, _ = held([3])
    assert torch.equal(dec.step(_tokens(2, 3)), ref)
    with pytest.raises(ValueError, match="at least one token"):
        dec.step(_tokens(2, 1)[:, :0])


def test_a_captured_step_keeps_its_buffers(stack):
    tokens = _tokens(1, 12)
    fed = tokens[:, :1].clone()
    dec, eager = (PagedDecoder(stack, rows=1, max_len=64, page_size=16) for _ in range(2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        dec.step(fed)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        logits = dec.step(fed)
        dec.advance()
    first, other = torch.cuda.CUDAGraph(), _tokens(1, 3, 5)
    with torch.cuda.graph(first):  # a size that was not run before
        wide = dec.step(other)
    for pos in range(12):
        if pos == 3:  # a larger step, and others who would take memory that it gave back
            assert torch.equal(dec.step(_tokens(1, 40, 9)), eager.step(_tokens(1, 40, 9)))
            junk = [torch.full((1 << k,), float("nan"), device=DEV) for k in range(8, 22)]
        if pos == 6:
            first.replay()
            assert torch.equal(wide, eager.step(other))
        fed.copy_(tokens[:, pos:pos + 1])
        g.replay()
        assert torch.equal(logits, eager.step(fed)), pos
        eager.advance()
    del junk
