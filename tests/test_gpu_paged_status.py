"""A wait that the attention of shared prefixes gives up is seen at the decoder.

The attention's word is set on the host's behalf, as its kernel sets it: no wait is made to run out.
"""
from __future__ import annotations

import pytest
import torch

from wal2026_b200 import paged_decode
from wal2026_b200.llama import LlamaShape, dense_llama

pytestmark = pytest.mark.gpu
SHAPE = LlamaShape(layers=2, hidden=256, mlp=512, heads=4, kv_heads=2, vocab=500)


def test_a_wait_given_up_in_one_layer_stays_seen(monkeypatch):
    dec = paged_decode.PagedDecoder(dense_llama(SHAPE, seed=1), rows=3, max_len=128, page_size=16, share=16)
    tokens = torch.randint(0, SHAPE.vocab, (3, 40), device="cuda")
    dec.step(tokens)
    dec.advance(torch.full((3,), 40, dtype=torch.int32, device="cuda"))
    dec.fork([0, 0, 0])
    assert dec.status.tolist() == [0]
    real, calls = paged_decode.kv8_attention_shared, []

    def shared(cache, layer, *args, status=None, **kw):
        real(cache, layer, *args, status=status, **kw)
        calls.append(status)
        if len(calls) == 3:  # the second step's first layer
            status.fill_(1)

    monkeypatch.setattr(paged_decode, "kv8_attention_shared", shared)
    seen = []
    for i in range(3):
        dec.step(tokens[:, :1])
        dec.advance()
        seen += dec.status.tolist()
    assert len(calls) == 6 and all(s is dec.status for s in calls) and seen == [0, 1, 1]
    dec.status.zero_()
    dec.step(tokens[:, :1])
    assert dec.status.tolist() == [0]


def test_a_captured_step_sets_the_same_word():
    dec = paged_decode.PagedDecoder(dense_llama(SHAPE, seed=1), rows=2, max_len=128, page_size=16, share=16)
    tokens = torch.randint(0, SHAPE.vocab, (2, 40), device="cuda")
    dec.step(tokens)
    dec.advance(torch.full((2,), 40, dtype=torch.int32, device="cuda"))
    dec.fork([1, 1])
    last = tokens[:, :1].contiguous()
    dec.step(last)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dec.step(last)
    dec.status.fill_(1)
    graph.replay()
    assert dec.status.tolist() == [1]  # only the caller clears it
    dec.status.zero_()
    graph.replay()
    assert dec.status.tolist() == [0]
