"""Shared attention calls that overlap: a stream and a workspace each, as the documentation asks for."""
from __future__ import annotations

import pytest
import torch

from tests.test_gpu_kv8_shared import DEV, E4M3, INT8, _check, _filled, _forks, _gen, _groups, _i32
from wal2026_b200.kv8 import kv8_attention_shared, kv8_attention_shared_workspace

pytestmark = pytest.mark.gpu


def _case(seed, dtype, hq, hkv, T, fork, length):
    P = 32
    table, lens, pages = _forks([("a", length, 13 * i) for i in range(fork)], P, T, seed)
    cache = _filled(pages, hkv, P, 128, dtype, seed)
    q = torch.randn(fork * T, hq * 128, device=DEV, generator=_gen(seed)).to(torch.bfloat16)
    groups, ws = _groups(table, lens, P, 64), kv8_attention_shared_workspace(cache, fork, hq, T)
    want = _check(cache, q, table, lens, groups)
    return (cache, 0, q, table, _i32(lens), groups, torch.empty_like(q), ws), want, torch.zeros(1, dtype=torch.int32, device=DEV)


def test_two_streams_at_once():
    cases = [_case(1, INT8, 16, 2, 1, 24, 6000), _case(2, E4M3, 8, 8, 3, 7, 3000)]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(20):
        for (args, _, status), s in zip(cases, streams):
            with torch.cuda.stream(s):
                kv8_attention_shared(*args, status=status)
    torch.cuda.synchronize()
    for args, want, status in cases:
        assert status.item() == 0 and torch.equal(args[6], want)


def test_two_branches_of_a_graph():
    cases = [_case(3, INT8, 16, 2, 1, 24, 6000), _case(4, INT8, 4, 1, 2, 40, 2500)]
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        side.wait_stream(torch.cuda.current_stream())
        for _ in range(4):
            kv8_attention_shared(*cases[0][0], status=cases[0][2])
            with torch.cuda.stream(side):
                kv8_attention_shared(*cases[1][0], status=cases[1][2])
        torch.cuda.current_stream().wait_stream(side)
    for _ in range(3):
        for args, _, _ in cases:
            args[6].zero_()
        graph.replay()
        for args, want, status in cases:
            assert status.item() == 0 and torch.equal(args[6], want)
