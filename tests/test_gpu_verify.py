"""Verification of drafted tokens on the GPU: equality with the definition in whole numbers, and its distribution."""
from __future__ import annotations

import pytest
import torch

from wal2026_b200.speculative import verify_drafts

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ONE = 1 << 38


def _units(p):
    return (torch.nan_to_num(p.double(), nan=0.0).clamp(0, 1) * ONE).round().long().tolist()


def _reference(target, draft, drafts, u, lens):
    B, T = drafts.shape
    V = target.shape[2]
    acc, tok = [], []
    for b in range(B):
        U = [int(float(v) * (1 << 24)) for v in u[b].double()]
        x = drafts[b].tolist()
        a, n = 0, max(0, min(T, lens[b]))
        while a < n and 0 <= x[a] < V:
            q = _units(draft[b, a, x[a]]) if draft is not None else ONE
            if U[a] * q >= _units(target[b, a, x[a]]) << 24:
                break
            a += 1
        p = _units(target[b, a])
        w = p
        if a < n:
            q = _units(draft[b, a]) if draft is not None else [ONE if i == x[a] else 0 for i in range(V)]
            w = [max(i - j, 0) for i, j in zip(p, q)]
        if not sum(w):
            w = p
        r, c, token = sum(w) * U[T] >> 24, 0, -1
        for i, v in enumerate(w):
            c += v
            if c > r:
                token = i
                break
        acc.append(a)
        tok.append(x[:a] + [token] + [-1] * (T - a))
    return acc, tok


def _run(target, draft, drafts, u, lens=None):
    B, T = drafts.shape
    acc = torch.full((B,), 55, dtype=torch.int32, device=DEV)
    tok = torch.full((B, T + 1), 55, dtype=torch.int32, device=DEV)
    verify_drafts(target, draft, drafts, u, acc, tok, draft_lens=None if lens is None else torch.tensor(lens, dtype=torch.int32, device=DEV))
    return acc.tolist(), tok.tolist()


def _inputs(B, T, V, seed, sharp=2.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    logits = torch.randn(B, T + 1, V, device=DEV, generator=g) * sharp
    other = logits[:, :T] + 0.5 * torch.randn(B, T, V, device=DEV, generator=g)
    target, draft = torch.softmax(logits, -1), torch.softmax(other, -1)
    drafts = torch.multinomial(draft.reshape(B * T, V), 1, generator=g).view(B, T).int() if T else torch.empty(B, 0, dtype=torch.int32, device=DEV)
    return target, draft, drafts, torch.rand(B, T + 1, device=DEV, generator=g)


@pytest.mark.parametrize("B,T,V", [(1, 1, 2), (3, 4, 1), (5, 3, 1001), (2, 8, 32000), (9, 2, 8193), (1, 4, 128256),
                                   (4, 0, 777), (2, 40, 130), (1, 1, 300001)])
@pytest.mark.parametrize("with_draft", [True, False])
def test_verify_equals_its_definition(B, T, V, with_draft):
    target, draft, drafts, u = _inputs(B, T, V, B + T + V)
    lens = [(T - b) % (T + 1) for b in range(B)]
    draft = draft if with_draft else None
    for ln in (None, lens, [T + 9] * B, [-1] * B):
        assert _run(target, draft, drafts, u, ln) == _reference(target, draft, drafts, u, [T] * B if ln is None else ln)


def test_verify_edges():
    V, T = 513, 3
    target, draft, drafts, u = _inputs(8, T, V, 5)
    u[0], u[1] = 0.0, 0.99999994
    target[2], draft[2] = draft[2, 0], draft[2, 0]       # the same distribution: an empty residual cannot be reached
    u[2] = 0.5
    target[3] = 0.0                                       # nothing has probability
    target[4, :, 7:] = float("nan")
    draft[4, 1] = float("inf")
    drafts[5, 1], drafts[6, 0] = -1, V                    # no such token
    target[7] = 0.0
    target[7, :, V - 1] = 1.0                             # a sure thing, at the end
    drafts[7] = V - 1
    for d in (draft, None):
        assert _run(target, d, drafts, u) == _reference(target, d, drafts, u, [T] * 8)


def test_verify_empty_residual_draws_from_the_target():
    # q >= p everywhere (not normalised), and a draft that is refused: the residual has nothing
    V = 300
    target = torch.full((1, 2, V), 1.0 / V, device=DEV)
    draft = torch.full((1, 1, V), 2.0 / V, device=DEV)
    drafts = torch.tensor([[5]], dtype=torch.int32, device=DEV)
    u = torch.tensor([[0.9, 0.5]], device=DEV)
    acc, tok = _run(target, draft, drafts, u)
    assert (acc, tok) == _reference(target, draft, drafts, u, [1]) and acc == [0] and tok[0][0] == 150


def test_verify_strided_rows_and_shared_distributions():
    B, T, V = 3, 2, 1000
    target, draft, drafts, u = _inputs(B, T, V, 8)
    wide = torch.zeros(B, T + 1, V + 24, device=DEV)
    wide[:, :, 3:3 + V] = target
    assert _run(wide[:, :, 3:3 + V], draft, drafts, u) == _reference(target, draft, drafts, u, [T] * B)
    one = draft[:1].expand(B, T, V)  # every sequence drafted from one distribution
    assert _run(target, one, drafts, u) == _reference(target, one, drafts, u, [T] * B)
    with pytest.raises(ValueError):
        _run(target[:, :1].expand(B, T + 1, V), draft, drafts, u)  # rows that are one and the same


def test_verify_leaves_the_targets_distribution():
    # whatever the drafts, the first token of a step is distributed as the target says: 200k trials over 6 tokens,
    # every frequency within 5 standard deviations
    g = torch.Generator(device=DEV).manual_seed(3)
    V, n = 6, 200000
    p = torch.tensor([0.05, 0.3, 0.1, 0.25, 0.2, 0.1], device=DEV)
    q = torch.tensor([0.3, 0.05, 0.25, 0.2, 0.1, 0.1], device=DEV)
    x = torch.multinomial(q, n, replacement=True, generator=g).int()
    u = torch.rand(n, 2, device=DEV, generator=g)
    counts = torch.zeros(V, device=DEV)
    for i in range(0, n, 50000):
        xs = x[i:i + 50000, None].contiguous()
        B = xs.shape[0]
        acc, tok = torch.empty(B, dtype=torch.int32, device=DEV), torch.empty(B, 2, dtype=torch.int32, device=DEV)
        verify_drafts(p.expand(B, 2, V).contiguous(), q.expand(B, 1, V).contiguous(), xs, u[i:i + 50000].contiguous(), acc, tok)
        counts += torch.bincount(tok[:, 0].long(), minlength=V)
    assert bool(((counts - n * p).abs() <= 5 * (n * p * (1 - p)).sqrt()).all())
