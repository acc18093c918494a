"""Shared attention with scales of either sign, as ``kv8_attention`` takes them.

The reference and its tolerance are those of ``test_gpu_kv8_shared``.
"""
from __future__ import annotations

import pytest
import torch

from tests.test_gpu_kv8_shared import DEV, E4M3, INT8, _check, _filled, _forks, _gen, _groups

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [INT8, E4M3])
@pytest.mark.parametrize("scale", [-0.3, -0.05, -4.0, 0.0, -0.0, 0.7])
@pytest.mark.parametrize("hq,hkv,hd,T,fork", [(8, 2, 64, 1, 4), (16, 2, 128, 3, 12), (4, 4, 128, 1, 2)])
def test_shared_attention_with_any_scale(dtype, scale, hq, hkv, hd, T, fork):
    P = 32
    table, lens, pages = _forks([("a", 900, 17 * i) for i in range(fork)], P, T, 5)
    cache = _filled(pages, hkv, P, hd, dtype, hd + T)
    q = torch.randn(fork * T, hq * hd, device=DEV, generator=_gen(3)).to(torch.bfloat16)
    groups = _groups(table, lens, P, 64)
    assert int((groups[3] > 0).sum()) == fork
    _check(cache, q, table, lens, groups, scale=scale)
