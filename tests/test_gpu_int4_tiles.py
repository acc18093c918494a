"""4-bit linears of more row tiles than the grid takes at once, as a vocabulary projection has.

The reference and its tolerance are those of ``test_gpu_int4``.
"""
from __future__ import annotations

import pytest
import torch

from tests.test_gpu_int4 import BF, DEV, F32, HF, _check, _gen, _layer
from wal2026_b200.int4 import Int4Linear

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True)])
@pytest.mark.parametrize("N,K", [(40011, 256), (20000, 1024), (5003, 8192)])
def test_int4_ctas_that_take_several_groups_of_tiles(group, zeros, N, K):
    # 296 CTAs at most: 40011 rows are 313 groups of eight tiles or more, 5003 rows 313 tiles of their own
    layer, w = _layer(N, K, group, zeros, N, bias=group == 64)
    for M, dtype, y_dtype in ((1, BF, BF), (5, HF, F32), (12, BF, F32), (24, HF, HF), (50, BF, BF)):
        x = torch.randn(M, K, device=DEV, generator=_gen(M)).to(dtype)
        y = torch.full((M, N), float("nan"), dtype=y_dtype, device=DEV)
        layer.gemv_into(x, y)
        _check(layer, w, x, y)
        again = torch.empty_like(y)
        layer.gemv_into(x, again)
        assert torch.equal(y, again)


def test_int4_rows_do_not_depend_on_the_rows_beside_them():
    layer, w = _layer(40011, 512, 64, True, 3)
    x = torch.randn(7, 512, device=DEV, generator=_gen(4)).to(BF)
    y = torch.empty(7, 40011, device=DEV, dtype=F32)
    layer.gemv_into(x, y)
    _check(layer, w, x, y)
    one = torch.empty(1, 40011, device=DEV, dtype=F32)
    for i in range(7):
        layer.gemv_into(x[i:i + 1], one)
        assert torch.equal(one[0], y[i])


@pytest.mark.parametrize("K", [32, 96, 160, 256])
def test_int4_an_infinite_scale_of_the_last_group(K):
    g = _gen(K)
    codes = torch.randint(0, 16, (33, K), device=DEV, generator=g, dtype=torch.uint8)
    scales = torch.rand(33, K // 32, device=DEV, generator=g).to(HF)
    scales[::2, -1] = float("inf")
    codes[:, K - 32:] = 11  # all three above the zero point
    x = torch.rand(3, K, device=DEV, generator=g).to(BF) + 1
    y = torch.empty(3, 33, device=DEV)
    Int4Linear(codes, scales).gemv_into(x, y)
    assert bool((y[:, ::2] == float("inf")).all()) and bool(y[:, 1::2].isfinite().all())
