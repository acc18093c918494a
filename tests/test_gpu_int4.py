"""4-bit linears on the GPU against the product in 64 bits.

Tolerance of a product: the weights c - z and the activations enter it exactly,
products and sums are fp32.  A sum of K terms in any order is off by at most
K * 2^-23 * sum |w x| (each addition rounds or cuts below 2^-23 of a partial sum of
that size); the scaling adds 2^-24 per group.  The rounding to bf16 or fp16 adds
eps / 2 of the value.
"""
from __future__ import annotations

import pytest
import torch

from wal2026_b200.int4 import Int4Linear, quantize_int4

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _layer(N, K, group, zeros, seed, bias=False):
    g = _gen(seed)
    codes = torch.randint(0, 16, (N, K), device=DEV, generator=g, dtype=torch.uint8)
    scales = (0.01 * torch.exp(torch.randn(N, K // group, device=DEV, generator=g))).to(HF)
    z = torch.randint(0, 16, (N, K // group), device=DEV, generator=g, dtype=torch.uint8) if zeros else None
    b = torch.randn(N, device=DEV, generator=g).to(BF) if bias else None
    w = (codes.double() - (8.0 if z is None else z.double().repeat_interleave(group, 1))) * scales.double().repeat_interleave(group, 1)
    return Int4Linear(codes, scales, z, b), w


def _check(layer, w, x, y):
    want, mag = x.double() @ w.T, x.double().abs() @ w.abs().T
    if layer.bias is not None:
        want, mag = want + layer.bias.double(), mag + layer.bias.double().abs()
    tol = mag * (layer.in_features + 8) * 2.0 ** -23
    if y.dtype != F32:
        tol = tol + want.abs() * torch.finfo(y.dtype).eps / 2 * 1.01 + (2.0 ** -25 if y.dtype == HF else 0)
    bad = ~((y.double() - want).abs() <= tol + 1e-30)
    assert not bool(bad.any()), (int(bad.sum()), float((y.double() - want).abs().max()))


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("x_dtype,y_dtype", [(BF, BF), (BF, F32), (HF, HF), (HF, F32), (BF, HF)])
@pytest.mark.parametrize("M,N,K", [(1, 1, 128), (1, 16, 256), (3, 17, 640), (8, 4096, 128), (9, 33, 1280), (16, 100, 4096),
                                   (17, 48, 384), (32, 65, 896), (33, 31, 256), (70, 15, 512)])
def test_int4_gemv_matches_the_product_in_64_bits(group, zeros, x_dtype, y_dtype, M, N, K):
    layer, w = _layer(N, K, group, zeros, M + N + K, bias=M % 2 == 1)
    x = torch.randn(M, K, device=DEV, generator=_gen(K)).to(x_dtype)
    y = torch.full((M, N), float("nan"), dtype=y_dtype, device=DEV)
    layer.gemv_into(x, y)
    _check(layer, w, x, y)
    again = torch.empty_like(y)
    layer.gemv_into(x, again)
    assert torch.equal(y, again)


@pytest.mark.parametrize("N,K,group", [(40, 32, 32), (16, 96, 32), (5, 14368, 32), (128, 14336, 64), (2000, 4096, 128)])
def test_int4_gemv_odd_columns_and_long_rows(N, K, group):
    layer, w = _layer(N, K, group, True, K)
    for M in (1, 5, 12, 24):
        x = (1 + torch.randn(M, K, device=DEV, generator=_gen(M))).to(BF)  # a mean: zero points matter
        y = torch.empty(M, N, dtype=F32, device=DEV)
        layer.gemv_into(x, y)
        _check(layer, w, x, y)


def test_int4_gemv_strided_rows_and_their_surroundings():
    layer, w = _layer(50, 256, 64, False, 4)
    big = torch.full((7, 400), float("nan"), dtype=BF, device=DEV)
    x = big[:, 8:264]
    x.copy_(torch.randn(7, 256, device=DEV, generator=_gen(1)))
    out = torch.full((9, 64), 5.0, dtype=F32, device=DEV)
    y = out[1:8, 3:53]
    layer.gemv_into(x, y)
    _check(layer, w, x, y)
    out[1:8, 3:53] = 5.0
    assert bool((out == 5.0).all())  # nothing else was written


def test_int4_weights_written_just_before_the_call():
    N, K, M = 4096, 2048, 3
    one, other = _layer(N, K, 128, True, 21)[0], _layer(N, K, 128, True, 22)[0]
    layer = _layer(N, K, 128, True, 23)[0]
    x = torch.randn(M, K, device=DEV, generator=_gen(2)).to(BF)
    want = [torch.empty(M, N, device=DEV) for _ in range(2)]
    one.gemv_into(x, want[0])
    other.gemv_into(x, want[1])
    got = [torch.empty(M, N, device=DEV) for _ in range(40)]
    for i, y in enumerate(got):
        for name in ("packed", "zeros", "scales"):
            getattr(layer, name).copy_(getattr((one, other)[i % 2], name))
        layer.gemv_into(x, y)
    assert all(torch.equal(y, want[i % 2]) for i, y in enumerate(got))


def test_int4_infinities_and_nan_stay_in_their_token():
    layer, w = _layer(64, 256, 32, True, 9)
    x = torch.randn(5, 256, device=DEV, generator=_gen(2)).to(BF)
    x[1, 7], x[3, 200] = float("nan"), float("inf")
    y = torch.empty(5, 64, dtype=F32, device=DEV)
    layer.gemv_into(x, y)
    _check(layer, w, x[::2], y[::2])
    assert bool(y[1].isnan().all())
    assert not bool(y[3].isfinite().any())


@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True)])
def test_int4_dequant_equals_its_definition(group, zeros):
    layer, w = _layer(37, 384, group, zeros, 3)
    assert torch.equal(layer.reconstruct_weight(F32).double(), w)  # 15 * 2^11 * scale fits fp32
    assert torch.equal(layer.reconstruct_weight(BF), w.float().to(BF))
    assert torch.equal(layer.reconstruct_weight(HF), w.float().to(HF))


@pytest.mark.parametrize("zero_points", [False, True])
def test_int4_from_dense_is_within_half_a_step(zero_points):
    g = _gen(8)
    w = torch.randn(300, 512, device=DEV, generator=g) * 0.02
    w[5] = 0.0
    w[6, :128] = 0.5 + 0.1 * torch.rand(128, device=DEV, generator=g)  # a group without a sign change
    layer = Int4Linear.from_dense(w.to(BF), 128, zero_points=zero_points)
    _, scale, _ = quantize_int4(w.to(BF), 128, zero_points=zero_points)
    step = scale.double().repeat_interleave(128, 1)
    err = (layer.reconstruct_weight(F32).double() - w.to(BF).double()).abs()
    # half a step inside the range; the symmetric range ends at 7 of 7.5 steps, and both lose what the rounding of
    # the scale (2^-11) and of the zero point (half a step) move the range's ends
    assert bool((err <= step * (0.5 + (0.5 if zero_points else 0.0) + 16 * 2.0 ** -11) + 1e-30).all())
    x = torch.randn(2, 3, 512, device=DEV, generator=g).to(BF)
    y = layer(x)
    assert y.shape == (2, 3, 300)
    _check(layer, layer.reconstruct_weight(F32).double(), x.view(6, 512), y.view(6, 300))
    assert torch.equal(layer(x.transpose(0, 1)), y.transpose(0, 1))
    assert layer(x[:0]).shape == (0, 3, 300)


def test_int4_on_another_stream_and_captured():
    layer, w = _layer(200, 512, 128, False, 6)
    x = torch.randn(4, 512, device=DEV, generator=_gen(5)).to(BF)
    y = torch.empty(4, 200, dtype=BF, device=DEV)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        layer.gemv_into(x, y)
    s.synchronize()
    _check(layer, w, x, y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.gemv_into(x, y)
    x.copy_(torch.randn(4, 512, device=DEV, generator=_gen(15)))
    y.zero_()
    graph.replay()
    _check(layer, w, x, y)


def test_int4_refusals():
    layer, _ = _layer(16, 128, 64, False, 1)
    x, y = torch.zeros(2, 128, dtype=BF, device=DEV), torch.zeros(2, 16, dtype=BF, device=DEV)
    for bad_x, bad_y in ((x.float(), y), (x[:, :64], y), (x.cpu(), y), (x, y.cpu()), (x, y[:1]), (x, y.double()),
                         (x.t().contiguous().t(), y), (x[0], y)):
        with pytest.raises(ValueError):
            layer.gemv_into(bad_x, bad_y)
    wide = torch.zeros(2, 132, dtype=BF, device=DEV)
    with pytest.raises(ValueError):
        layer.gemv_into(wide[:, 1:129], y)  # rows that are not 16-byte aligned
    assert layer(wide[:, 1:129]).shape == (2, 16)  # the module copies them
    with pytest.raises(ValueError):
        layer(torch.zeros(2, 127, dtype=BF, device=DEV))
    layer.gemv_into(x[:0], y[:0])
