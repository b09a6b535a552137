"""The 8-bit product with fp32 output on a real MI355X, against float64.

Tolerances: a bf16 MFMA adds 32 products, each of them exact, to its accumulator within 2^-22 of the sum of all magnitudes
(measured over all pairs of e4m3 values); ldexp is exact; the addition to the total, and the bias, round by 2^-24 of the
value.  With n = ceil(K / 128) blocks of four MFMAs an element is off by at most (4 + 1) n + 1 times 2^-22 of the sum of its
magnitudes.  In the 2-norm these errors are independent: an MFMA's is 2^-22 of the magnitudes of 32 products, about
0.64 sqrt(32) = 3.6 of their sum's size, and the n blocks add up like the sums themselves; the total rounds n times, by
2^-24 of at most its size.
"""
import math

import pytest
import torch

from test_gpu_fp8 import BLK, widen

pytestmark = pytest.mark.gpu


def operands(dev, M, N, K):
    from src import ops
    g = torch.Generator(device=dev).manual_seed(M + 3 * N + 7 * K)
    x = torch.randn(M, K, generator=g, device=dev) * torch.exp(2 * torch.randn(M, 1, generator=g, device=dev))
    x = x * torch.exp(torch.randn(1, K, generator=g, device=dev))
    w = torch.randn(N, K, generator=g, device=dev) * torch.exp(torch.randn(N, 1, generator=g, device=dev))
    return (*ops.quantize_fp8(x), *ops.quantize_fp8_weight(w), torch.randn(N, generator=g, device=dev))


def check(y, xq, xs, wq, ws, bias):
    K = xq.shape[1]
    a, b = widen(xq, xs, 1), widen(wq, ws, BLK)
    want = a @ b.t().contiguous()
    mag = a.abs() @ b.abs().t().contiguous()
    if bias is not None:
        want, mag = want + bias.double(), mag + bias.double().abs()
    n = -(-K // BLK)
    assert y.dtype == torch.float32 and y.shape == want.shape
    err = (y.double() - want).abs()
    assert bool((err <= (5 * n + 1) * 2.0 ** -22 * mag).all())
    if want.numel() >= 256:      # (a mean)
        assert float(err.norm() / want.norm()) < 2.0 ** -22 * (4 + math.sqrt(n))


@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 16, 128), (2, 5, 17), (16, 48, 200), (17, 130, 127), (32, 2304, 768),
                                   (33, 129, 1000), (64, 64, 129), (100, 257, 384), (128, 128, 128), (129, 300, 2049),
                                   (256, 256, 256), (257, 511, 640), (300, 1000, 272), (513, 384, 1664), (777, 3001, 768),
                                   (3001, 2300, 400), (300, 1001, 16500), (20, 300, 8330), (2999, 2177, 8330), (1, 700, 5632)])
def test_fp32_product(dev, M, N, K):
    from src import ops
    xq, xs, wq, ws, bias = operands(dev, M, N, K)
    check(ops.fp8_matmul(xq, xs, wq, ws, bias=bias, out_dtype=torch.float32), xq, xs, wq, ws, bias)
    check(ops.fp8_matmul(xq, xs, wq, ws, out_dtype=torch.float32), xq, xs, wq, ws, None)


@pytest.mark.parametrize("M,N,K,ldc", [(20, 300, 256, 301), (300, 1000, 272, 1001), (3001, 2300, 400, 2303), (130, 200, 256, 256)])
def test_c_entry_writes_only_its_elements(dev, M, N, K, ldc):
    """Output rows of an odd stride at an odd element, and nothing written between or behind the rows."""
    from src import _native as N_
    xq, xs, wq, ws, bias = operands(dev, M, N, K)
    for first in (1, 4):
        buf = torch.full((first + (M + 130) * ldc,), 777.0, device=dev)
        rc = N_.lib().ldm_gemm_fp8_f32(M, N, K, xq.data_ptr(), xq.stride(0), xs.data_ptr(), xs.stride(0), wq.data_ptr(),
                                       wq.stride(0), ws.data_ptr(), ws.stride(0), bias.data_ptr(), buf.data_ptr() + 4 * first, ldc,
                                       N_.stream())
        torch.cuda.synchronize()
        assert rc == 0
        got = buf[first:].view(M + 130, ldc)
        assert bool((got[:, N:] == 777).all()) and bool((buf[:first] == 777).all()) and bool((got[M:] == 777).all())
        check(got[:M, :N], xq, xs, wq, ws, bias)


@pytest.mark.parametrize("M,N,K", [(5, 33, 40), (130, 140, 200), (300, 300, 392)])
def test_ignores_what_lies_behind_the_last_column(dev, M, N, K):
    """Rows whose memory behind column K holds the e4m3 NaN (both operands), rows behind the last one likewise."""
    from src import ops
    xq0, xs, wq0, ws, _ = operands(dev, M, N, K)
    ld = -(-K // 16) * 16 + 32
    xb = torch.full((M + 2, ld), 0x7f, dtype=torch.uint8, device=dev)
    wb = torch.full((N + 2, ld), 0x7f, dtype=torch.uint8, device=dev)
    xb[:M, :K] = xq0.view(torch.uint8)
    wb[:N, :K] = wq0.view(torch.uint8)
    xq, wq = xb.view(torch.float8_e4m3fn)[:M, :K], wb.view(torch.float8_e4m3fn)[:N, :K]
    check(ops.fp8_matmul(xq, xs, wq, ws, out_dtype=torch.float32), xq0, xs, wq0, ws, None)


@pytest.mark.parametrize("M,N", [(3, 40), (200, 300)])
def test_scale_codes_of_the_whole_range(dev, M, N):
    """Powers outside fp32 whose products are inside it, the NaN code, NaN values, zeros."""
    from src import ops

    def code(v, *shape):
        return torch.full(shape, v, dtype=torch.uint8, device=dev).view(torch.float8_e8m0fnu)

    def product(value, ca, cb):
        x = torch.full((M, 256), 0.0, device=dev)
        w = torch.full((N, 256), 0.0, device=dev)
        x[:, 130] = w[:, 130] = value
        return ops.fp8_matmul(x.to(torch.float8_e4m3fn), code(ca, M, 2), w.to(torch.float8_e4m3fn), code(cb, -(-N // 128), 2),
                              out_dtype=torch.float32)
    assert bool((product(2.0 ** -9, 254, 140) == 2.0 ** 122).all())       # 2^140 alone would be infinite, and 0 of it NaN
    assert bool((product(448.0, 1, 103) == 448.0 ** 2 * 2.0 ** -150).all())
    assert bool((product(0.0, 254, 254) == 0).all())
    assert bool((product(1.0, 254, 254) == math.inf).all())
    assert bool((product(1.0, 0, 0) == 0).all())
    assert bool(product(1.0, 255, 100).isnan().all()) and bool(product(0.0, 100, 255).isnan().all())
    xq, xs, wq, ws, _ = operands(dev, M, N, 256)
    x = xq.float()
    x[1, 200] = math.nan
    y = ops.fp8_matmul(x.to(torch.float8_e4m3fn), xs, wq, ws, out_dtype=torch.float32)
    keep = [i for i in range(M) if i != 1]
    assert bool(y[1].isnan().all())
    check(y[keep], xq[keep], xs[keep], wq, ws, None)


@torch.no_grad()
def test_linear_in_fp32_shapes_streams_and_graph(dev):
    from src import ops
    lin = torch.nn.Linear(192, 500).to(dev)
    pack = ops.Fp8Weights([lin.weight], [lin.bias])
    x = torch.randn(2, 3, 7, 192, device=dev).bfloat16()
    y = ops.fp8_linear(x, pack, out_dtype=torch.float32)
    assert y.shape == (2, 3, 7, 500) and y.dtype == torch.float32
    xq, xs = ops.quantize_fp8(x.view(42, 192))
    check(y.reshape(42, 500), xq, xs, *pack.get()[:2], lin.bias)
    # the bf16 output is the same product, its truncation (1.5e-5 of the largest of eight) and one rounding away
    y16 = ops.fp8_linear(x, pack)
    assert float((y16.double() - y.double()).norm() / y.double().norm()) < 2.0 ** -8
    assert ops.fp8_linear(x[0, 0, 0], pack, out_dtype=torch.float32).shape == (500,)
    assert ops.fp8_linear(x[:0], pack, out_dtype=torch.float32).shape == (0, 3, 7, 500)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        z = ops.fp8_linear(x, pack, out_dtype=torch.float32)
    torch.cuda.synchronize()
    assert torch.equal(z, y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        z = ops.fp8_linear(x, pack, out_dtype=torch.float32)
    for i in range(3):
        x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(i)).to(dev))
        want = ops.fp8_linear(x, pack, out_dtype=torch.float32)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(z, want)
