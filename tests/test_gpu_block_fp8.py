"""The 8-bit block products on the GPU against the oracle (oracle/block_fp8_np.py).

Codes and scales are equal. Products: a float32 evaluation of n rounded steps is off by at most
n 2^-24 times the sum of its terms' magnitudes; a block's 128 products are exact and added in
128 steps at most, blocks and slices follow in one step each, and the scale adds two: 132 + 2
blocks. Results stored in bfloat16 add half a step, 2^-8 of themselves, and are made by the 8-bit
matrix instruction, which cuts each product at 2^-13 of the largest of the (at most) 16 that it
adds together (measured: a product of 2^-13 of its neighbour counts, one of 2^-14 does not). The
largest is no more than the sum of the 16 magnitudes, so a group loses at most 16 2^-13 of its
magnitudes' sum, and so does the whole: 2^-9 = 2^15 steps of 2^-24 (random terms: 2^-18)."""
import math

import numpy as np
import pytest
import torch

from oracle import block_fp8_np as bf
from test_gpu_train_ops import DTYPES, dtypes, f64, near

pytestmark = pytest.mark.gpu


def steps(K, dtype=torch.float32):
    return 132 + 2 * -(-K // 128) + (2 ** 15 if dtype == torch.bfloat16 else 0)


def values(shape, dtype, seed, wide=0.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g)
    if wide:
        x = x * torch.exp(wide * torch.randn(*shape[:-1], 1, generator=g))
    return x.to(dtype)


def same_quantised(pkg, q, x, rows):
    c, s = bf.quantize(f64(x), rows)
    assert q.cols == x.shape[1] and q.codes.dtype == torch.float8_e4m3fn
    assert q.codes.shape == c.shape and q.scales.shape == s.shape
    assert np.array_equal(f64(q.codes.float()), c)
    assert np.array_equal(q.scales.cpu().numpy(), s)
    assert np.allclose(f64(pkg.fp8_dequantize(q)), bf.rounded(f64(x), rows), rtol=2.0 ** -23, atol=0)


@dtypes
@pytest.mark.parametrize("R,C", [(1, 1), (1, 1536), (3, 127), (128, 128), (129, 257), (300, 1001), (127, 640),
                                 (1000, 8), (5, 4097)])
def test_quantize(pkg, dev, R, C, dtype):
    x = values((R, C), dtype, R + C, 3.0).to(dev)
    for tiles in (False, True):
        same_quantised(pkg, pkg.fp8_quantize(x, tiles), x, 128 if tiles else 1)
        same_quantised(pkg, pkg.fp8_quantize(x, tiles, True), x.t(), 128 if tiles else 1)


def test_quantize_strides_and_sizes_of_values(pkg, dev):
    wide = values((200, 400), torch.float32, 1, 2.0).to(dev)
    for dt in DTYPES.values():
        w = wide.to(dt)
        for x in (w[:, 3:259], w[::3, :130], w.t(), w[:1].expand(140, 400), w[:, ::2], w[5:6, 7:]):
            same_quantised(pkg, pkg.fp8_quantize(x), x, 1)
            same_quantised(pkg, pkg.fp8_quantize(x, True, True), x.t(), 128)
    # blocks of zeros, of magnitudes that are stored as zeros, of fp32's ends; every code's neighbourhood
    x = torch.zeros(140, 384)
    x[1] = 1e-31
    x[2] = 2.0 ** -100
    x[3, :200] = torch.nextafter(torch.tensor(2.0 ** -100), torch.tensor(1.0))
    x[4] = 3.4e38 * torch.linspace(-1, 1, 384)
    x[5, 0] = 448
    x[5, 1:128] = torch.arange(1, 128, dtype=torch.uint8).view(torch.float8_e4m3fn).float().nan_to_num(1) * (1 + 2.0 ** -5)
    x[6, 0], x[6, 1:255] = 448, torch.linspace(0, 2.0 ** -7, 254)
    x[7:] = values((133, 384), torch.float32, 5, 8.0)
    x = x.to(dev)
    for tiles in (False, True):
        same_quantised(pkg, pkg.fp8_quantize(x, tiles), x, 128 if tiles else 1)
        same_quantised(pkg, pkg.fp8_quantize(x, tiles, True), x.t(), 128 if tiles else 1)
    assert pkg.fp8_quantize(x[:0]).codes.shape == (0, 384)


def test_not_finite(pkg, dev):
    """A block with an infinity or a NaN stands for values that are not finite, and only it."""
    for bad in (math.inf, -math.inf, math.nan):
        x = values((70, 300), torch.float32, 1).to(dev)
        x[3, 140] = bad
        v = f64(pkg.fp8_dequantize(pkg.fp8_quantize(x)))
        assert not np.isfinite(v[3, 128:256]).all() and not np.isfinite(v[3, 140])
        v[3, 128:256] = 0
        assert np.isfinite(v).all()
        w = values((300, 40), torch.float32, 2).to(dev)
        for M in (70, 20):
            y = f64(pkg.fp8_matmul(x[:M], w))
            assert not np.isfinite(y[3]).any()
            assert np.isfinite(np.delete(y, 3, 0)).all()


SIZES = [(1, 1, 1), (1, 1536, 6144), (2, 100, 33), (31, 1000, 70), (32, 128, 256), (33, 129, 127), (64, 4608, 96),
         (128, 128, 128), (200, 768, 300), (257, 65, 513), (1000, 1537, 131), (2048, 256, 768), (5003, 200, 64)]


@dtypes
@pytest.mark.parametrize("M,K,N", SIZES)
def test_block_matmul(pkg, dev, M, K, N, dtype):
    """Every pair of operands: scales of rows or tiles on both sides, codes or values."""
    x, w = values((M, K), dtype, M + K, 1.0).to(dev), values((N, K), dtype, N, 1.0).to(dev)
    xv = {1: bf.rounded(f64(x)), 128: bf.rounded(f64(x), 128)}
    wv = {1: bf.rounded(f64(w)), 128: bf.rounded(f64(w), 128)}
    for tw in (128, 1):
        b = pkg.fp8_quantize(w, tw == 128)
        for ta in (1, 128):
            want, mag = xv[ta] @ wv[tw].T, np.abs(xv[ta]) @ np.abs(wv[tw].T)
            y = pkg.fp8_block_matmul(pkg.fp8_quantize(x, ta == 128), b, dtype)
            assert y.shape == (M, N) and y.dtype == dtype
            near(y, want, mag, steps(K, dtype), (ta, tw))
            if ta == 1:
                near(pkg.fp8_block_matmul(x, b), want, mag, steps(K, dtype), "values")
                near(pkg.fp8_block_matmul(x, b, torch.float32), want, mag, steps(K), "values, fp32")


@dtypes
@pytest.mark.parametrize("M,K,N", [(1, 65536, 40), (1, 65537, 3), (7, 4608, 130), (16, 4096, 65), (17, 4000, 64),
                                   (32, 2048, 31), (32, 2049, 31), (3, 1537, 1000)])
def test_few_rows_of_values(pkg, dev, M, K, N, dtype):
    """Values on both sides of what a launch quantises itself (512 blocks): the products of their
    codes, whose order of sums is the same, bit for bit; rows apart and at any element."""
    x, w = values((M, K), dtype, M + K, 1.0).to(dev), values((N, K), dtype, N, 1.0).to(dev)
    wide = torch.zeros(M, K + 9, dtype=dtype, device=dev)
    wide[:, 3:K + 3] = x
    for tiles in (False, True):
        b = pkg.fp8_quantize(w, tiles)
        for out in DTYPES.values():
            want = pkg.fp8_block_matmul(pkg.fp8_quantize(x), b, out)
            assert torch.equal(pkg.fp8_block_matmul(x, b, out), want)
            assert torch.equal(pkg.fp8_block_matmul(wide[:, 3:K + 3], b, out), want)
    v, u = bf.rounded(f64(x)), f64(pkg.fp8_dequantize(b))
    near(want, v @ u.T, np.abs(v) @ np.abs(u).T, steps(K, want.dtype))


@pytest.mark.parametrize("M,K,N,slices", [(2040, 1100, 8100, 1), (130, 9000, 140, 15), (400, 2050, 700, 6)])
def test_forms(pkg, dev, M, K, N, slices):
    """Tiles of 256 x 256 with ragged edges, and sliced sums, against float64."""
    x, w = values((M, K), torch.bfloat16, 1, 1.0).to(dev), values((N, K), torch.bfloat16, 2, 1.0).to(dev)
    a, b = pkg.fp8_quantize(x), pkg.fp8_quantize(w, True)
    need = pkg._lib.lib().tmoe_fp8_gemm_workspace_bytes(M, N, K, pkg._lib.TMOE_BF16, 0)
    assert (need == 0) == (slices == 1) and need >= 4 * M * N * (slices if slices > 1 else 0)
    v, u = pkg.fp8_dequantize(a).double(), pkg.fp8_dequantize(b).double()
    near(pkg.fp8_block_matmul(a, b), f64(v @ u.t()), f64(v.abs() @ u.abs().t()), steps(K, torch.bfloat16) + 16)


def test_operands_as_they_lie(pkg, dev):
    """Rows of codes apart, unaligned or every other; scales in any order, one for all; uint8."""
    M, N, K = 70, 90, 300
    x, w = values((M, K), torch.float32, 1).to(dev), values((N, K), torch.float32, 2).to(dev)
    a, b = pkg.fp8_quantize(x), pkg.fp8_quantize(w, True)
    want = pkg.fp8_block_matmul(a, b, torch.float32)
    big = torch.zeros(N, 500, dtype=torch.uint8, device=dev)
    for off, codes in ((0, big[:, :384]), (16, big[:, 16:400]), (5, big[:, 5:389])):
        big.zero_()
        codes.copy_(b.codes.view(torch.uint8))
        for s in (b.scales, b.scales.t().contiguous().t()):
            got = pkg.fp8_block_matmul(a, pkg.BlockFp8(codes, s, K), torch.float32)
            assert torch.equal(got, want), off
    half = pkg.BlockFp8(a.codes[::2], a.scales[::2], K)
    assert torch.equal(pkg.fp8_block_matmul(half, b, torch.float32), want[::2])
    one = pkg.BlockFp8(a.codes, torch.ones(1, 1, device=dev).expand(M, 3), K)
    near(pkg.fp8_block_matmul(one, b, torch.float32), f64(a.codes.float())[:, :K] @ f64(pkg.fp8_dequantize(b)).T,
         np.abs(f64(a.codes.float())[:, :K]) @ np.abs(f64(pkg.fp8_dequantize(b)).T), steps(K))
    deep = x.view(7, 10, K)
    assert torch.equal(pkg.fp8_block_matmul(deep, b), want.view(7, 10, N))
    assert torch.equal(pkg.fp8_block_matmul(x[0], b), pkg.fp8_block_matmul(x[:1], b)[0])
    assert pkg.fp8_block_matmul(x[:0], b).shape == (0, N)
    assert pkg.fp8_block_matmul(pkg.fp8_quantize(x[:0]), b).shape == (0, N)


@dtypes
@pytest.mark.parametrize("M,K,N", SIZES)
def test_matmul_and_gradients(pkg, dev, M, K, N, dtype):
    x, w, dy = (values(s, dtype, sum(s), 1.0) for s in ((M, K), (K, N), (M, N)))
    o = bf.matmul(f64(x), f64(w), f64(dy))
    xl, wl = x.to(dev).requires_grad_(), w.to(dev).requires_grad_()
    y = pkg.fp8_matmul(xl, wl)
    dx, dw = torch.autograd.grad(y, (xl, wl), dy.to(dev))
    assert y.dtype == dx.dtype == dw.dtype == dtype
    near(y, o["y"], o["y_mag"], steps(K, dtype), "y")
    near(dx, o["dx"], o["dx_mag"], steps(N, dtype), "dx")
    near(dw, o["dw"], o["dw_mag"], steps(M, dtype), "dw")
    for got, name in ((y, "y"), (dx, "dx"), (dw, "dw")):    # and no more than a rounding in the whole
        off = np.linalg.norm(f64(got) - o[name])
        assert off <= (2.0 ** -8 + 2.0 ** -14 if dtype == torch.bfloat16 else 2.0 ** -20) * np.linalg.norm(o[name]), name
    # one gradient alone, and none
    y2 = pkg.fp8_matmul(xl, wl.detach())
    d2, = torch.autograd.grad(y2, xl, dy.to(dev))
    near(d2, o["dx"], o["dx_mag"], steps(N, dtype), "dx alone")
    d3, = torch.autograd.grad(pkg.fp8_matmul(xl.detach(), wl), wl, dy.to(dev))
    assert torch.equal(d3, dw)
    with torch.no_grad():
        y4 = pkg.fp8_matmul(xl, wl)
    assert not y4.requires_grad
    near(y4, o["y"], o["y_mag"], steps(K, dtype), "y without gradients")


@dtypes
def test_one_gradient_of_two(pkg, dev, dtype):
    """What is asked of a product that kept both operands, one at a time and again: the same bits."""
    x, w = (values(s, dtype, sum(s)).to(dev).requires_grad_() for s in ((150, 200), (200, 70)))
    dy = values((150, 70), dtype, 3).to(dev)
    y = pkg.fp8_matmul(x, w)
    both = torch.autograd.grad(y, (x, w), dy, retain_graph=True)
    for leaf, want in zip((x, w), both):
        got, = torch.autograd.grad(y, leaf, dy, retain_graph=True)
        assert torch.equal(got, want)
    (y * dy).sum().backward()
    assert torch.equal(x.grad, both[0]) and torch.equal(w.grad, both[1])
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, x, dy)


def test_matmul_views(pkg, dev):
    """Leading axes, strided and expanded operands and gradients, no tokens."""
    x, w = values((6, 11, 200), torch.float32, 1).to(dev).requires_grad_(), values((300, 200), torch.float32, 2).to(dev)
    wt = w.t().requires_grad_()
    y = pkg.fp8_matmul(x, wt)
    assert y.shape == (6, 11, 300)
    dx, dw = torch.autograd.grad(y.sum(1).sum(), (x, wt))
    o = bf.matmul(f64(x).reshape(66, 200), f64(wt), np.ones((66, 300)))
    near(dx.reshape(66, 200), o["dx"], o["dx_mag"], steps(300))
    near(dw, o["dw"], o["dw_mag"], steps(66))
    e = torch.empty(0, 200, device=dev, requires_grad=True)
    y = pkg.fp8_matmul(e, wt)
    dx, dw = torch.autograd.grad(y.sum(), (e, wt))
    assert y.shape == (0, 300) and dx.shape == (0, 200) and (dw == 0).all() and dw.shape == wt.shape
    v = pkg.fp8_matmul(x[0, 0], wt)
    assert v.shape == (300,)


def test_second_derivative_is_refused(pkg, dev):
    x = values((8, 64), torch.float32, 1).to(dev).requires_grad_()
    w = values((64, 8), torch.float32, 1).to(dev).requires_grad_()
    d, = torch.autograd.grad(pkg.fp8_matmul(x, w).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        d.sum().backward()


def test_captured_and_streams(pkg, dev):
    """Captured passes that share a pool, replayed on new values with eager calls in between; other
    streams; the same bits each time."""
    K, N = 640, 300
    w = values((K, N), torch.bfloat16, 1).to(dev).requires_grad_()
    for M in (20, 1500):
        x = values((M, K), torch.bfloat16, 2).to(dev).requires_grad_()
        dy = values((M, N), torch.bfloat16, 3).to(dev)

        def step(v):
            y = pkg.fp8_matmul(v, w)
            return (y, *torch.autograd.grad(y, (v, w), dy))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(x)
        torch.cuda.current_stream().wait_stream(side)
        first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(first):
            a = step(x)
        with torch.cuda.graph(second, pool=first.pool()):
            b = step(x)
        for seed in range(4):
            new = values((M, K), torch.bfloat16, 10 + seed).to(dev)
            with torch.no_grad():
                x.copy_(new)
            first.replay()
            got = [t.clone() for t in a]
            second.replay()
            want = step(new.requires_grad_())
            torch.cuda.synchronize()
            for p, q, r in zip(got, want, b):
                assert torch.equal(p, q) and torch.equal(r, q)
        with torch.cuda.stream(side):
            other = step(new)
        side.synchronize()
        for p, q in zip(other, want):
            assert torch.equal(p, q)


@pytest.mark.parametrize("M,K,N", [(2040, 1100, 8100), (4096, 1024, 4096), (2049, 129, 8200)])
def test_wide_tiles_in_the_whole(pkg, dev, M, K, N):
    """bfloat16 results of tiles of 256 x 256 are no more than their own rounding off in each row's and
    each column's norm. What the 8-bit instruction cuts is, for terms without an order, 2^-18 of their
    magnitudes' sum, which is sqrt(K) at most times their own root of squares: 2^-18 sqrt(K) < 2^-12."""
    x, w = values((M, K), torch.bfloat16, 3).to(dev), values((N, K), torch.bfloat16, 4).to(dev)
    a, b = pkg.fp8_quantize(x), pkg.fp8_quantize(w, True)
    assert pkg._lib.lib().tmoe_fp8_gemm_workspace_bytes(M, N, K, pkg._lib.TMOE_BF16, 0) == 0
    want = pkg.fp8_dequantize(a).double() @ pkg.fp8_dequantize(b).double().t().contiguous()
    got = pkg.fp8_block_matmul(a, b)
    off = got.double() - want
    exact = pkg.fp8_block_matmul(a, b, torch.float32).double()
    for axis in (0, 1):
        size = want.norm(dim=axis)
        assert (off.norm(dim=axis) <= (2.0 ** -8 + 2.0 ** -12) * size).all()
        assert ((exact - want).norm(dim=axis) <= 2.0 ** -20 * size).all()
