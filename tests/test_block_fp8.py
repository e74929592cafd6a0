"""The 8-bit block products on the CPU: the oracle (oracle/block_fp8_np.py) against torch's
conversions and closed forms, and the refusals of the C ABI and of the Python entry points (none
reaches a GPU)."""
import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import block_fp8_np as bf


def test_e4m3_is_torchs():
    v = torch.cat([torch.linspace(-463, 463, 20001), torch.linspace(-0.05, 0.05, 4001),
                   torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float().nan_to_num(0),
                   torch.tensor([17.0, 19.0, 2 ** -10, 3 * 2 ** -10, -2 ** -10, 2 ** -9 * 7.5])])
    assert np.array_equal(bf.to_e4m3(v.numpy()), v.to(torch.float8_e4m3fn).double().numpy())


@pytest.mark.parametrize("rows", [1, 128])
def test_quantize_oracle(rows):
    g = np.random.default_rng(rows)
    x = (g.normal(size=(200, 300)) * np.exp(g.normal(size=(200, 1)) * 4)).astype(np.float32)
    x[:, 128:256] *= 1e-36
    x[3] = 0
    c, s = bf.quantize(x, rows)
    assert c.shape == (200, 384) and s.shape == (-(-200 // rows), 3) and (c[:, 300:] == 0).all()
    v = bf.rounded(x, rows)
    step = np.repeat(np.repeat(s, 128, 1)[:, :300], rows, 0)[:200]
    # half a step of the code, and the two roundings before it
    tol = np.maximum(np.abs(x) * 2.0 ** -4, step * 2.0 ** -10) * (1 + 2.0 ** -20)
    assert np.all(np.abs(v - x) <= tol + (step == 0) * bf.TINY)
    assert np.abs(c).max() == 448


def test_matmul_oracle_is_the_product():
    g = np.random.default_rng(0)
    x, w, dy = (g.normal(size=s).astype(np.float32) for s in ((50, 200), (200, 70), (50, 70)))
    o = bf.matmul(x, w, dy)
    for got, want in ((o["y"], x @ w), (o["dx"], dy @ w.T), (o["dw"], x.T @ dy)):
        assert np.linalg.norm(got - want) < 0.06 * np.linalg.norm(want)


def _op(pkg, **kw):
    t = pkg._lib.TmoeFp8Operand()
    for k, v in dict(dict(codes=64, scales=64, rows=64, row_bytes=256, scale_row=1, scale_block=64, tiles=0),
                     **kw).items():
        setattr(t, k, v)
    return t


BAD = [(dict(rows=-1), -1), (dict(rows=2 ** 23 + 1), -2), (dict(codes=0), -1), (dict(scales=0), -1),
       (dict(codes=72), -1), (dict(scales=66), -1), (dict(row_bytes=264), -1), (dict(row_bytes=128), -1),
       (dict(row_bytes=2 ** 24 + 16), -1), (dict(scale_row=-1), -1), (dict(scale_block=-1), -1)]


@pytest.mark.parametrize("kw,code", BAD)
def test_abi_refuses_operands(pkg, kw, code):
    L = pkg._lib.lib()
    good, bad = _op(pkg), _op(pkg, **kw)
    r = ctypes.byref
    assert L.tmoe_fp8_gemm(r(bad), r(good), 200, 0, 64, 64, 1 << 40, None) == code
    assert L.tmoe_fp8_gemm(r(good), r(bad), 200, 0, 64, 64, 1 << 40, None) == code
    assert L.tmoe_last_error().startswith(b"tmoe_fp8_gemm: ")
    assert L.tmoe_fp8_gemm_values(64, 64, 200, 0, r(bad), 200, 0, 64, 64, 1 << 40, None) == code
    R = bad.rows if bad.rows != 64 else 64
    if R > 0:
        assert L.tmoe_fp8_quantize(64, R, 200, 200, 0, r(bad), None, None) == code
        assert L.tmoe_fp8_quantize(64, 200, R, R, 0, None, r(bad), None) == code


def test_abi_refusals(pkg):
    L = pkg._lib.lib()
    r, a = ctypes.byref, _op(pkg)
    need = L.tmoe_fp8_gemm_workspace_bytes
    assert need(-1, 64, 64, 0, 0) == need(4, 0, 64, 0, 0) == need(4, 64, 0, 0, 0) == need(2 ** 23 + 1, 1, 1, 0, 1) == 0
    assert need(64, 64, 64, 2, 1) == 0
    assert need(16, 64, 300, 0, 1) == 0 and need(100, 64, 300, 0, 1) >= 100 * 384 + 100 * 12
    assert L.tmoe_fp8_gemm(None, r(a), 200, 0, 64, 64, 1 << 40, None) == -1
    assert L.tmoe_fp8_gemm(r(a), None, 200, 0, 64, 64, 1 << 40, None) == -1
    for K, dt, out, ws, n, code in ((0, 0, 64, 64, 1 << 40, -1), (2 ** 23 + 1, 0, 64, 64, 1 << 40, -2),
                                    (200, 2, 64, 64, 1 << 40, -1), (200, 0, 0, 64, 1 << 40, -1),
                                    (200, 0, 72, 64, 1 << 40, -1), (200, 0, 64, 72, 1 << 40, -1)):
        assert L.tmoe_fp8_gemm(r(a), r(a), K, dt, out, ws, n, None) == code
        assert L.tmoe_fp8_gemm_values(64, 64, max(K, 200), 0, r(a), K, dt, out, ws, n, None) == code
    n = need(64, 64, 200, 0, 1)
    assert n > 0 and L.tmoe_fp8_gemm_values(64, 64, 200, 0, r(a), 200, 0, 64, 64, n - 1, None) == -1
    assert L.tmoe_fp8_gemm_values(64, 64, 200, 0, r(a), 200, 0, 64, 0, n, None) == -1
    big = _op(pkg, rows=64, row_bytes=4096)
    split = need(64, 64, 4096, 0, 0)
    assert split == 0 or L.tmoe_fp8_gemm(r(big), r(big), 4096, 0, 64, 64, split - 1, None) == -1
    for x, M, rs, dt, code in ((0, 64, 200, 0, -1), (65, 64, 200, 0, -1), (64, 64, 199, 0, -1), (64, 64, 200, 2, -1),
                               (64, -1, 200, 0, -1), (64, 2 ** 23 + 1, 200, 0, -2)):
        assert L.tmoe_fp8_gemm_values(x, M, rs, dt, r(a), 200, 0, 64, 64, 1 << 40, None) == code
    assert L.tmoe_fp8_gemm_values(0, 0, 0, 0, r(a), 200, 0, 0, 0, 0, None) == 0
    e = _op(pkg, rows=0, codes=0, scales=0)
    assert L.tmoe_fp8_gemm(r(e), r(a), 200, 0, 0, 0, 0, None) == 0
    assert L.tmoe_fp8_gemm(r(a), r(e), 200, 0, 64, 64, 1 << 40, None) == -1
    q = L.tmoe_fp8_quantize
    c, t = _op(pkg, rows=200), _op(pkg, tiles=1)
    assert q(64, 64, 200, 200, 0, None, None, None) == -1          # nothing wanted
    assert q(64, 64, 200, 200, 2, r(a), None, None) == -1
    assert q(64, -1, 200, 200, 0, r(a), None, None) == -1 and q(64, 64, 0, 200, 0, r(a), None, None) == -1
    assert q(0, 64, 200, 200, 0, r(a), None, None) == -1 and q(65, 64, 200, 200, 0, r(a), None, None) == -1
    assert q(64, 64, 200, 199, 0, r(a), None, None) == -1
    assert q(64, 64, 200, 200, 0, r(a), r(a), None) == -1          # cols of 64 rows for 200 columns
    assert q(64, 64, 200, 200, 0, r(t), r(c), None) == -1          # tiles in one
    tc = _op(pkg, rows=200, tiles=1)
    assert q(64, 64, 200, 200, 0, r(t), r(tc), None) == -1         # steps that are not exchanged
    assert q(0, 0, 200, 200, 0, r(a), None, None) == 0


def test_python_refusals(pkg):
    x, w = torch.zeros(4, 200), torch.zeros(200, 6)
    q = pkg.BlockFp8(torch.zeros(4, 256, dtype=torch.uint8), torch.zeros(4, 2), 200)
    for f, args, text in [
            (pkg.fp8_matmul, (x.double(), w.double()), "dtype"), (pkg.fp8_matmul, (x, w.bfloat16()), "dtypes"),
            (pkg.fp8_matmul, (x, w.t()), "expected"), (pkg.fp8_matmul, (x, w[:, :0]), "expected"),
            (pkg.fp8_matmul, (x[:, :0], w[:0]), "expected"), (pkg.fp8_matmul, (x, w[None]), "expected"),
            (pkg.fp8_matmul, (torch.zeros(()), w), "expected"), (pkg.fp8_matmul, (x, w), "HIP devices only"),
            (pkg.fp8_quantize, (x.double(),), "dtype"), (pkg.fp8_quantize, (x[0],), "expected"),
            (pkg.fp8_quantize, (x[:, :0],), "expected"), (pkg.fp8_quantize, (x.requires_grad_(),), "gradient"),
            (pkg.fp8_quantize, (x.detach(),), "HIP devices only"),
            (pkg.fp8_quantize, (x.detach()[:0], False, True), "no rows"),
            (pkg.fp8_block_matmul, (x.detach()[:, :100], q), "rows of 200"),
            (pkg.fp8_block_matmul, (x, q), "gradient"), (pkg.fp8_block_matmul, (x.detach(), q), "HIP devices only"),
            (pkg.fp8_block_matmul, (q, q), "HIP devices only"),
            (pkg.fp8_block_matmul, (q, q._replace(codes=q.codes[:0], scales=q.scales[:0])), "no rows"),
            (pkg.fp8_block_matmul, (q, q._replace(codes=q.codes[:, :128])), "codes"),
            (pkg.fp8_block_matmul, (q, q._replace(codes=q.codes.float())), "codes"),
            (pkg.fp8_block_matmul, (q, q._replace(scales=torch.zeros(4, 1))), "scales"),
            (pkg.fp8_block_matmul, (q, q._replace(scales=torch.zeros(3, 2))), "scales"),
            (pkg.fp8_block_matmul, (q, q._replace(scales=torch.zeros(4, 2, dtype=torch.float64))), "scales"),
            (pkg.fp8_block_matmul, (q, q._replace(scales=torch.zeros(4, 2, requires_grad=True))), "gradient"),
            (pkg.fp8_block_matmul, (q, q, torch.float16), "float16")]:
        with pytest.raises(RuntimeError, match=text):
            f(*args)
    with pytest.raises(ValueError, match="rows of"):
        pkg.fp8_block_matmul(q, q._replace(cols=199))
    with pytest.raises(TypeError):
        pkg.fp8_block_matmul(x.detach(), w)
    with torch.autograd.forward_ad.dual_level():
        d = torch.autograd.forward_ad.make_dual(x.detach(), x.detach() + 1)
        for f, args in ((pkg.fp8_matmul, (d, w)), (pkg.fp8_quantize, (d,)), (pkg.fp8_block_matmul, (d, q))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                f(*args)


def test_dequantize(pkg):
    g = np.random.default_rng(1)
    x = g.normal(size=(130, 140)).astype(np.float32)
    for rows in (1, 128):
        c, s = bf.quantize(x, rows)
        q = pkg.BlockFp8(torch.tensor(c).to(torch.float8_e4m3fn), torch.tensor(s), 140)
        assert np.allclose(pkg.fp8_dequantize(q).numpy(), bf.rounded(x, rows), rtol=1e-6)
        q = q._replace(codes=q.codes.view(torch.uint8))
        assert np.allclose(pkg.fp8_dequantize(q).numpy(), bf.rounded(x, rows), rtol=1e-6)
