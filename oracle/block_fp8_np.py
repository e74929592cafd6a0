"""Matrices in 8 bits with a float32 scale for each block of 128, and their products in float64
(numpy). No counterpart in the reference."""
import numpy as np

BLOCK, E4M3_MAX, TINY = 128, 448.0, 2.0 ** -100


def to_e4m3(v):
    """float64 values rounded to the nearest e4m3 value, even ones on ties; |v| < 464."""
    v = np.asarray(v, np.float64)
    _, e = np.frexp(np.abs(v))
    step = np.exp2(np.maximum(e - 1, -6) - 3.0)
    return np.rint(v / step) * step


def quantize(x, rows=1):
    """x (R, C) float32 in blocks of rows x 128: (code values (R, C padded), scales), scales
    (ceil(R / rows), ceil(C / 128)) float32. Finite x."""
    x = np.asarray(x, np.float32)
    R, C = x.shape
    p = np.zeros((R + -R % rows, C + -C % BLOCK), np.float32)
    p[:R, :C] = x
    b = p.reshape(p.shape[0] // rows, rows, -1, BLOCK)
    top = np.abs(b).max((1, 3))
    some = top > np.float32(TINY)
    safe = np.where(some, top, np.float32(1))
    scale = np.where(some, safe / np.float32(E4M3_MAX), np.float32(0)).astype(np.float32)
    inv = np.where(some, np.float32(E4M3_MAX) / safe, np.float32(0)).astype(np.float32)
    prod = (b * inv[:, None, :, None]).astype(np.float32)
    return to_e4m3(prod).reshape(p.shape)[:R], scale


def values(codes, scales):
    """float64 values of code values (rows, cols padded) and scales of each row or 128 rows."""
    codes = np.asarray(codes, np.float64)
    s = np.asarray(scales, np.float64)
    if s.shape[0] != codes.shape[0]:
        s = np.repeat(s, BLOCK, 0)[:codes.shape[0]]
    return codes * np.repeat(s, BLOCK, 1)


def rounded(x, rows=1):
    """The float64 values that quantised x stands for."""
    c, s = quantize(x, rows)
    if rows > 1:
        return values(c, np.repeat(s, rows, 0)[:c.shape[0]])[:, :x.shape[1]]
    return values(c, s)[:, :x.shape[1]]


def matmul(x, w, dy=None):
    """y = q(x) q(w) with its terms' magnitudes, and with dy the gradients and theirs."""
    xv, wv = rounded(x), rounded(w, BLOCK)
    out = {"y": xv @ wv, "y_mag": np.abs(xv) @ np.abs(wv)}
    if dy is not None:
        d, xt, dt = rounded(dy), rounded(x.T), rounded(dy.T)
        out.update(dx=d @ wv.T, dx_mag=np.abs(d) @ np.abs(wv.T), dw=xt @ dt.T, dw_mag=np.abs(xt) @ np.abs(dt.T))
    return out
