"""float64 restatement of the training operators around the expert contraction, with the
gradients written out by hand: the router with its losses, the block norms, the AdamW step
and its 8-bit states. TEST INFRASTRUCTURE, only tests import it.

Beside each value a function returns what its error is measured by: the sum of the
magnitudes of the terms that it is made of (keys that end in "_mag"). A float32 evaluation
in n steps is off by at most n 2^-24 times that.
"""
from __future__ import annotations

import numpy as np


def _sig(g):
    with np.errstate(over="ignore"):
        return 1.0 / (1.0 + np.exp(-g))


# ---- router ---------------------------------------------------------------------

def router(raw, k, tau, cap=10.0, mask=None, dw=None, dlb=0.0, dz=0.0):
    raw = np.asarray(raw, np.float64)
    B, E = raw.shape
    on = np.ones(B, bool) if mask is None else np.asarray(mask, bool)
    raw = np.where(on[:, None], raw, 0.0)
    N = int(on.sum())
    n = max(N, 1)
    idx = np.argsort(-raw, axis=-1, kind="stable")[:, :k]
    th = np.tanh(raw / cap)
    a = cap * th
    ea = np.exp(a - cap)
    lse = cap + np.log(ea.sum(-1))
    soft = ea / ea.sum(-1, keepdims=True)
    ep = np.exp((a - cap) / tau)
    P = ep / ep.sum(-1, keepdims=True)
    top = np.take_along_axis(P, idx, -1)
    s = top.sum(-1, keepdims=True) + 1e-6
    w = top / s
    sel = np.zeros((B, E))
    np.put_along_axis(sel, idx, 1.0, -1)
    sel *= on[:, None]
    counts = sel.sum(0)
    Psum = (P * on[:, None]).sum(0)
    out = {"lb": E * np.sum(counts / n * Psum / n), "z": np.sum(lse ** 2 * on) / n,
           "counts": counts.astype(np.int64), "idx": np.where(on[:, None], idx, -1),
           "w": w * on[:, None]}
    dw = np.zeros((B, k)) if dw is None else np.asarray(dw, np.float64)
    dot = (dw * w).sum(-1, keepdims=True)
    g = np.tile(dlb * E * counts / n ** 2, (B, 1))
    gm = np.abs(g)
    gs = np.zeros((B, E))
    np.put_along_axis(gs, idx, (dw - dot) / s, -1)
    g = g + gs
    np.put_along_axis(gs, idx, (np.abs(dw) + (np.abs(dw) * w).sum(-1, keepdims=True)) / s, -1)
    gm = gm + gs
    da = P * (g - (P * g).sum(-1, keepdims=True)) / tau + dz * 2 * lse[:, None] * soft / n
    dam = P * (gm + (P * gm).sum(-1, keepdims=True)) / tau + abs(dz) * 2 * np.abs(lse[:, None]) * soft / n
    out["draw"] = da * (1 - th ** 2) * on[:, None]
    out["draw_mag"] = dam * on[:, None]
    return out


# ---- block norm -----------------------------------------------------------------

def block_norm(x=None, y=None, gate=None, post_weight=None, gamma=None, next_weight=None, eps=1e-5,
               dr=None, dh=None):
    def f8(t):
        return None if t is None else np.asarray(t, np.float64)
    x, y, gate, post, gam, nxt, dr, dh = map(f8, (x, y, gate, post_weight, gamma, next_weight, dr, dh))
    o = {}
    u, um = y, np.abs(y)
    if gate is not None:
        sg = _sig(gate)
        u = y * gate * sg
        um = np.abs(u) * (1 + np.abs(gate))     # the sigmoid's argument is rounded too
    f, fm = u, um
    if post is not None:
        iu = 1 / np.sqrt((u * u).mean(-1, keepdims=True) + eps)
        tu = (np.abs(u) * um).mean(-1, keepdims=True) * iu * iu     # the mean's own error
        f = u * iu * post
        fm = (um + np.abs(u) * tu) * iu * np.abs(post)
    g = f if gam is None else f * gam
    r = g if x is None else x + g
    rm = (fm if gam is None else fm * np.abs(gam)) + (0 if x is None else np.abs(x))
    o["r"], o["r_mag"] = r, rm
    D = np.zeros_like(y) if dr is None else dr
    Dm = np.abs(D)
    if nxt is not None:
        ir = 1 / np.sqrt((r * r).mean(-1, keepdims=True) + eps)
        tr = (np.abs(r) * rm).mean(-1, keepdims=True) * ir * ir
        nr = r * ir
        nrm = (rm + np.abs(r) * tr) * ir
        o["h"], o["h_mag"] = nr * nxt, nrm * np.abs(nxt)
        if dh is not None:
            q = dh * nxt
            dot = (q * nr).mean(-1, keepdims=True)
            dotm = (np.abs(q) * nrm).mean(-1, keepdims=True)
            D = D + (q - nr * dot) * ir
            Dm = Dm + ((np.abs(q) + np.abs(nr) * np.abs(dot)) * (1 + tr) + np.abs(nr) * dotm
                       + nrm * np.abs(dot)) * ir
            o["dnext_weight"], o["dnext_weight_mag"] = (dh * nr).sum(0), (np.abs(dh) * nrm).sum(0)
    if x is not None:
        o["dx"], o["dx_mag"] = D, Dm
    if gam is not None:
        o["dgamma"], o["dgamma_mag"] = (D * f).sum(0), (Dm * np.abs(f) + np.abs(D) * fm).sum(0)
        D, Dm = D * gam, Dm * np.abs(gam)
    if post is not None:
        nu, num = u * iu, (um + np.abs(u) * tu) * iu
        o["dpost_weight"], o["dpost_weight_mag"] = (D * nu).sum(0), (Dm * np.abs(nu) + np.abs(D) * num).sum(0)
        q, qm = D * post, Dm * np.abs(post)
        dot = (q * nu).mean(-1, keepdims=True)
        dotm = (qm * np.abs(nu) + np.abs(q) * num).mean(-1, keepdims=True)
        D = (q - nu * dot) * iu
        Dm = (qm + np.abs(nu) * dotm + num * np.abs(dot) + (np.abs(q) + np.abs(nu * dot)) * tu) * iu
    if gate is not None:
        ds = sg * (1 + gate * (1 - sg))
        o["dgate"] = D * y * ds
        o["dgate_mag"] = Dm * np.abs(y) * sg * (1 + np.abs(gate)) ** 2
        Dm = Dm * np.abs(gate) * sg * (1 + np.abs(gate))
        D = D * gate * sg
    o["dy"], o["dy_mag"] = D, Dm
    return o


# ---- AdamW ----------------------------------------------------------------------

def adamw(p, g, m, v, step, lr, b1, b2, eps, wd):
    p, g, m, v = (np.asarray(t, np.float64) for t in (p, g, m, v))
    mm = b1 * np.abs(m) + (1 - b1) * np.abs(g)
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    den = np.sqrt(v) / np.sqrt(1 - b2 ** step) + eps
    rate = lr / (1 - b1 ** step)
    return {"p": p * (1 - lr * wd) - rate * m / den, "p_mag": np.abs(p) + rate * mm / den,
            "m": m, "m_mag": mm, "v": v, "v_mag": v}


def e4m3_values():
    """The value of each code 0 .. 126 (the non-negative finite ones, ascending)."""
    c = np.arange(127)
    e, f = c >> 3, c & 7
    return np.where(e > 0, (8 + f) * 2.0 ** (e - 10), f * 2.0 ** -9)


def mix32(h):
    h = np.asarray(h, np.uint64) & 0xFFFFFFFF
    h = ((h ^ (h >> np.uint64(16))) * np.uint64(0x85EBCA6B)) & np.uint64(0xFFFFFFFF)
    h = ((h ^ (h >> np.uint64(13))) * np.uint64(0xC2B2AE35)) & np.uint64(0xFFFFFFFF)
    return h ^ (h >> np.uint64(16))


def randoms(n, tensor, seed, step):
    """The two numbers in (0, 1) of each of a tensor's n elements (below 2^32 of them)."""
    key = mix32((seed + step * 0x9E3779B1) & 0xFFFFFFFF)
    e = (np.arange(n, dtype=np.uint64) + np.uint64((tensor * 0x9E3779B9) & 0xFFFFFFFF)) & np.uint64(0xFFFFFFFF)
    h = mix32(e ^ key)
    return ((h >> np.uint64(16)).astype(np.float64) + 0.5) / 65536, ((h & np.uint64(0xFFFF)).astype(np.float64) + 0.5) / 65536


def encode8(t, root, u):
    """(codes, scales) of t's elements in blocks of 256, rounded by the numbers u: t signed, or
    where root the roots of t, up with the chance that keeps the square's mean."""
    t = np.asarray(t, np.float64)
    n = t.size
    pad = -n % 256
    b = np.abs(np.sqrt(t) if root else t)
    s = np.pad(b, (0, pad)).reshape(-1, 256).max(1) / 448.0
    sf = np.where(s > 0, s, 1.0).repeat(256)[:n]
    a = np.minimum(b / sf, 448.0)
    val = e4m3_values()
    lo = np.searchsorted(val, a, side="right") - 1
    hi = np.minimum(lo + 1, 126)
    x, y, z = (a, val[lo], val[hi]) if not root else (a * a, val[lo] ** 2, val[hi] ** 2)
    chance = np.where(hi > lo, (x - y) / np.where(hi > lo, z - y, 1.0), 0.0)
    c = np.where(u < chance, hi, lo)
    if root:
        c = np.where((c == 0) & (a > 0), 1, c)
    else:
        c = np.where(t < 0, c + 128, c)
    return c.astype(np.uint8), s


def decode8(codes, scales):
    c = np.asarray(codes, np.uint8)
    v = e4m3_values()[np.minimum(c & 127, 126)] * np.where(c >= 128, -1.0, 1.0)
    return v * np.asarray(scales, np.float64).repeat(256)[:c.size]
