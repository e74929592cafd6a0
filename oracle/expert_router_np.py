"""Routing to experts by softmax or sigmoid scores with a bias and groups, in float64 (numpy),
and the gradient of the logits from the formula:

    s = softmax(raw) or 1 / (1 + exp(-raw));  b = s + bias;  a group's worth = its two largest b
    idx = the k largest b of the top_groups worthiest groups, the lowest index first on ties
    w = scale s[idx] / (sum s[idx] + 1e-20), or scale s[idx]

No counterpart in the reference."""
import numpy as np


def _ranked(v, n):
    """Indices of the n largest of each row, NaN above every number, the lowest index on ties."""
    key = np.where(np.isnan(v), 2, np.where(np.isposinf(v), 1, 0))
    val = np.where(np.isfinite(v) | np.isneginf(v), v, 0.0)
    order = np.lexsort((np.broadcast_to(np.arange(v.shape[1]), v.shape), -val, -key), axis=-1)
    return order[:, :n]


def route(raw, k, score="softmax", bias=None, groups=1, top_groups=None, renormalize=True, scale=1.0,
          mask=None, dw=None):
    """dict of idx, w, counts, and with dw of draw and draw_mag (its terms' magnitudes)."""
    raw = np.asarray(raw, np.float64)
    B, E = raw.shape
    top_groups = groups if top_groups is None else top_groups
    on = np.ones(B, bool) if mask is None else np.asarray(mask, bool)
    x = np.where(on[:, None], raw, 0.0)
    with np.errstate(invalid="ignore", over="ignore"):
        if score == "softmax":
            e = np.exp(x - x.max(-1, keepdims=True, initial=-np.inf))
            s = e / e.sum(-1, keepdims=True)
            off = None
        else:
            s, off = 1 / (1 + np.exp(-x)), 1 / (1 + np.exp(x))
    b = s if bias is None else s + np.asarray(bias, np.float64)
    if bias is None and groups == 1:
        b = x
    if groups > 1:
        per = b.reshape(B, groups, E // groups)
        two = np.take_along_axis(per, _ranked(per.reshape(B * groups, -1), 2).reshape(B, groups, -1), -1)
        kept = _ranked(two.sum(-1) if two.shape[-1] > 1 else two[..., 0], top_groups)
        open_ = np.zeros((B, groups), bool)
        np.put_along_axis(open_, kept, True, 1)
        closed = ~np.repeat(open_, E // groups, 1)
        order = _ranked(b, E)                   # the closed ones fall away
        idx = np.array([[e for e in row if not c[e]][:k] for row, c in zip(order, closed)]).reshape(B, k)
    else:
        idx = _ranked(b, k)
    t = np.take_along_axis(s, idx, 1)
    total = t.sum(-1, keepdims=True) + 1e-20
    w = scale * (t / total if renormalize else t)
    sel = np.zeros((B, E))
    np.put_along_axis(sel, idx, 1.0, 1)
    out = {"idx": np.where(on[:, None], idx, -1), "w": w * on[:, None],
           "counts": (sel * on[:, None]).sum(0).astype(np.int64), "s": s}
    if dw is None:
        return out
    dw = np.asarray(dw, np.float64)
    u = t / total
    g = scale / total * (dw - (dw * u).sum(-1, keepdims=True)) if renormalize else scale * dw
    far = np.abs(dw) + np.abs(dw[:, :1])
    mag = scale / total * (far + (far * u).sum(-1, keepdims=True)) if renormalize else scale * np.abs(dw)
    full, full_mag = np.zeros((B, E)), np.zeros((B, E))
    np.put_along_axis(full, idx, g, 1)
    np.put_along_axis(full_mag, idx, mag, 1)
    if score == "softmax":
        d = s * (full - (full * s).sum(-1, keepdims=True))
        m = s * (full_mag + (full_mag * s).sum(-1, keepdims=True))
    else:
        d, m = full * s * off, full_mag * s * off
    out["draw"], out["draw_mag"] = d * on[:, None], m * on[:, None]
    return out
