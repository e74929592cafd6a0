"""The Muon step and its orthogonalisation in float64 (numpy). No counterpart in the reference.

    m = mu m + g;  u = g + mu m (nesterov) or m;  X = u / (|u| + eps), transposed where it is tall
    `steps` times X = a X + (b A + c A A) X, A = X X^T
    p = p (1 - lr wd) - lr rms sqrt(max(rows, cols)) X
"""
import numpy as np

COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def orthogonalize(u, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    """(X, off): X of each matrix of u (..., rows, cols), and what its Frobenius norm may be off
    (...) where each step of the products is rounded to 2^-24 of its magnitude: a step makes an
    error of at most `n` roundings of |a| + |b| + |c| times the norm of X, and takes the error that
    X has to at most `a` times it (the largest slope of the polynomial on singular values)."""
    u = np.asarray(u, np.float64)
    tall = u.shape[-2] > u.shape[-1]
    X = np.swapaxes(u, -1, -2) if tall else u
    X = X / (np.sqrt((X * X).sum((-1, -2), keepdims=True)) + eps)
    a, b, c = coefficients
    n = max(X.shape[-2:]) / 16 + 32          # the instruction adds 16 products at a time
    norm = lambda x: np.sqrt((x * x).sum((-1, -2)))  # noqa: E731
    off = n * 2.0 ** -24 * norm(X)
    for _ in range(steps):
        A = X @ np.swapaxes(X, -1, -2)
        off = abs(a) * off + n * 2.0 ** -24 * (abs(a) + abs(b) + abs(c)) * norm(X)
        X = a * X + (b * A + c * (A @ A)) @ X
    return (np.swapaxes(X, -1, -2) if tall else X), off


def muon(p, g, m, lr, mu=0.95, nesterov=True, wd=0.1, rms=0.2, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    """dict of p, m, and off: what p's matrices may be off in the Frobenius norm but for p's own
    rounding."""
    p, g, m = (np.asarray(t, np.float64) for t in (p, g, m))
    m = mu * m + g
    X, off = orthogonalize(g + mu * m if nesterov else m, steps, coefficients, eps)
    rate = lr * rms * np.sqrt(max(p.shape[-2:]))
    return {"p": p * (1 - lr * wd) - rate * X, "m": m, "off": rate * off}
