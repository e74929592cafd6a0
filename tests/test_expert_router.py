"""The expert router on the CPU: the float64 oracle (oracle/expert_router_np.py) against autograd,
differences and closed forms, and the refusals of the C ABI and of the Python entry points (none
reaches a GPU)."""
import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import expert_router_np as er

D = torch.float64
FORMS = [dict(score="softmax"), dict(score="sigmoid"), dict(score="softmax", renormalize=False, scale=2.5),
         dict(score="sigmoid", renormalize=False), dict(score="sigmoid", groups=4, top_groups=2, scale=1.5),
         dict(score="softmax", groups=3, top_groups=1), dict(score="sigmoid", bias=True, groups=2),
         dict(score="softmax", bias=True), dict(score="softmax", bias=True, groups=12, top_groups=5)]


@pytest.mark.parametrize("form", FORMS, ids=lambda f: "-".join(f"{k}{v}" for k, v in f.items()))
@pytest.mark.parametrize("k", [1, 3])
def test_oracle_gradient(form, k):
    g = np.random.default_rng(k)
    B, E = 9, 12
    f = dict(form)
    raw, dw = g.normal(size=(B, E)) * 2, g.normal(size=(B, k))
    if f.pop("bias", None):
        f["bias"] = g.normal(size=E) * 0.2
    mask = g.random(B) < 0.7
    o = er.route(raw, k, mask=mask, dw=dw, **f)
    t = torch.tensor(raw, requires_grad=True)
    s = torch.softmax(t, -1) if f["score"] == "softmax" else torch.sigmoid(t)
    idx = torch.tensor(np.where(o["idx"] < 0, 0, o["idx"]))
    top = s.gather(1, idx)
    w = f.get("scale", 1.0) * (top / (top.sum(-1, keepdim=True) + 1e-20) if f.get("renormalize", True) else top)
    w = w * torch.tensor(mask)[:, None]
    assert np.allclose(o["w"], w.detach().numpy(), rtol=1e-12)
    (w * torch.tensor(dw)).sum().backward()
    assert np.allclose(o["draw"], t.grad.numpy(), rtol=1e-9, atol=1e-15)
    assert np.all(np.abs(o["draw"]) <= o["draw_mag"] * (1 + 1e-12) + 1e-18)
    # the selection by its definition, a token at a time
    b = s.detach().numpy() + (0 if f.get("bias") is None else f["bias"])
    if f.get("bias") is None and f.get("groups", 1) == 1:
        b = raw
    G, T = f.get("groups", 1), f.get("top_groups", f.get("groups", 1))
    for r in range(B):
        if not mask[r]:
            assert (o["idx"][r] == -1).all()
            continue
        groups = np.split(np.arange(E), G)
        worth = [sum(sorted(b[r][m])[-2:]) for m in groups]
        live = sorted(np.concatenate([groups[i] for i in sorted(range(G), key=lambda i: -worth[i])[:T]]))
        want = sorted(live, key=lambda e: -b[r][e])[:k]
        assert list(o["idx"][r]) == want
    assert o["counts"].sum() == k * mask.sum()


def test_oracle_differences():
    g = np.random.default_rng(2)
    raw, dw = g.normal(size=(4, 6)), g.normal(size=(4, 2))
    for f in (dict(score="sigmoid"), dict(score="softmax", renormalize=False)):
        draw = er.route(raw, 2, dw=dw, **f)["draw"]
        for i in range(4):
            for e in range(6):
                h = np.zeros_like(raw)
                h[i, e] = 1e-6
                up, dn = (er.route(raw + s * h, 2, **f) for s in (1, -1))
                assert np.array_equal(up["idx"], dn["idx"])
                assert ((up["w"] - dn["w"]) * dw).sum() / 2e-6 == pytest.approx(draw[i, e], abs=1e-8)


def test_oracle_ties_and_nan():
    nan, inf = math.nan, math.inf
    o = er.route([[1, 3, 3, 2, 3, 3], [0, -0.0, 0, 0, 0, 0], [40, 41, 42, 1, 2, 3], [1, nan, 3, inf, nan, 2]], 3,
                 score="sigmoid")
    assert o["idx"].tolist() == [[1, 2, 4], [0, 1, 2], [2, 1, 0], [1, 4, 3]]
    # as scores the sigmoids of 40 and more are all one in float64
    o = er.route([[40, 41, 42, 1, 2, 3]], 3, score="sigmoid", bias=np.zeros(6))
    assert o["idx"].tolist() == [[0, 1, 2]]


def _router(pkg, **kw):
    t = pkg._lib.TmoeExpertRouter()
    for k, v in dict(dict(raw=64, row_stride=8, B=4, E=8, k=2, groups=1, top_groups=1, dtype=0, score=1,
                          renormalize=1, scale=1.0), **kw).items():
        setattr(t, k, v)
    return t


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=2), -1), (dict(score=2), -1), (dict(B=-1), -1), (dict(E=0), -1), (dict(k=0), -1),
    (dict(E=257, row_stride=257), -2), (dict(E=64, row_stride=64, k=17), -2), (dict(B=2 ** 30 + 1), -2),
    (dict(groups=0), -1), (dict(groups=3), -1), (dict(groups=9), -1), (dict(groups=4, top_groups=5), -1),
    (dict(groups=4, top_groups=0), -1), (dict(groups=8, top_groups=1), -1), (dict(k=9), -1),
    (dict(scale=0.0), -1), (dict(scale=math.nan), -1), (dict(scale=math.inf), -1), (dict(scale=-1.0), -1),
    (dict(raw=0), -1), (dict(row_stride=7), -1), (dict(raw=66), -1), (dict(bias=66), -1)])
def test_abi_refusals(pkg, kw, code):
    L = pkg._lib.lib()
    r = _router(pkg, **kw)
    assert L.tmoe_expert_router_forward(ctypes.byref(r), 64, 64, 64, 64, 1 << 30, None) == code
    assert L.tmoe_last_error().startswith(b"tmoe_expert_router_forward: ")
    assert L.tmoe_expert_router_backward(ctypes.byref(r), 64, 64, 64, 64, None) == code


def test_abi_refuses_pointers(pkg):
    L = pkg._lib.lib()
    r = _router(pkg)
    need = L.tmoe_expert_router_workspace_bytes(4, 8)
    assert need > 0 and L.tmoe_expert_router_workspace_bytes(-1, 8) == 0
    assert L.tmoe_expert_router_workspace_bytes(4, 257) == 0
    assert L.tmoe_expert_router_forward(None, 64, 64, 64, 64, 1 << 20, None) == -1
    for args in ((0, 64, 64, 64, need), (64, 0, 64, 64, need), (64, 64, 0, 64, need), (64, 64, 64, 0, need),
                 (68, 64, 64, 64, need), (64, 66, 64, 64, need), (64, 64, 68, 64, need), (64, 64, 64, 66, need),
                 (64, 64, 64, 64, need - 1)):
        assert L.tmoe_expert_router_forward(ctypes.byref(r), *args, None) == -1
    for args in ((0, 64, 64, 64), (64, 0, 64, 64), (64, 64, 0, 64), (64, 64, 64, 0), (68, 64, 64, 64),
                 (64, 66, 64, 64), (64, 64, 66, 64), (64, 64, 64, 66)):
        assert L.tmoe_expert_router_backward(ctypes.byref(r), *args, None) == -1
    e = _router(pkg, B=0, raw=0, row_stride=0)
    assert L.tmoe_expert_router_backward(ctypes.byref(e), 0, 0, 0, 0, None) == 0


def test_python_refusals(pkg):
    f = pkg.fused_expert_router
    raw = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="score"):
        f(raw, 2, score="tanh")
    for args, kw, text in [
            ((raw.double(), 2), {}, "dtype"), ((raw[0], 2), {}, r"\(B, E\)"), ((raw, 0), {}, "top_k"),
            ((torch.zeros(4, 257), 2), {}, "experts"), ((torch.zeros(4, 64), 17), {}, "top_k"),
            ((raw, 2), dict(groups=3), "groups"), ((raw, 2), dict(groups=0), "groups"),
            ((raw, 2), dict(groups=2, top_groups=3), "groups"), ((raw, 3), dict(groups=4, top_groups=1), "open"),
            ((raw, 9), {}, "open"), ((raw, 2), dict(scale=0.0), "scale"), ((raw, 2), dict(scale=1e39), "scale"),
            ((raw, 2), dict(scale=1e-50), "scale"),
            ((raw, 2), dict(bias=torch.zeros(7)), "bias"), ((raw, 2), dict(bias=torch.zeros(8, dtype=D)), "bias"),
            ((raw, 2), dict(bias=torch.zeros(8, requires_grad=True)), "gradient"),
            ((raw, 2), dict(mask=torch.ones(3, dtype=torch.bool)), "mask"),
            ((raw, 2), dict(mask=torch.ones(4)), "mask"), ((raw, 2), {}, "HIP devices only")]:
        with pytest.raises(RuntimeError, match=text):
            f(*args, **kw)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(raw, raw + 1)
        with pytest.raises(RuntimeError, match="forward-mode"):
            f(dual, 2)
