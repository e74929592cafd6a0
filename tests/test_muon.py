"""The Muon step on the CPU: the oracle (oracle/muon_np.py) against singular values, the refusals of
the C ABI and of the Python entry points (none reaches a GPU), the optimizer's bookkeeping."""
import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import muon_np as mn


@pytest.mark.parametrize("shape", [(1, 5), (7, 7), (30, 12), (3, 8, 20)])
def test_oracle_acts_on_singular_values(shape):
    g = np.random.default_rng(len(shape))
    u = g.normal(size=shape)
    X, off = mn.orthogonalize(u)
    U, s, V = np.linalg.svd(u, full_matrices=False)
    s = s / (np.sqrt((u * u).sum((-1, -2)))[..., None] + 1e-7)
    a, b, c = mn.COEFFICIENTS
    for _ in range(5):
        s = a * s + b * s ** 3 + c * s ** 5
    assert np.allclose(X, (U * s[..., None, :]) @ V, atol=1e-10)
    assert np.all((s > 0.3) & (s < 1.3)) and np.all(off > 0) and off.shape == shape[:-2]


def test_oracle_step():
    g = np.random.default_rng(0)
    p, q, m = g.normal(size=(6, 9)), g.normal(size=(6, 9)), g.normal(size=(6, 9))
    o = mn.muon(p, q, m, 0.1, wd=0.5)
    assert np.allclose(o["m"], 0.95 * m + q)
    X, _ = mn.orthogonalize(q + 0.95 * o["m"])
    assert np.allclose(o["p"], 0.95 * p - 0.1 * 0.2 * 3 * X)
    assert np.allclose(mn.muon(p, q, m, 0.1, nesterov=False)["p"],
                       0.99 * p - 0.06 * mn.orthogonalize(o["m"])[0])
    z = mn.orthogonalize(np.zeros((3, 4)))[0]
    assert (z == 0).all()


def _tensor(pkg, **kw):
    t = pkg._lib.TmoeMuonTensor()
    for k, v in dict(dict(p=64, g=64, m=64, batch=2, rows=8, cols=16), **kw).items():
        setattr(t, k, v)
    return t


def _args(pkg, **kw):
    a = pkg._lib.TmoeMuonStep()
    for k, v in dict(dict(lr=0.02, momentum=0.95, weight_decay=0.1, update_rms=0.2, eps=1e-7,
                          coefficients=(ctypes.c_double * 3)(*mn.COEFFICIENTS), steps=5, nesterov=1, dtype=0,
                          write_only=0), **kw).items():
        setattr(a, k, (ctypes.c_double * 3)(*v) if k == "coefficients" else v)
    return a


@pytest.mark.parametrize("tk,ak,code", [
    (dict(batch=-1), {}, -1), (dict(rows=-1), {}, -1), (dict(cols=-1), {}, -1), (dict(rows=2 ** 22 + 1), {}, -2),
    (dict(rows=2 ** 17, cols=2 ** 17), {}, -2), (dict(batch=2 ** 36), {}, -2), (dict(p=0), {}, -1),
    (dict(g=0), {}, -1), (dict(p=66), {}, -1), (dict(g=66), {}, -1), (dict(m=66), {}, -1),
    ({}, dict(dtype=2), -1), ({}, dict(steps=0), -1), ({}, dict(steps=17), -1), ({}, dict(momentum=1.0), -1),
    ({}, dict(momentum=-0.1), -1), ({}, dict(momentum=math.nan), -1), ({}, dict(lr=-1.0), -1),
    ({}, dict(lr=math.inf), -1), ({}, dict(weight_decay=-1.0), -1), ({}, dict(update_rms=math.nan), -1),
    ({}, dict(eps=0.0), -1), ({}, dict(eps=math.inf), -1), ({}, dict(eps=1e-60), -1),
    ({}, dict(coefficients=(5.0, 0.0, 0.0)), -1), ({}, dict(coefficients=(math.nan, 0, 0)), -1),
    ({}, dict(coefficients=(1.0, -40.0, 39.5)), -1), ({}, dict(coefficients=(1.9, 0.0, 0.0)), -1)])
def test_abi_refusals(pkg, tk, ak, code):
    L = pkg._lib.lib()
    t, a = _tensor(pkg, **tk), _args(pkg, **ak)
    assert L.tmoe_muon_step(ctypes.byref(t), 1, ctypes.byref(a), 256, 1 << 40, None) == code
    assert L.tmoe_last_error().startswith(b"tmoe_muon_step: ")


def test_abi_workspace_and_empty(pkg):
    L = pkg._lib.lib()
    t, a = _tensor(pkg), _args(pkg)
    r = ctypes.byref
    need = L.tmoe_muon_workspace_bytes(r(t), 1)
    assert need >= 2 * 2 * (4 + 4) * 64 * 64      # X, X', A and B in two parts each, of two matrices
    assert L.tmoe_muon_workspace_bytes(r(t), 0) == 0 and L.tmoe_muon_workspace_bytes(None, 1) == 0
    assert L.tmoe_muon_workspace_bytes(r(_tensor(pkg, rows=2 ** 23)), 1) == 0
    assert L.tmoe_muon_workspace_bytes(r(_tensor(pkg, rows=-1)), 1) == 0
    for ws, n in ((0, need), (256, need - 1), (64, need)):
        assert L.tmoe_muon_step(r(t), 1, r(a), ws, n, None) == -1
    assert L.tmoe_muon_step(r(t), 1, None, 256, need, None) == -1
    assert L.tmoe_muon_step(None, 1, r(a), 256, need, None) == -1
    assert L.tmoe_muon_step(r(t), -1, r(a), 256, need, None) == -1
    for kw in (dict(batch=0), dict(rows=0), dict(cols=0)):
        e = _tensor(pkg, p=0, g=0, m=0, **kw)
        assert L.tmoe_muon_workspace_bytes(r(e), 1) == 0
        assert L.tmoe_muon_step(r(e), 1, r(a), 0, 0, None) == 0
    assert L.tmoe_muon_step(None, 0, r(a), 0, 0, None) == 0


def test_python_refusals(pkg):
    p, g, m = torch.zeros(4, 6), torch.zeros(4, 6), torch.zeros(4, 6)
    step = lambda a, b, c, **kw: pkg.muon_step(a, b, c, lr=0.1, **kw)  # noqa: E731
    for args, kw, text in [
            (([p], [g, g], [m]), {}, "for 2 gradients"), (([p], [g], []), {}, "momenta"),
            (([p], [g.double()], [m]), {}, "dtype"), (([p.bfloat16()], [g], [m]), {}, "parameter"),
            (([p, p], [g, g.bfloat16()], [m, m]), {}, "the first of"), (([p[0]], [g[0]], [m[0]]), {}, "matrices"),
            (([p], [g.t()], [m]), {}, "parameter"), (([p], [g], [m.bfloat16()]), {}, "momentum"),
            (([p], [g], [m.t()]), {}, "momentum"), (([p.t().contiguous().t()], [g], [m]), {}, "contiguous"),
            (([p], [g], [m.t().contiguous().t()]), {}, "contiguous"), (([p, p], [g, g], [m, m.clone()]), {}, "share"),
            (([p], [p], [m]), {}, "gradient shares"), (([p], [m], [m]), {}, "gradient shares"),
            (([p], [g.to_sparse()], [m]), {}, "sparse"), (([p], [g], [m]), dict(steps=0), "steps"),
            (([p], [g], [m]), dict(steps=17), "steps"), (([p], [g], [m]), {}, "HIP devices only")]:
        with pytest.raises(RuntimeError, match=text):
            step(*args, **kw)
    for kw in (dict(momentum=1.0), dict(weight_decay=-1.0), dict(update_rms=-1.0), dict(eps=0.0),
               dict(coefficients=(1.0, 2.0))):
        with pytest.raises(ValueError):
            step([p], [g], [m], **kw)
    with pytest.raises(TypeError, match="list"):
        step(p, [g], [m])
    step([], [], [])
    assert pkg.orthogonalize([]) == []
    for x, text in ((g[0], "matrices"), (g.double(), "dtype"), (g.clone().requires_grad_(), "gradient"),
                    (g, "HIP devices only")):
        with pytest.raises(RuntimeError, match=text):
            pkg.orthogonalize(x)
    with pytest.raises(ValueError):
        pkg.orthogonalize(g, eps=0.0)
    with torch.autograd.forward_ad.dual_level():
        d = torch.autograd.forward_ad.make_dual(g, g + 1)
        with pytest.raises(RuntimeError, match="forward-mode"):
            pkg.orthogonalize(d)


def test_optimizer_options_and_states(pkg):
    w = torch.nn.Parameter(torch.zeros(4, 6))
    for kw in (dict(lr=-1.0), dict(momentum=1.0), dict(weight_decay=-0.1), dict(update_rms=-1.0), dict(steps=0),
               dict(eps=0.0), dict(coefficients=(1.0,))):
        with pytest.raises(ValueError):
            pkg.FusedMuon([w], **kw)
    with pytest.raises(ValueError, match="no matrix"):
        pkg.FusedMuon([torch.nn.Parameter(torch.zeros(4))])
    opt = pkg.FusedMuon([{"params": [w], "lr": 0.5}])
    with pytest.raises(ValueError):
        opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(2, 2))], "steps": 99})
    assert opt.step() is None and not opt.state            # no gradient: nothing to do
    opt.state[w]["momentum_buffer"] = torch.full((4, 6), 0.5)
    sd = opt.state_dict()
    b = torch.nn.Parameter(torch.zeros(4, 6, dtype=torch.bfloat16))
    new = pkg.FusedMuon([b])
    new.load_state_dict(sd)
    got = new.state[b]["momentum_buffer"]
    assert got.dtype == torch.float32 and (got == 0.5).all() and new.param_groups[0]["lr"] == 0.5
    assert got.data_ptr() != sd["state"][0]["momentum_buffer"].data_ptr()
    wrong = pkg.FusedMuon([torch.nn.Parameter(torch.zeros(6, 4))])
    with pytest.raises(ValueError, match="momentum"):
        wrong.load_state_dict(sd)
    with pytest.raises(ValueError, match="momentum"):
        pkg.FusedMuon([torch.nn.Parameter(torch.zeros(4, 6))]).load_state_dict(
            {**sd, "state": {0: {"exp_avg": torch.zeros(4, 6)}}})
    with pytest.raises(ValueError, match="steps"):
        new.load_state_dict({**sd, "param_groups": [{**sd["param_groups"][0], "steps": 0}]})


def test_coefficients_are_refused_with_the_group(pkg):
    w = torch.nn.Parameter(torch.zeros(4, 6))
    for c in ((5.0, 0.0, 0.0), (1.0, -40.0, 39.5), (math.nan, 0.0, 0.0)):
        with pytest.raises(ValueError, match="do not stay in range"):
            pkg.FusedMuon([w], coefficients=c)
        opt = pkg.FusedMuon([w])
        with pytest.raises(ValueError, match="do not stay in range"):
            opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(2, 2))], "coefficients": c})
        sd = opt.state_dict()
        with pytest.raises(ValueError, match="do not stay in range"):
            opt.load_state_dict({**sd, "param_groups": [{**sd["param_groups"][0], "coefficients": c}]})
        with pytest.raises(RuntimeError, match="do not stay in range"):
            pkg.muon_step([], [], [], lr=0.1, coefficients=c)
    with pytest.raises(ValueError):
        pkg.FusedMuon([w], lr=math.inf)
