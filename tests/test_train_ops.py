"""The training operators around the expert contraction, on the CPU: the float64 oracle
(oracle/train_ops_np.py) against autograd, differences and closed forms, the refusals of the
C ABI and of the Python entry points (none reaches a GPU), the optimizer's bookkeeping."""
import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import train_ops_np as tn
from oracle import train_router_np as tr

D = torch.float64


# ---- the oracle -----------------------------------------------------------------

def _router_torch(raw, k, tau, cap, mask):
    B, E = raw.shape
    on = torch.ones(B, dtype=D) if mask is None else mask.to(D)
    cap_ = cap * torch.tanh(torch.where(on[:, None] > 0, raw, 0.0) / cap)
    P = torch.softmax(cap_ / tau, -1)
    idx = torch.sort(raw.detach(), dim=-1, descending=True, stable=True).indices[:, :k]
    top = P.gather(1, idx)
    w = top / (top.sum(-1, keepdim=True) + 1e-6) * on[:, None]
    sel = torch.zeros_like(P).scatter_(1, idx, 1.0) * on[:, None]
    n = max(float(on.sum()), 1.0)
    lb = E * ((sel.sum(0) / n) * ((P * on[:, None]).sum(0) / n)).sum()
    z = (torch.logsumexp(cap_, -1) ** 2 * on).sum() / n
    return w, lb, z


@pytest.mark.parametrize("B,E,k,tau,padded", [(1, 2, 1, 0.5, 0), (23, 8, 2, 0.5, 0), (40, 6, 6, 2.0, 0.4),
                                              (17, 33, 5, 1.25, 0.3), (9, 8, 2, 0.7, 1.0)])
def test_router_oracle_gradient(B, E, k, tau, padded):
    g = np.random.default_rng(B + E)
    raw = g.normal(size=(B, E)) * 6
    mask = g.random(B) >= padded if padded else None
    dw = g.normal(size=(B, k))
    o = tn.router(raw, k, tau, 10.0, mask, dw, 0.3, 0.2)
    t = torch.tensor(raw, requires_grad=True)
    w, lb, z = _router_torch(t, k, tau, 10.0, None if mask is None else torch.tensor(mask))
    (w * torch.tensor(dw)).sum().add(0.3 * lb).add(0.2 * z).backward()
    assert np.allclose(o["w"], w.detach().numpy(), rtol=1e-12, atol=1e-15)
    assert o["lb"] == pytest.approx(lb.item(), rel=1e-12) and o["z"] == pytest.approx(z.item(), rel=1e-12)
    assert np.allclose(o["draw"], t.grad.numpy(), rtol=1e-9, atol=1e-14)
    assert np.all(np.abs(o["draw"]) <= o["draw_mag"] * (1 + 1e-12))
    if mask is None:      # the training layer's own restatement
        r = tr.route(raw, k, tau, True)
        assert np.array_equal(r["idx"], o["idx"]) and np.allclose(r["top_p"], o["w"], rtol=1e-12)
        assert r["z_loss"] == pytest.approx(o["z"], rel=1e-12)
        assert r["lb_loss"] == pytest.approx(o["lb"], rel=1e-6)     # float32-cast there


def test_router_oracle_differences():
    """The gradient against differences of lb, z and the weights' sum."""
    g = np.random.default_rng(5)
    raw, dw, k, tau = g.normal(size=(6, 5)) * 4, g.normal(size=(6, 2)), 2, 0.8
    mask = np.array([1, 1, 0, 1, 1, 1], bool)

    def loss(r):
        o = tn.router(r, k, tau, 10.0, mask)
        return (o["w"] * dw).sum() + 0.7 * o["lb"] + 0.1 * o["z"]
    draw = tn.router(raw, k, tau, 10.0, mask, dw, 0.7, 0.1)["draw"]
    for i in range(6):
        for e in range(5):
            h = np.zeros_like(raw)
            h[i, e] = 1e-6
            assert (loss(raw + h) - loss(raw - h)) / 2e-6 == pytest.approx(draw[i, e], abs=2e-8)


NORM_FORMS = [("x", "y"), ("y", "gate"), ("x", "y", "gamma"), ("y", "next"), ("y", "post"),
              ("x", "y", "gamma", "next"), ("y", "gate", "post"), ("x", "y", "post", "next"),
              ("x", "y", "gate", "post", "gamma", "next")]
_KEY = {"post": "post_weight", "next": "next_weight"}


def norm_inputs(form, T, d, seed, dtype=torch.float32):
    """Operands of a form as CPU tensors of dtype, and dr, dh."""
    g = torch.Generator().manual_seed(seed)
    n = {}
    for f in form:
        if f in ("x", "y", "gate"):
            n[f] = (torch.randn(T, d, generator=g) * (3.0 if f == "x" else 1.0)).to(dtype)
        else:
            n[_KEY.get(f, f)] = (0.7 + 0.3 * torch.randn(d, generator=g)).to(dtype)
    return n, torch.randn(T, d, generator=g).to(dtype), torch.randn(T, d, generator=g).to(dtype)


def _norm_torch(x=None, y=None, gate=None, post_weight=None, gamma=None, next_weight=None, eps=1e-5):
    def rms(v, w):
        return v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps) * w
    u = y if gate is None else y * torch.nn.functional.silu(gate)
    u = u if post_weight is None else rms(u, post_weight)
    u = u if gamma is None else gamma * u
    r = u if x is None else x + u
    return r, None if next_weight is None else rms(r, next_weight)


@pytest.mark.parametrize("form", NORM_FORMS, ids="+".join)
def test_norm_oracle_gradient(form):
    n, dr, dh = norm_inputs(form, 5, 12, len(form), D)
    has_h = "next" in form
    o = tn.block_norm(**{k: v.numpy() for k, v in n.items()}, dr=dr.numpy(), dh=dh.numpy() if has_h else None)
    t = {k: v.clone().requires_grad_() for k, v in n.items()}
    r, h = _norm_torch(**t)
    grads = torch.autograd.grad((r, h) if has_h else (r,), list(t.values()), (dr, dh) if has_h else (dr,))
    assert np.allclose(o["r"], r.detach().numpy(), rtol=1e-12)
    assert not has_h or np.allclose(o["h"], h.detach().numpy(), rtol=1e-12)
    for k, gr in zip(t, grads):
        assert np.allclose(o["d" + k], gr.numpy(), rtol=1e-9, atol=1e-12), k
        assert np.all(np.abs(o["d" + k]) <= o["d" + k + "_mag"] * (1 + 1e-9)), k


def test_adamw_oracle_is_torchs():
    g = torch.Generator().manual_seed(0)
    p = torch.randn(50, generator=g, dtype=D).requires_grad_()
    q, m, v = p.detach().numpy().copy(), np.zeros(50), np.zeros(50)
    opt = torch.optim.AdamW([p], lr=3e-3, betas=(0.8, 0.95), eps=1e-6, weight_decay=0.1)
    for step in range(1, 6):
        p.grad = torch.randn(50, generator=g, dtype=D)
        opt.step()
        o = tn.adamw(q, p.grad.numpy(), m, v, step, 3e-3, 0.8, 0.95, 1e-6, 0.1)
        q, m, v = o["p"], o["m"], o["v"]
        assert np.allclose(q, p.detach().numpy(), rtol=1e-12)


def test_e4m3_and_encoding_means():
    val = tn.e4m3_values()
    assert np.array_equal(val, torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy())
    g = np.random.default_rng(3)
    t = np.concatenate([[0.0, 1.0, -1.0, 1e-9, 0.3], g.normal(size=295) * np.exp(g.normal(size=295) * 3)])
    n = 4000
    for root in (False, True):
        x = np.abs(t) if root else t
        mean = np.zeros(t.size)
        for i in range(n):
            c, s = tn.encode8(x, root, (g.integers(0, 65536, t.size) + 0.5) / 65536)
            d = tn.decode8(c, s)
            mean += (d * d if root else d) / n
        # a code's mean over n draws is off by its step / (2 sqrt(n)) in the deviation; five
        # of them, the 2^-17 of the numbers' own grid, and what is kept from rounding to zero
        sf = s.repeat(256)[:t.size]
        a = np.abs(np.sqrt(x) if root else x) / sf
        lo = np.clip(np.searchsorted(val, a, side="right") - 1, 0, 125)
        z = val ** 2 if root else val
        step = (z[lo + 1] - z[lo]) * (sf * sf if root else sf)
        bound = step * (2.5 / math.sqrt(n) + 2.0 ** -17)
        kept = (a < val[1]) if root else np.zeros(t.size, bool)
        assert np.all(np.abs(mean - x)[~kept] <= bound[~kept] + 1e-12 * np.abs(x)[~kept])
        assert np.all(mean[kept & (a > 0)] >= x[kept & (a > 0)] * (1 - 1e-12))


# ---- refusals -------------------------------------------------------------------

OK = 0x10000   # an aligned dummy address, never dereferenced


def _router(pkg, **kw):
    d = dict(raw=OK, row_stride=8, B=4, E=8, k=2, dtype=0, cap=10.0, temperature=0.5)
    d.update(kw)
    return ctypes.byref(pkg._lib.TmoeRouter(**d))


@pytest.mark.parametrize("kw,code,msg", [
    (dict(k=9), -1, "k=9"), (dict(k=0), -1, "k=0"), (dict(B=-1), -1, "B=-1"), (dict(E=0), -1, "E=0"),
    (dict(E=300, row_stride=300), -2, "256"), (dict(E=32, k=17, row_stride=32), -2, "16"),
    (dict(B=1 << 31), -2, "2^30"), (dict(dtype=2), -1, "dtype"), (dict(cap=0.0), -1, "cap"),
    (dict(cap=math.inf), -1, "cap"), (dict(temperature=0.0), -1, "temperature"),
    (dict(temperature=math.nan), -1, "temperature"), (dict(raw=None), -1, "raw"),
    (dict(row_stride=7), -1, "row_stride"), (dict(raw=OK + 2), -1, "misaligned"),
    (dict(temperature_dev=OK + 2), -1, "misaligned"),
])
def test_router_abi_refuses(pkg, kw, code, msg):
    L = pkg._lib.lib()
    ws = L.tmoe_router_workspace_bytes(4, 8)
    for rc in (L.tmoe_router_forward(_router(pkg, **kw), OK, OK, OK, OK, OK, OK, OK, ws, None),
               L.tmoe_router_backward(_router(pkg, **kw), OK, OK, OK, OK, OK, OK, OK, None)):
        assert rc == code and msg in L.tmoe_last_error().decode()


def test_router_abi_refuses_pointers(pkg):
    L = pkg._lib.lib()
    ws = L.tmoe_router_workspace_bytes(4, 8)
    assert ws > 0 and L.tmoe_router_workspace_bytes(-1, 8) == 0 == L.tmoe_router_workspace_bytes(4, 300)
    r = _router(pkg)
    for i in range(7):
        for bad in (None, OK + 2):
            a = [OK] * 7
            a[i] = bad
            assert L.tmoe_router_forward(r, *a, ws, None) == -1, (i, bad)
    assert L.tmoe_router_forward(r, *[OK] * 7, ws - 1, None) == -1
    assert "workspace" in L.tmoe_last_error().decode()
    assert L.tmoe_router_forward(None, *[OK] * 7, ws, None) == -1
    for i in (0, 1, 2, 6):
        a = [OK] * 7
        a[i] = None
        assert L.tmoe_router_backward(r, *a, None) == -1, i
    for i in range(7):
        a = [OK] * 7
        a[i] = OK + 2
        assert L.tmoe_router_backward(r, *a, None) == -1, i
    assert L.tmoe_router_backward(_router(pkg, B=0, raw=None), *[None] * 7, None) == 0


def _norm(pkg, **kw):
    d = dict(x=OK, y=OK, gate=OK, x_stride=64, y_stride=64, gate_stride=64, post_weight=OK, gamma=OK,
             next_weight=OK, T=40, d=64, dtype=0, eps=1e-5)
    d.update(kw)
    return ctypes.byref(pkg._lib.TmoeBlockNorm(**d))


def test_norm_abi_refuses(pkg):
    L = pkg._lib.lib()
    ws = L.tmoe_block_norm_workspace_bytes(40, 64, 0)
    assert ws > 0 and L.tmoe_block_norm_workspace_bytes(4, 20000, 0) == 0
    assert L.tmoe_block_norm_workspace_bytes(4, 64, 5) == 0

    def fwd(n, r=OK, h=OK, inv=OK):
        return L.tmoe_block_norm_forward(n, r, h, inv, None)

    def bwd(n, inv=OK, dr=OK, drs=64, dh=OK, dhs=64, out=(OK,) * 6, ws_=OK, nws=None):
        return L.tmoe_block_norm_backward(n, inv, dr, drs, dh, dhs, *out, ws_, ws if nws is None else nws, None)
    for kw, code in ((dict(dtype=2), -1), (dict(T=-1), -1), (dict(d=0), -1), (dict(d=20000), -2),
                     (dict(T=1 << 31), -2), (dict(eps=-1.0), -1), (dict(eps=math.nan), -1), (dict(y=None), -1),
                     (dict(x_stride=63), -1), (dict(gate_stride=0), -1), (dict(x=OK + 1), -1),
                     (dict(gamma=OK + 2), -1)):
        assert fwd(_norm(pkg, **kw)) == code, kw
        assert bwd(_norm(pkg, **kw)) == code, kw
    n = _norm(pkg)
    assert fwd(None) == -1 and bwd(None) == -1
    assert fwd(n, h=None) == -1 and fwd(_norm(pkg, next_weight=None)) == -1
    assert fwd(_norm(pkg, next_weight=None), r=None, h=None) == -1
    assert fwd(n, r=OK + 1) == -1 and fwd(n, inv=OK + 2) == -1
    assert bwd(n, inv=None) == -1 and bwd(n, drs=1) == -1 and bwd(n, dhs=1) == -1
    assert bwd(n, nws=ws - 1) == -1 and bwd(n, ws_=None) == -1
    for kw in (dict(x=None), dict(gate=None), dict(post_weight=None), dict(gamma=None), dict(next_weight=None)):
        assert bwd(_norm(pkg, **kw)) == -1, kw
    assert fwd(_norm(pkg, T=0, y=None)) == 0


def test_adamw_abi_refuses(pkg):
    L, lib = pkg._lib.lib(), pkg._lib

    def call(t=None, count=1, **kw):
        d = dict(lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.1, step=1, dtype=0, state_bits=32)
        d.update(kw)
        q = dict(p=OK, g=OK, m=OK, v=OK, m_scale=OK, v_scale=OK, n=4)
        q.update(t or {})
        return L.tmoe_adamw_step(ctypes.byref(lib.TmoeAdamwTensor(**q)), count, ctypes.byref(lib.TmoeAdamwStep(**d)),
                                 None)
    for kw in (dict(dtype=2), dict(state_bits=16), dict(beta1=1.0), dict(beta2=-0.1), dict(eps=-1.0),
               dict(lr=math.nan), dict(lr=math.inf), dict(weight_decay=-1.0), dict(step=0), dict(step_dev=OK + 4),
               dict(count=-1)):
        assert call(**kw) == -1, kw
    for t in (dict(n=-1), dict(p=None), dict(g=None), dict(m=None), dict(v=None), dict(p=OK + 2), dict(m=OK + 1)):
        assert call(t) == -1, t
    assert call(dict(m_scale=None), state_bits=8) == -1
    assert call(dict(n=(1 << 36) + 1)) == -2
    assert call(dict(n=0, p=None)) == 0 and L.tmoe_adamw_step(None, 1, None, None) == -1


def test_python_entry_points_refuse(pkg):
    x, w = torch.randn(4, 8), torch.ones(8)
    cases = [
        (lambda: pkg.fused_router(x, 2, 0.5), "HIP devices only"),
        (lambda: pkg.fused_router(x, 9, 0.5), "top_k"),
        (lambda: pkg.fused_router(x, 0, 0.5), "top_k"),
        (lambda: pkg.fused_router(torch.randn(2, 300), 2, 0.5), "256"),
        (lambda: pkg.fused_router(x[0], 2, 0.5), "raw"),
        (lambda: pkg.fused_router(x.double(), 2, 0.5), "dtype"),
        (lambda: pkg.fused_router(x, 2, 0.0), "temperature"),
        (lambda: pkg.fused_router(x, 2, 0.5, scale=-1), "scale"),
        (lambda: pkg.fused_router(x, 2, 0.5, mask=torch.ones(4)), "mask"),
        (lambda: pkg.fused_router(x, 2, 0.5, mask=torch.ones(3, dtype=torch.bool)), "mask"),
        (lambda: pkg.fused_block_norm(x, x), "HIP devices only"),
        (lambda: pkg.fused_block_norm(), "x or y"),
        (lambda: pkg.fused_block_norm(x), "next_weight"),
        (lambda: pkg.fused_block_norm(x, gamma=w, next_weight=w), "next_weight"),
        (lambda: pkg.fused_block_norm(x, x[:3]), "shapes"),
        (lambda: pkg.fused_block_norm(y=x, gate=x[:, :1]), "shapes"),
        (lambda: pkg.fused_block_norm(x, x, gamma=torch.ones(7)), "weight"),
        (lambda: pkg.fused_block_norm(x, x, gamma=torch.ones(8, 1)), "weight"),
        (lambda: pkg.fused_block_norm(x, x, gamma=w.bfloat16()), "dtypes"),
        (lambda: pkg.fused_block_norm(x.half(), x.half()), "dtype"),
        (lambda: pkg.fused_block_norm(x, x, eps=-1e-5), "eps"),
        (lambda: pkg.fused_block_norm(y=torch.randn(1, 16385)), "16384"),
        (lambda: pkg.fused_block_norm(y=torch.tensor(1.0)), "d"),
    ]
    for f, msg in cases:
        with pytest.raises(RuntimeError, match=msg):
            f()
    with pytest.raises(TypeError):
        pkg.fused_block_norm(x, 3.0)


def test_adamw_python_refuses(pkg):
    def t(*shape, dtype=torch.float32):
        return torch.zeros(*shape, dtype=dtype)

    def step(p, g, m, v, **kw):
        pkg.adamw_step(p, g, m, v, **{**dict(step=1, lr=1e-3), **kw})
    p = t(4, 8)
    for args, kw, msg in [
        (([p], [t(4, 8)], [t(4, 8)], [t(4, 8)]), {}, "HIP devices only"),
        (([p], [t(4, 7)], [t(4, 8)], [t(4, 8)]), {}, "gradient"),
        (([p], [t(4, 8, dtype=torch.bfloat16)], [t(4, 8)], [t(4, 8)]), {}, "gradient"),
        (([p], [t(4, 8).to_sparse()], [t(4, 8)], [t(4, 8)]), {}, "sparse"),
        (([p], [t(4, 8)], [t(8, 4).t()], [t(4, 8)]), {}, "laid out"),
        (([p], [t(4, 8)], [t(4, 8, dtype=torch.bfloat16)], [t(4, 8)]), {}, "laid out"),
        (([t(4, 16)[:, ::2]], [t(4, 8)], [t(4, 8)], [t(4, 8)]), {}, "gaps"),
        (([p, p], [t(4, 8)] * 2, [t(4, 8), t(4, 8)], [t(4, 8), t(4, 8)]), {}, "share memory"),
        (([p], [t(4, 8)], [p], [t(4, 8)]), {}, "share memory"),
        (([p], [t(4, 8)], [t(4, 8)], []), {}, "for 1 parameters"),
        (([p], [t(4, 8)], [t(4, 8)], [t(4, 8)]), dict(step=0), "step"),
        (([p], [t(4, 8)], [t(4, 8)], [t(4, 8)]), dict(step=torch.tensor(1.0)), "step"),
        (([t(4, 8, dtype=D)], [t(4, 8, dtype=D)], [t(4, 8)], [t(4, 8)]), {}, "dtype"),
    ]:
        with pytest.raises(RuntimeError, match=msg):
            step(*args, **kw)
    with pytest.raises(ValueError):
        step([p], [p], [p], [p], betas=(1.0, 0.9))
    with pytest.raises(ValueError):
        step([p], [p], [p], [p], lr=-1.0)
    with pytest.raises(TypeError):
        step(p, [p], [p], [p])
    step([], [], [], [])        # nothing to do
    q8 = dict(step=1, lr=1e-3)
    codes, sc = lambda: t(32, dtype=torch.uint8), lambda n=1: t(n)
    with pytest.raises(RuntimeError, match="scales"):
        pkg.adamw_step_8bit([p], [t(4, 8)], [codes()], [sc(2)], [codes()], [sc()], **q8)
    with pytest.raises(RuntimeError, match="codes"):
        pkg.adamw_step_8bit([p], [t(4, 8)], [codes()[:31]], [sc()], [codes()], [sc()], **q8)
    with pytest.raises(RuntimeError, match="HIP devices only"):
        pkg.adamw_step_8bit([p], [t(4, 8)], [codes()], [sc()], [codes()], [sc()], **q8)
    for kw in (dict(state_bits=16), dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(eps=-1.0)):
        with pytest.raises(ValueError):
            pkg.FusedAdamW([torch.nn.Parameter(p)], **kw)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_optimizer_state_keeps_its_dtypes(pkg, monkeypatch, bits, dtype):
    """state_dict -> load_state_dict gives the same states bit for bit (torch would cast them
    to the parameter's dtype), and the count goes on from there. The step itself is a stand-in."""
    import mamba_tuckermoe_amd.adamw as ad
    seen = []
    monkeypatch.setattr(ad, "_run", lambda *a: seen.append(a))

    def make():
        torch.manual_seed(1)
        ps = [torch.nn.Parameter(torch.randn(300, 3).to(dtype)), torch.nn.Parameter(torch.randn(5).to(dtype))]
        for p in ps:
            p.grad = torch.ones_like(p)
        return ps, pkg.FusedAdamW(ps, state_bits=bits)
    ps, opt = make()
    opt.step()
    opt.step()
    assert [a[6] for a in seen] == [1, 2] and len(seen[0][0]) == 2
    for p in ps:
        for k, v in opt.state[p].items():
            if isinstance(v, torch.Tensor):
                (v.view(torch.uint8) if v.element_size() == 1 else v).fill_(3)
    ps2, opt2 = make()
    opt2.load_state_dict(opt.state_dict())
    for p, q in zip(ps, ps2):
        a, b = opt.state[p], opt2.state[q]
        assert set(a) == set(b) and b["step"] == 2
        for k, v in a.items():
            if isinstance(v, torch.Tensor):
                assert b[k].dtype == v.dtype and b[k].data_ptr() != v.data_ptr()
                assert torch.equal(v.view(torch.uint8), b[k].view(torch.uint8))
    opt2.step()
    assert seen[-1][6] == 3
    # a parameter that comes later counts from its own first step
    late = torch.nn.Parameter(torch.randn(4).to(dtype))
    opt2.add_param_group({"params": [late]})
    late.grad = torch.ones_like(late)
    opt2.step()
    assert sorted(a[6] for a in seen[-2:]) == [1, 4]


def test_block_train_shares_the_inference_blocks_parameters(pkg):
    cfg = pkg.TuckerMoEConfig(kmoe_num_experts=4, kmoe_r1=4, kmoe_r2=64, kmoe_r3=64)
    a, b = pkg.TuckerFFNTrain(64, cfg), pkg.TuckerFFN(64, cfg)
    assert set(a.state_dict()) == set(b.state_dict())
    b.load_state_dict(a.state_dict())


def test_training_layer_mask_needs_the_fused_router(pkg):
    m = pkg.TuckerMoETrain(64, 48, num_experts=4, r2=64, r3=64)
    with pytest.raises(RuntimeError, match="fused_router"):
        m(torch.randn(3, 64), mask=torch.ones(3, dtype=torch.bool))


def _counting(pkg, monkeypatch):
    """The module with a stand-in for its launch, and what that was called with: a list of
    (parameters' ids, step)."""
    import mamba_tuckermoe_amd.adamw as ad
    seen = []
    monkeypatch.setattr(ad, "_run", lambda *a: seen.append(([id(p) for p in a[0]], int(a[6]))))
    return ad, seen


def _step_of(opt, params, on):
    for p, o in zip(params, on):
        p.grad = torch.ones_like(p) if o else None
    opt.step()


@pytest.mark.parametrize("reload", [False, True])
def test_optimizer_counts_follow_the_parameter(pkg, monkeypatch, reload):
    """A parameter without a gradient rests: its count and its bias corrections stand still, on
    the device as on the host, also where it began with others or was loaded with them."""
    _, seen = _counting(pkg, monkeypatch)
    pattern = [(1, 1, 0), (0, 1, 0), (1, 1, 1), (1, 0, 1), (1, 0, 0), (0, 1, 1), (1, 1, 1), (1, 1, 1)]
    runs = []
    for capturable in (False, True):
        ps = [torch.nn.Parameter(torch.ones(3)) for _ in range(3)]
        opt = pkg.FusedAdamW([{"params": ps[:2]}, {"params": ps[2:]}], capturable=capturable)
        took, got = [0, 0, 0], []
        for i, on in enumerate(pattern):
            seen.clear()
            _step_of(opt, ps, on)
            took = [a + b for a, b in zip(took, on)]
            steps = {q: n for ids, n in seen for q in ids}
            assert steps == {id(p): n for p, n, o in zip(ps, took, on) if o}, (capturable, i)
            assert [int(opt.state[p]["step"]) if p in opt.state else 0 for p in ps] == took
            if reload:
                opt.load_state_dict(opt.state_dict())
        runs.append(took)
    assert runs[0] == runs[1]


def test_optimizer_refuses_to_part_captured_counts(pkg, monkeypatch):
    """What a captured step counts together, a step of some of them cannot part; nor can a
    capture of some of those that stepped together. Nothing changes where it is refused."""
    ad, seen = _counting(pkg, monkeypatch)
    ps = [torch.nn.Parameter(torch.ones(3)) for _ in range(2)]
    opt = pkg.FusedAdamW(ps, capturable=True)
    _step_of(opt, ps, (1, 1))
    monkeypatch.setattr(ad, "_capturing", lambda d: True)
    with pytest.raises(RuntimeError, match="before the capture"):
        _step_of(opt, ps, (1, 0))
    _step_of(opt, ps, (1, 1))
    monkeypatch.setattr(ad, "_capturing", lambda d: False)
    with pytest.raises(RuntimeError, match="captured together"):
        _step_of(opt, ps, (0, 1))
    assert len(seen) == 2 and [int(opt.state[p]["step"]) for p in ps] == [2, 2]
    _step_of(opt, ps, (1, 1))
    opt.load_state_dict(opt.state_dict())
    _step_of(opt, ps, (0, 1))
    assert [int(opt.state[p]["step"]) for p in ps] == [3, 4]
    monkeypatch.setattr(ad, "_capturing", lambda d: True)      # parted: each its own
    _step_of(opt, ps, (0, 1))
    monkeypatch.setattr(ad, "_capturing", lambda d: False)
    _step_of(opt, ps, (1, 0))
    assert [int(opt.state[p]["step"]) for p in ps] == [4, 5]


@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_makes_no_state_in_a_capture(pkg, monkeypatch, bits):
    """State made inside a capture would be cleared by every replay, or, where the step is
    refused, never: a first step there is refused and leaves nothing behind, for any group."""
    ad, seen = _counting(pkg, monkeypatch)
    for capturable, msg in ((True, "first step"), (False, "capturable")):
        ps = [torch.nn.Parameter(torch.ones(300)) for _ in range(2)]
        opt = pkg.FusedAdamW([{"params": ps[:1]}, {"params": ps[1:]}], state_bits=bits, capturable=capturable)
        monkeypatch.setattr(ad, "_capturing", lambda d: True)
        with pytest.raises(RuntimeError, match=msg):
            _step_of(opt, ps, (1, 1))
        assert not opt.state and not seen
        monkeypatch.setattr(ad, "_capturing", lambda d: False)
        _step_of(opt, ps, (1, 0))
        monkeypatch.setattr(ad, "_capturing", lambda d: True)
        seen.clear()
        with pytest.raises(RuntimeError, match=msg):      # the second group's
            _step_of(opt, ps, (1, 1))
        assert list(opt.state) == [ps[0]] and not seen and int(opt.state[ps[0]]["step"]) == 1
        monkeypatch.setattr(ad, "_capturing", lambda d: False)
        _step_of(opt, ps, (1, 1))
        assert [int(opt.state[p]["step"]) for p in ps] == [2, 1]
        seen.clear()
    # a capture that was refused for one group has captured no other's counts
    ps = [torch.nn.Parameter(torch.ones(3)) for _ in range(3)]
    opt = pkg.FusedAdamW([{"params": ps[:2]}, {"params": ps[2:]}], state_bits=bits, capturable=True)
    _step_of(opt, ps, (1, 1, 0))
    monkeypatch.setattr(ad, "_capturing", lambda d: True)
    with pytest.raises(RuntimeError, match="first step"):
        _step_of(opt, ps, (1, 1, 1))
    monkeypatch.setattr(ad, "_capturing", lambda d: False)
    _step_of(opt, ps, (0, 1, 0))
    assert [int(opt.state[p]["step"]) for p in ps[:2]] == [1, 2]


def test_forward_mode_is_refused(pkg):
    """An operand with a tangent: the outputs would have none, a derivative of zero."""
    import torch.autograd.forward_ad as fw
    x, w, ones = torch.randn(4, 8), torch.ones(8), lambda: torch.ones(4, 8)
    with fw.dual_level():
        def dual(t):
            return fw.make_dual(t, torch.ones_like(t))
        norm = dict(x=x, y=x, gate=x, post_weight=w, gamma=w, next_weight=w)
        calls = [lambda: pkg.fused_router(dual(x), 2, 0.5), lambda: pkg.fused_block_norm(dual(x), next_weight=w),
                 lambda: pkg.adamw_step([dual(ones())], [ones()], [ones()], [ones()], step=1, lr=1.0),
                 lambda: pkg.adamw_step([ones()], [dual(ones())], [ones()], [ones()], step=1, lr=1.0)]
        calls += [lambda k=k: pkg.fused_block_norm(**{**norm, k: dual(norm[k])}) for k in norm]
        for f in calls:
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                f()
            with torch.no_grad(), pytest.raises(RuntimeError, match="no forward-mode derivative"):
                f()
        with torch.inference_mode(), pytest.raises(RuntimeError, match="HIP devices only"):
            pkg.fused_router(dual(x), 2, 0.5)       # where no tangent is asked for
    with pytest.raises(RuntimeError, match="HIP devices only"):
        pkg.fused_router(x, 2, 0.5)


def test_adamw_gradients_that_overlap_what_is_written(pkg):
    """A gradient in the memory of a parameter or a state at another offset would be read after
    it is written, or before; the very elements that are written are fine, and so is a
    gradient in another order, which is copied first."""
    def step(p, g, m, v, msg):
        with pytest.raises(RuntimeError, match=msg):
            pkg.adamw_step(p, g, m, v, step=1, lr=1e-3)

    def z(n=32):
        return torch.zeros(n)
    a = z(128)
    for o, bad in ((1, True), (31, True), (-1, True), (32, False), (-32, False), (0, False)):
        g = a[48 + o:80 + o]
        msg = "a gradient shares memory" if bad else "HIP devices only"
        step([a[48:80]], [g], [z()], [z()], msg)
        step([z()], [g], [a[48:80]], [z()], msg)
        step([z()], [g], [z()], [a[48:80]], msg)
        step([z(), a[48:80], z()], [z(), z(), g], [z(), z(), z()], [z(), z(), z()],
             "a gradient shares memory" if bad or o == 0 else "HIP devices only")
    sq = z(64).view(8, 8)
    step([sq], [sq.t()], [z(64).view(8, 8)], [z(64).view(8, 8)], "HIP devices only")
    g = z()
    step([z(), z()], [g, g], [z(), z()], [z(), z()], "HIP devices only")     # one that two share
    codes, sc = torch.zeros(64, dtype=torch.uint8), z(1)
    for g in (codes.view(torch.float32)[1:9], codes.view(torch.float32)[:8]):
        with pytest.raises(RuntimeError, match="a gradient shares memory"):
            pkg.adamw_step_8bit([z(8)], [g], [codes[:8]], [sc], [codes[8:16]], [z(1)], step=1, lr=1e-3)
    with pytest.raises(RuntimeError, match="a gradient shares memory"):
        pkg.adamw_step_8bit([z(1)], [sc], [codes[:1]], [sc], [codes[8:9]], [z(1)], step=1, lr=1e-3)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("capturable", [False, True])
def test_optimizer_takes_up_torchs_adamw(pkg, monkeypatch, capturable, dtype):
    """A torch.optim.AdamW's state: its moments in float32 and the parameter's layout, its counts
    and its numbers; the next step is the one after its last."""
    _, seen = _counting(pkg, monkeypatch)
    torch.manual_seed(2)
    ps = [torch.nn.Parameter(torch.randn(5, 7).to(dtype)), torch.nn.Parameter(torch.randn(3).to(dtype))]
    topt = torch.optim.AdamW([{"params": ps[:1], "lr": 0.5}, {"params": ps[1:]}], lr=2e-3, weight_decay=0.3,
                             capturable=False)
    for on in ((1, 1), (1, 0), (1, 1)):
        for p, o in zip(ps, on):
            p.grad = torch.randn_like(p) if o else None
        topt.step()
    qs = [torch.nn.Parameter(torch.zeros(7, 5, dtype=dtype).t()), torch.nn.Parameter(torch.zeros(3, dtype=dtype))]
    opt = pkg.FusedAdamW([{"params": qs[:1]}, {"params": qs[1:]}], seed=9, capturable=capturable)
    sd = topt.state_dict()
    for g in sd["param_groups"]:
        g["capturable"] = capturable
    opt.load_state_dict(sd)
    assert [(g["lr"], g["weight_decay"], g["state_bits"], g["seed"], g["capturable"]) for g in opt.param_groups] == [
        (0.5, 0.3, 32, 9, capturable), (2e-3, 0.3, 32, 9, capturable)]
    for p, q in zip(ps, qs):
        for k in ("exp_avg", "exp_avg_sq"):
            t = opt.state[q][k]
            assert t.dtype == torch.float32 and t.stride() == q.stride() and not t.requires_grad
            assert torch.equal(t, topt.state[p][k].float())
        q.grad = torch.ones_like(q)
    opt.step()
    assert [(ids, n) for ids, n in seen] == [([id(qs[0])], 4), ([id(qs[1])], 3)]
    assert [int(opt.state[q]["step"]) for q in qs] == [4, 3]


def test_optimizer_refuses_other_states(pkg):
    """... at the load, which changes nothing."""
    def saved(cls, **kw):
        p = torch.nn.Parameter(torch.ones(300))
        p.grad = torch.ones_like(p)
        opt = cls([p], **kw)
        opt.step()
        return opt.state_dict()
    adamw = torch.optim.AdamW
    short = saved(adamw)
    short["state"][0]["exp_avg"] = torch.ones(1)
    for bits, sd, msg in ((8, saved(adamw), "state_bits 8"), (32, saved(torch.optim.SGD, lr=0.1, momentum=0.9), "state_bits 32"),
                          (32, saved(adamw, amsgrad=True), "amsgrad"), (32, saved(adamw, maximize=True), "maximize"),
                          (32, short, "exp_avg"),
                          (32, saved(torch.optim.Adam, weight_decay=0.1), "L2")):
        p = torch.nn.Parameter(torch.ones(300))
        opt = pkg.FusedAdamW([p], lr=0.125, state_bits=bits)
        with pytest.raises(ValueError, match=msg):
            opt.load_state_dict(sd)
        assert not opt.state and opt.param_groups[0]["lr"] == 0.125 and opt.param_groups[0]["state_bits"] == bits
    two = [torch.nn.Parameter(torch.ones(3)) for _ in range(2)]
    with pytest.raises(ValueError):
        pkg.FusedAdamW([{"params": two[:1]}, {"params": two[1:]}]).load_state_dict(saved(adamw))


@pytest.mark.parametrize("capturable", [False, True])
def test_optimizer_refused_step_is_not_counted(pkg, monkeypatch, capturable):
    """A step that the call refuses leaves the counts of what it did not launch."""
    import mamba_tuckermoe_amd.adamw as ad
    fail, seen = [], []

    def run(params, *a):
        if any(p is q for p in params for q in fail):
            raise RuntimeError("refused")
        seen.append(int(a[5]))
    monkeypatch.setattr(ad, "_run", run)
    ps = [torch.nn.Parameter(torch.ones(3)), torch.nn.Parameter(torch.ones(3).bfloat16())]
    opt = pkg.FusedAdamW([{"params": ps[:1]}, {"params": ps[1:]}], capturable=capturable)
    _step_of(opt, ps, (1, 1))
    fail.append(ps[1])
    for _ in range(2):
        with pytest.raises(RuntimeError, match="refused"):
            _step_of(opt, ps, (0, 1))
    assert [int(opt.state[p]["step"]) for p in ps] == [1, 1]
    with pytest.raises(RuntimeError, match="refused"):
        _step_of(opt, ps, (1, 1))
    assert [int(opt.state[p]["step"]) for p in ps] == [2, 1]      # the first group's was launched
    fail.clear()
    _step_of(opt, ps, (0, 1))
    assert seen == [1, 1, 2, 2] and [int(opt.state[p]["step"]) for p in ps] == [2, 2]


def test_optimizer_checks_each_groups_own_values(pkg):
    def p():
        return [torch.nn.Parameter(torch.ones(3))]
    for kw in (dict(state_bits=16), dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(eps=-1.0), dict(weight_decay=-0.1),
               dict(lr=math.nan)):
        with pytest.raises(ValueError, match="FusedAdamW"):
            pkg.FusedAdamW([{"params": p()}, {"params": p(), **kw}])
        opt = pkg.FusedAdamW(p())
        with pytest.raises(ValueError, match="FusedAdamW"):
            opt.add_param_group({"params": p(), **kw})
        assert len(opt.param_groups) == 1
        with pytest.raises(ValueError, match="FusedAdamW"):      # defaults, even where no group uses them
            pkg.FusedAdamW([{"params": p(), "state_bits": 8, "lr": 1.0, "betas": (0.9, 0.9), "eps": 1e-8,
                             "weight_decay": 0.0}], **kw)
    assert pkg.FusedAdamW([{"params": p(), "state_bits": 8}]).param_groups[0]["state_bits"] == 8
