"""The training operators around the expert contraction on the GPU against the float64 oracle
(oracle/train_ops_np.py).

Tolerances: a float32 evaluation of n rounded steps is off by at most n 2^-24 times the sum of
its terms' magnitudes (the oracle's *_mag), and a result stored in bfloat16 by another half
step, 2^-8 of itself. n: a norm's value is made of under 64 operations on top of a sum over a
row, whose longest chain is 64 elements of a thread, 6 exchanges in a wave and 16 waves; a
column's sum adds its rows' chain (under T / 4) and 80 planes. In the router the capped logit
is cap times a tanh that is off by under 8 steps, and enters an exponential twice over tau."""
import numpy as np
import pytest
import torch

from oracle import train_ops_np as tn
from oracle import tucker_moe_np as onp
from test_train_ops import NORM_FORMS, norm_inputs

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
dtypes = pytest.mark.parametrize("dtype", list(DTYPES.values()), ids=list(DTYPES))


def f64(t):
    return t.detach().double().cpu().numpy()


def near(got, want, mag, n, what=""):
    """got within n steps of float32 (and its own rounding) of want."""
    g = f64(got)
    tol = n * U * np.abs(mag) + 1e-37
    if got.dtype == torch.bfloat16:
        tol = tol * (1 + 2.0 ** -8) + 2.0 ** -8 * np.abs(want) + 1e-38
    bad = ~(np.abs(g - want) <= tol)
    assert not bad.any(), (what, int(bad.sum()), float(np.max(np.abs(g - want) / tol)))


# ---- router ---------------------------------------------------------------------

def _logits(B, E, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(B, E, generator=g) * 3 + torch.randn(B, 1, generator=g) * 4).to(dtype)


def _check_router(pkg, raw, k, tau, cap, mask, seed, call=None):
    B, E = raw.shape
    g = torch.Generator().manual_seed(seed + 1)
    dw, dlb, dz = torch.randn(B, k, generator=g), torch.tensor(0.7), torch.tensor(0.05)
    leaf = raw.detach().requires_grad_()
    r = call(leaf) if call else pkg.fused_router(leaf, k, tau, cap, mask)
    draw, = torch.autograd.grad((r.weights, r.lb_loss, r.z_loss), leaf,
                                (dw.to(raw.device), dlb.to(raw.device), dz.to(raw.device)))
    assert draw.dtype == raw.dtype and r.idx.dtype == r.counts.dtype == torch.int64
    tau = float(tau)
    o = tn.router(f64(raw), k, tau, cap, None if mask is None else mask.cpu().numpy(), dw.numpy(), 0.7, 0.05)
    n = 16 * cap / tau + 128
    assert np.array_equal(r.idx.cpu().numpy(), o["idx"])
    assert np.array_equal(r.counts.cpu().numpy(), o["counts"])
    near(r.weights, o["w"], o["w"], n, "w")
    near(r.lb_loss, o["lb"], o["lb"], n, "lb")
    near(r.z_loss, o["z"], 2 * np.sqrt(o["z"]) * (8 * cap + 32) + 16 * o["z"], 1, "z")
    near(draw, o["draw"], o["draw_mag"], 4 * n, "draw")


@dtypes
@pytest.mark.parametrize("B,E,k,tau,padded", [
    (1, 1, 1, 0.5, 0), (1, 8, 2, 0.5, 0), (5, 3, 3, 2.0, 0), (257, 8, 2, 1.1, 0.3), (1000, 33, 5, 0.5, 0.5),
    (4096, 16, 2, 2.0, 0), (333, 64, 16, 0.9, 0.1), (129, 100, 4, 1.0, 0), (70, 256, 8, 0.5, 0.2),
    (20001, 8, 2, 0.5, 0.25), (300, 255, 16, 1.5, 0)])
def test_router(pkg, dev, B, E, k, tau, padded, dtype):
    mask = None
    if padded:
        mask = (torch.rand(B, generator=torch.Generator().manual_seed(B)) >= padded).to(dev)
    _check_router(pkg, _logits(B, E, dtype, B + E).to(dev), k, tau, 10.0, mask, B)


def test_router_strides_cap_and_no_grad(pkg, dev):
    wide = _logits(77, 40, torch.float32, 3).to(dev)
    for raw in (wide[:, 8:24], wide[:, 1:12], wide.t()[:, :30], wide[::3, :16], wide[:1].expand(9, 40)):
        _check_router(pkg, raw, 2, 0.7, 4.0, None, 5)
    mask = (torch.arange(154, device=dev) % 3 > 0)[::2]
    _check_router(pkg, wide, 3, 0.7, 30.0, mask, 5)
    with torch.no_grad():
        a = pkg.fused_router(wide.requires_grad_(), 2, 0.5)
    b = pkg.fused_router(wide, 2, 0.5)
    assert not a.weights.requires_grad and b.weights.requires_grad and not b.idx.requires_grad
    for x, y in zip(a, b):
        assert torch.equal(x, y)


def test_router_ties_and_extremes(pkg, dev):
    """Equal logits: the lowest index; infinities; logits far past the cap, which is flat there
    in float32 but whose order is the logits' own; -0 is 0."""
    inf = float("inf")
    raw = torch.tensor([[1.0, 3, 3, 2, 3, 3, -1, 3], [0.0, -0.0, 0, 0, -0.0, 0, 0, 0],
                        [500.0, 400, 900, 800, 1e30, 3e38, 2, 1], [-inf, -inf, 5, -inf, 4, -inf, -inf, -inf],
                        [inf, 0, inf, 1, 2, 3, 4, 5], [-inf] * 8, [-1e30] * 7 + [-2e30]], device=dev)
    for dt in DTYPES.values():
        _check_router(pkg, raw.to(dt), 3, 0.5, 10.0, None, 1)


@dtypes
@pytest.mark.parametrize("E,k", [(4, 4), (8, 8), (11, 11), (37, 16), (64, 6), (100, 16), (256, 16)])
def test_router_near_ties_and_padding(pkg, dev, E, k, dtype):
    """Logits a few places apart or equal, over all lanes of a token and in tokens of one wave
    with others that are not; rows of -inf beside widths that no lane count divides."""
    g = torch.Generator().manual_seed(E)
    B = 200
    raw = _logits(B, E, torch.float32, E)
    near_ = (torch.full((B, E), 1.0).view(torch.int32) + torch.randint(0, 400, (B, E), generator=g).int()).view(torch.float32)
    raw[::2] = near_[::2] * torch.where(torch.rand(B, 1, generator=g) < 0.5, -1.0, 1.0)[::2]
    raw[1::6] = torch.randint(0, 3, (B, E), generator=g).float()[1::6]
    raw[3] = -float("inf")
    raw[5, : E // 2] = -float("inf")
    raw[9, E // 2:] = -float("inf")
    mask = (torch.rand(B, generator=g) < 0.8).to(dev)
    mask[torch.tensor([3, 5, 9])] = True
    _check_router(pkg, raw.to(dtype).to(dev), k, 0.9, 10.0, mask, 4)


def test_router_no_tokens(pkg, dev):
    """No tokens, and none that the mask leaves: zero losses, counts and gradients; what the
    left-out rows hold does not matter, and a NaN row spoils its own row alone."""
    r = pkg.fused_router(torch.empty(0, 8, device=dev).requires_grad_(), 2, 0.5)
    assert r.idx.shape == (0, 2) and r.lb_loss.item() == r.z_loss.item() == 0 and not r.counts.any()
    assert torch.autograd.grad(r.lb_loss + r.z_loss + r.weights.sum(), r.weights.grad_fn.next_functions[0][0].variable)[
        0].shape == (0, 8)
    raw = torch.full((5, 8), float("nan"), device=dev).requires_grad_()
    r = pkg.fused_router(raw, 2, 0.5, mask=torch.zeros(5, dtype=torch.bool, device=dev))
    d, = torch.autograd.grad(r.lb_loss + r.z_loss + r.weights.sum(), raw)
    assert r.lb_loss.item() == r.z_loss.item() == 0 and not r.counts.any() and not d.any()
    assert (r.idx == -1).all() and not r.weights.any()
    raw = _logits(300, 8, torch.float32, 2).to(dev)
    mask = torch.ones(300, dtype=torch.bool, device=dev)
    mask[7] = mask[250] = False
    raw[7], raw[250, 3] = float("nan"), float("inf")
    _check_router(pkg, raw, 2, 0.5, 10.0, mask, 3)
    r = pkg.fused_router(raw, 2, 0.5)                       # row 7 counts now
    assert r.idx[7].tolist() == [0, 1] and r.weights[7].isnan().all()
    assert r.weights[torch.arange(300, device=dev) != 7].isfinite().all()
    raw[7] = 0.0
    raw[7, 5] = float("nan")                                # a NaN ranks first
    assert pkg.fused_router(raw, 2, 0.5).idx[7].tolist() == [5, 0]


def test_router_partial_gradients(pkg, dev):
    """Each of the three alone; a temperature on the device; weights' gradient strided."""
    raw = _logits(200, 8, torch.float32, 9).to(dev).requires_grad_()
    tau = torch.tensor(0.8, device=dev)
    _check_router(pkg, raw, 2, tau, 10.0, None, 4)
    r = pkg.fused_router(raw, 2, torch.tensor(0.8))          # on the CPU: a number
    s = pkg.fused_router(raw, 2, 0.8)
    assert torch.equal(r.weights, s.weights)
    dw = torch.randn(2, 200, device=dev).t()
    for i, (out, seed) in enumerate(((r.weights, dw), (r.lb_loss, None), (r.z_loss, None))):
        got, = torch.autograd.grad(out, raw, seed, retain_graph=True)
        z = [np.zeros((200, 2)), 0.0, 0.0]
        z[i] = f64(dw) if i == 0 else 1.0
        o = tn.router(f64(raw), 2, np.float64(np.float32(0.8)), 10.0, None, *z)
        near(got, o["draw"], o["draw_mag"], 4 * (160 / 0.8 + 128))


# ---- block norm -----------------------------------------------------------------

def _check_norm(pkg, n, dr, dh, eps=1e-5, shape=None):
    """n: operands on the device (any strides), checked forward and backward."""
    leaf = {k: v.detach().requires_grad_() for k, v in n.items()}
    r, h = pkg.fused_block_norm(**leaf, eps=eps)
    outs, seeds = [r], [dr]
    if h is not None:
        outs.append(h)
        seeds.append(dh)
    grads = torch.autograd.grad(outs, list(leaf.values()), seeds)
    d = n["y"].shape[-1]

    def flat(t):
        return f64(t).reshape(-1, d) if t.dim() != 1 or t.shape == n["y"].shape else f64(t)
    o = tn.block_norm(**{k: flat(v) for k, v in n.items()}, eps=eps, dr=flat(dr),
                      dh=flat(dh) if h is not None else None)
    T = n["y"].numel() // d
    steps = 64 + 64 + 6 + 16
    near(r.reshape(-1, d), o["r"], o["r_mag"], steps, "r")
    if h is not None:
        near(h.reshape(-1, d), o["h"], o["h_mag"], steps, "h")
    for k, g in zip(leaf, grads):
        assert g.dtype == n[k].dtype and g.shape == n[k].shape
        col = n[k].dim() == 1 and n[k].shape != n["y"].shape
        near(g if col else g.reshape(-1, d), o["d" + k], o["d" + k + "_mag"],
             2 * steps + (T / 4 + 80 if col else 0), "d" + k)
    with torch.no_grad():
        r2, h2 = pkg.fused_block_norm(**leaf, eps=eps)
    assert torch.equal(r, r2) and (h is None or torch.equal(h, h2)) and not r2.requires_grad


@dtypes
@pytest.mark.parametrize("form", NORM_FORMS, ids="+".join)
def test_norm_forms(pkg, dev, form, dtype):
    for T, d in ((1, 768), (37, 320), (19, 1001), (4, 2304)):
        n, dr, dh = norm_inputs(form, T, d, T, dtype)
        _check_norm(pkg, {k: v.to(dev) for k, v in n.items()}, dr.to(dev), dh.to(dev))


@dtypes
@pytest.mark.parametrize("T,d", [(1, 1), (2, 7), (3, 33), (5, 64), (130, 512), (67, 520), (33, 1024), (9, 1032),
                                 (2049, 768), (4100, 72), (5, 4608), (3, 8192), (2, 8200), (2, 9999), (3, 16384)])
def test_norm_sizes(pkg, dev, T, d, dtype):
    n, dr, dh = norm_inputs(NORM_FORMS[-1], T, d, T + d, dtype)
    _check_norm(pkg, {k: v.to(dev) for k, v in n.items()}, dr.to(dev), dh.to(dev))


@dtypes
@pytest.mark.parametrize("T,d", [(300, 6150), (5, 8192), (270, 9216), (7, 12290), (3, 16381)])
@pytest.mark.parametrize("form", [("y", "gate"), ("x", "y", "gamma", "next"), ("y", "gate", "post"),
                                  ("x", "y", "gate", "post", "next"), NORM_FORMS[-1]], ids="+".join)
def test_norm_wide_rows(pkg, dev, form, T, d, dtype):
    """Rows whose backward reads them twice, more of them than work-groups and fewer, the two
    halves of one projection."""
    n, dr, dh = norm_inputs(form, T, d, T + d, dtype)
    n = {k: v.to(dev) for k, v in n.items()}
    if "gate" in n:
        both = torch.cat([n["y"], n["gate"]], -1)
        n["y"], n["gate"] = both[:, :d], both[:, d:]
    _check_norm(pkg, n, dr.to(dev), dh.to(dev))


@dtypes
def test_norm_wide_rows_partial_gradients(pkg, dev, dtype):
    """One gradient at a time, and of one output alone, as all of them, bit for bit."""
    for form in (NORM_FORMS[-1], ("x", "y", "gamma", "next")):
        for d in (9216, 16384):
            n, dr, dh = norm_inputs(form, 4, d, d, dtype)
            n = {k: v.to(dev).requires_grad_() for k, v in n.items()}
            r, h = pkg.fused_block_norm(**n)
            dr, dh = dr.to(dev), dh.to(dev)
            full = torch.autograd.grad((r, h), list(n.values()), (dr, dh), retain_graph=True)
            for k, g in zip(n, full):
                one = torch.autograd.grad((r, h), n[k], (dr, dh), retain_graph=True)[0]
                assert torch.equal(one, g), (k, d)
            alone = torch.autograd.grad(h, list(n.values()), dh, retain_graph=True)
            zero = torch.autograd.grad((r, h), list(n.values()), (torch.zeros_like(r), dh))
            for k, a, b in zip(n, alone, zero):
                assert torch.equal(a, b), (k, d)


@dtypes
def test_norm_strides(pkg, dev, dtype):
    """Halves of one projection, rows at an odd stride, leading axes, a transposed operand, an
    expanded gradient: as the contiguous ones."""
    T, d = 24, 136
    n, dr, dh = norm_inputs(("x", "y", "gate", "gamma", "next"), T, d, 5, dtype)
    n = {k: v.to(dev) for k, v in n.items()}
    dr, dh = dr.to(dev), dh.to(dev)
    both = torch.cat([n["y"], n["gate"]], -1)
    odd = torch.zeros(T, d + 3, dtype=dtype, device=dev)
    odd[:, 1:d + 1] = n["x"]
    _check_norm(pkg, {**n, "y": both[:, :d], "gate": both[:, d:]}, dr, dh)
    _check_norm(pkg, {**n, "x": odd[:, 1:d + 1]}, dr, dh)
    _check_norm(pkg, {**n, "x": n["x"].t().contiguous().t()}, dr[:1].expand(T, d), dh)
    lead = {k: v.view(2, 3, 4, d) if v.dim() == 2 else v for k, v in n.items()}
    lead["y"], lead["gate"] = both.view(2, 3, 4, 2 * d)[..., :d], both.view(2, 3, 4, 2 * d)[..., d:]
    lead["x"] = n["x"].view(2, 3, 4, d).transpose(0, 1).contiguous().transpose(0, 1)
    _check_norm(pkg, lead, dr.view(2, 3, 4, d), dh.view(2, 3, 4, d))
    one = {k: v[0] if v.dim() == 2 else v for k, v in n.items()}
    _check_norm(pkg, one, dr[0], dh[0])
    w = torch.stack([n["gamma"], n["next_weight"]], -1)        # weights that are not contiguous
    _check_norm(pkg, {**n, "gamma": w[:, 0], "next_weight": w[:, 1]}, dr, dh)


def test_norm_first_block_and_partial_gradients(pkg, dev):
    """x alone with the next norm; gradients through r alone, h alone, of some operands only."""
    n, dr, dh = norm_inputs(("x", "y", "gamma", "next"), 50, 200, 8)
    n = {k: v.to(dev).requires_grad_() for k, v in n.items()}
    dr, dh = dr.to(dev), dh.to(dev)
    x, w = n["x"], n["next_weight"]
    r, h = pkg.fused_block_norm(x, next_weight=w)
    assert r is x
    dx, dw = torch.autograd.grad(h, (x, w), dh)
    o = tn.block_norm(y=f64(x), next_weight=f64(w), dr=np.zeros((50, 200)), dh=f64(dh))
    near(h, o["h"], o["h_mag"], 150)
    near(dx, o["dy"], o["dy_mag"], 300)
    near(dw, o["dnext_weight"], o["dnext_weight_mag"], 400)
    r, h = pkg.fused_block_norm(**n)
    zero = np.zeros((50, 200))
    for out, seed, a, b in ((r, dr, f64(dr), None), (h, dh, zero, f64(dh))):
        o = tn.block_norm(**{k: f64(v) for k, v in n.items()}, dr=a, dh=zero if b is None else b)
        grads = torch.autograd.grad(out, list(n.values()), seed, retain_graph=True)
        for k, g in zip(n, grads):
            near(g, o["d" + k], o["d" + k + "_mag"], 400, k)
    full = torch.autograd.grad((r, h), list(n.values()), (dr, dh), retain_graph=True)
    for k, g in zip(n, full):           # one at a time, the same bits
        assert torch.equal(torch.autograd.grad((r, h), n[k], (dr, dh), retain_graph=True)[0], g), k
    y = n["y"].detach()
    r, h = pkg.fused_block_norm(n["x"], y, gamma=n["gamma"].detach())
    assert torch.equal(torch.autograd.grad(r, n["x"], dr)[0], dr) and h is None


def test_norm_empty_and_extreme_rows(pkg, dev):
    n, dr, dh = norm_inputs(NORM_FORMS[-1], 0, 64, 1)
    leaf = {k: v.to(dev).requires_grad_() for k, v in n.items()}
    r, h = pkg.fused_block_norm(**leaf)
    assert r.shape == h.shape == (0, 64)
    for k, g in zip(leaf, torch.autograd.grad((r, h), list(leaf.values()), (r.detach(), h.detach()))):
        assert g.shape == leaf[k].shape and not g.any(), k
    # a row of zeros (rms = sqrt(eps)), huge and tiny rows, saturated gates
    n, dr, dh = norm_inputs(NORM_FORMS[-1], 6, 192, 2)
    for k in ("x", "y"):
        n[k][0] = 0
        n[k][1] *= 1e12
        n[k][2] *= 1e-12
    n["gate"][3], n["gate"][4] = 60.0, -60.0
    n["gate"][0, :5] = 0
    _check_norm(pkg, {k: v.to(dev) for k, v in n.items()}, dr.to(dev), dh.to(dev))
    # a row that is not finite leaves the others as they are
    m = {k: v.to(dev) for k, v in n.items()}
    r, h = pkg.fused_block_norm(**m)
    m["y"] = m["y"].clone()
    m["y"][5, 3] = float("nan")
    r2, h2 = pkg.fused_block_norm(**m)
    assert torch.equal(r[:5], r2[:5]) and torch.equal(h[:5], h2[:5]) and h2[5].isnan().all()


# ---- AdamW ----------------------------------------------------------------------

SHAPES = [(3,), (), (256,), (257,), (1,), (31, 33), (4, 64, 65), (1000, 130), (0, 5), (2, 255)]


def _adamw_inputs(dev, dtype, seed, shapes=SHAPES):
    g = torch.Generator().manual_seed(seed)
    p = [(torch.randn(s, generator=g) * 0.05).to(dtype).to(dev) for s in shapes]
    gr = [(torch.randn(s, generator=g) * 0.01).to(dtype).to(dev) for s in shapes]
    m = [(torch.randn(s, generator=g) * 0.003).to(dev) for s in shapes]
    v = [(torch.rand(s, generator=g) * 1e-4).to(dev) for s in shapes]
    return p, gr, m, v


HYPER = dict(lr=2e-3, betas=(0.9, 0.97), eps=1e-8, weight_decay=0.1)


def _oracle(p, g, m, v, step, h=HYPER):
    return tn.adamw(f64(p), f64(g), f64(m) if torch.is_tensor(m) else m, f64(v) if torch.is_tensor(v) else v, step,
                    h["lr"], *h["betas"], h["eps"], h["weight_decay"])


@dtypes
@pytest.mark.parametrize("step", [1, 7, 100000])
def test_adamw_32(pkg, dev, dtype, step):
    p, g, m, v = _adamw_inputs(dev, dtype, step)
    want = [_oracle(*t, step) for t in zip(p, g, m, v)]
    vers = [t._version for t in p]
    pkg.adamw_step(p, g, m, v, step=step, **HYPER)
    for i, o in enumerate(want):
        near(m[i], o["m"], o["m_mag"], 8, "m")
        near(v[i], o["v"], o["v_mag"], 8, "v")
        near(p[i], o["p"], o["p_mag"], 32, "p")
        assert p[i]._version > vers[i]


def test_adamw_layouts_and_many(pkg, dev):
    """Transposed parameters with gradients in another order, views at odd offsets, more tensors
    than one launch takes; a step count on the device."""
    shapes = [(5, 9)] * 130 + [(300, 7)]
    p, g, m, v = _adamw_inputs(dev, torch.float32, 4, shapes)
    p[0], m[0], v[0] = (t[0].t().contiguous().t() for t in (p, m, v))
    base = torch.zeros(200, device=dev)
    p[1] = base[1:46].view(5, 9)
    m[2] = torch.zeros(100, device=dev)[3:48].view(5, 9)
    want = [_oracle(*t, 12) for t in zip(p, g, m, v)]
    pkg.adamw_step(p, g, m, v, step=torch.tensor(12, device=dev), **HYPER)
    for i, o in enumerate(want):
        near(p[i], o["p"], o["p_mag"], 32, i)
        near(m[i], o["m"], o["m_mag"], 8, i)
    assert not base[0].any() and not base[46:].any()


def test_adamw_zero_gradient_and_nonfinite(pkg, dev):
    p, g, m, v = _adamw_inputs(dev, torch.float32, 5, [(700,)])
    g[0].zero_()
    m[0].zero_()
    v[0].zero_()
    q = p[0].clone()
    pkg.adamw_step(p, g, m, v, step=1, **HYPER)             # 0 / (0 + eps)
    assert torch.allclose(p[0], q * (1 - 2e-4), rtol=1e-6, atol=0) and not m[0].any()
    g[0][5] = float("nan")
    pkg.adamw_step(p, g, m, v, step=2, **HYPER)
    ok = torch.arange(700, device=dev) != 5
    assert p[0][5].isnan() and p[0][ok].isfinite().all()


def _codes(t, root):
    """float32 values as nearest codes and scales, on the CPU."""
    n = t.numel()
    b = torch.nn.functional.pad(t.reshape(-1).float(), (0, -n % 256)).view(-1, 256)
    s = b.abs().amax(1) / 448.0
    q = (b / torch.where(s > 0, s, 1.0)[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    return q.view(torch.uint8).view(-1)[:n].clone().view(torch.float8_e4m3fn), s


def _inputs8(dev, dtype, seed, shapes=SHAPES):
    p, g, m, v = _adamw_inputs(dev, dtype, seed, shapes)
    mq, ms = zip(*[_codes(t.cpu(), False) for t in m])
    rq, rs = zip(*[_codes(t.cpu().sqrt(), True) for t in v])
    return p, g, *[[t.to(dev) for t in l] for l in (mq, ms, rq, rs)]


@dtypes
@pytest.mark.parametrize("step", [1, 9])
def test_adamw_8(pkg, dev, dtype, step):
    """The parameters against the oracle from the decoded states; the scales; each code against
    the oracle's with the same numbers: equal but where the chance is within rounding of the
    number, and there one code off."""
    p, g, mq, ms, rq, rs = _inputs8(dev, dtype, step)
    old = [(tn.decode8(a.view(torch.uint8).cpu().numpy(), f64(b)), tn.decode8(c.view(torch.uint8).cpu().numpy(), f64(d)))
           for a, b, c, d in zip(mq, ms, rq, rs)]
    want = [_oracle(a, b, m.reshape(a.shape), (r * r).reshape(a.shape), step) for a, b, (m, r) in zip(p, g, old)]
    pkg.adamw_step_8bit(p, g, mq, ms, rq, rs, step=step, seed=77, **HYPER)
    differ = total = 0
    for i, o in enumerate(want):
        near(p[i], o["p"], o["p_mag"], 40, "p")
        n = p[i].numel()
        um, ur = tn.randoms(n, i, 77, step)
        for q, s, t, root, u in ((mq[i], ms[i], o["m"], False, um), (rq[i], rs[i], o["v"], True, ur)):
            c, sc = tn.encode8(t.reshape(-1), root, u)
            near(s, sc, sc, 12, "scale")
            got = q.view(torch.uint8).cpu().numpy().astype(int)
            off = np.abs((got & 127) - (c.astype(int) & 127))
            assert (off <= 1).all() and ((got & 128) == (c & 128))[off == 0].all()
            differ += int((off > 0).sum())
            total += n
    # a float32 chance is off by under 64 steps of its argument's 16 places: 2^-14 of the draws at most
    assert differ <= 2.0 ** -14 * total + 1, (differ, total)


def test_adamw_8_is_repeatable_and_seeded(pkg, dev):
    runs = []
    for seed in (5, 5, 6):
        p, g, mq, ms, rq, rs = _inputs8(dev, torch.float32, 3)
        for step in (1, 2, 3):
            pkg.adamw_step_8bit(p, g, mq, ms, rq, rs, step=step, seed=seed, **HYPER)
        runs.append([t.view(torch.uint8).clone() for t in mq + rq] + [t.clone() for t in p])
    assert all(torch.equal(a, b) for a, b in zip(runs[0], runs[1]))
    assert not all(torch.equal(a, b) for a, b in zip(runs[0], runs[2]))
    p, g, mq, ms, rq, rs = _inputs8(dev, torch.float32, 3)       # uint8 bits, the step on the device
    for step in (1, 2, 3):
        pkg.adamw_step_8bit(p, g, [t.view(torch.uint8) for t in mq], ms, [t.view(torch.uint8) for t in rq], rs,
                            step=torch.tensor(step, device=dev), seed=5, **HYPER)
    assert all(torch.equal(a, b.view(torch.uint8)) for a, b in zip(runs[0], mq + rq))


def test_adamw_8_slow_average_reaches_its_value(pkg, dev):
    """beta2 = 0.99 and one gradient for 400 steps: v must come to (1 - beta2^t) g^2 in the mean
    (rounded to nearest it stands still at a tenth of it). The relative deviation of one
    element's v is under the walk's, sqrt(sum of its steps' variances) < 0.5; of the mean of
    65536 of them six deviations are 1.2%."""
    n = 65536
    g = [torch.full((n,), 0.01, device=dev)]
    g[0][::256] = 0.02                                      # each block's scale is another element's
    p, codes = [torch.zeros(n, device=dev)], lambda: [torch.zeros(n, dtype=torch.uint8, device=dev)]
    scales = lambda: [torch.zeros(n // 256, device=dev)]
    mq, ms, rq, rs = codes(), scales(), codes(), scales()
    for step in range(1, 401):
        pkg.adamw_step_8bit(p, g, mq, ms, rq, rs, step=step, lr=1e-4, betas=(0.9, 0.99), weight_decay=0.0, seed=1)
    from mamba_tuckermoe_amd.adamw import dequantize_state
    v = dequantize_state(rq[0], rs[0]).double() ** 2
    m = dequantize_state(mq[0], ms[0]).double()
    want = 1 - 0.99 ** 400
    assert abs((v / g[0].double() ** 2).mean().item() / want - 1) < 0.012
    assert abs((m / g[0].double()).mean().item() - 1) < 0.012
    assert rq[0].min() > 0


def test_adamw_8_zero_and_nonfinite_blocks(pkg, dev):
    n = 1024
    p, g, mq, ms, rq, rs = _inputs8(dev, torch.float32, 2, [(n,)])
    g[0].zero_()
    for t in mq + rq:
        t.view(torch.uint8).zero_()
    q = p[0].clone()
    pkg.adamw_step_8bit(p, g, mq, ms, rq, rs, step=1, **HYPER)
    assert torch.allclose(p[0], q * (1 - 2e-4), rtol=1e-6, atol=0)
    assert not ms[0].any() and not rs[0].any() and not rq[0].view(torch.uint8).any()
    g[0].fill_(0.01)
    g[0][300] = float("inf")
    pkg.adamw_step_8bit(p, g, mq, ms, rq, rs, step=2, **HYPER)
    ok = torch.ones(n, dtype=torch.bool, device=dev)
    ok[256:512] = False
    pkg.adamw_step_8bit(p, g, mq, ms, rq, rs, step=3, **HYPER)
    assert p[0][ok].isfinite().all() and not p[0][300].isfinite()
    assert ms[0][[0, 2, 3]].isfinite().all() and not ms[0][1].isfinite()


@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_against_torch(pkg, dev, bits):
    """FusedAdamW over steps with a parameter that gets its gradients late; 32-bit states
    against torch's AdamW in float64, 8-bit ones against the functional call."""
    torch.manual_seed(0)
    ps = [torch.nn.Parameter(torch.randn(s, device=dev) * 0.05) for s in ((70, 40), (300,), (9,))]
    ref = [torch.nn.Parameter(p.detach().double()) for p in ps]
    opt = pkg.FusedAdamW(ps, state_bits=bits, seed=3, **HYPER)
    topt = torch.optim.AdamW(ref, **HYPER)
    for step in range(1, 6):
        for i, (p, r) in enumerate(zip(ps, ref)):
            if i == 2 and step < 3:
                continue
            p.grad = torch.randn(p.shape, device=dev) * 0.01
            r.grad = p.grad.double()
        opt.step()
        topt.step()
    assert opt.state[ps[0]]["step"] == 5 and opt.state[ps[2]]["step"] == 3
    for p, r in zip(ps, ref):
        if bits == 32:
            # five steps of 32 roundings of p and of updates of lr
            assert (p.double() - r).abs().max() <= 5 * 32 * U * (r.abs().max() + 10 * HYPER["lr"])
        else:
            # an update is at most lr |m| / sqrt(v); states off by a code, 1/8, in each
            assert (p.double() - r).abs().max() <= 5 * HYPER["lr"] * 4


# ---- streams, graphs, autograd ---------------------------------------------------

def test_side_stream(pkg, dev):
    raw = _logits(5000, 16, torch.float32, 1).to(dev)
    n, dr, dh = norm_inputs(NORM_FORMS[-1], 500, 256, 1)
    n = {k: v.to(dev) for k, v in n.items()}
    dr, dh = dr.to(dev), dh.to(dev)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        _check_router(pkg, raw, 2, 0.5, 10.0, None, 1)
        _check_norm(pkg, n, dr, dh)
        p, g, m, v = _adamw_inputs(dev, torch.float32, 1)
        want = [_oracle(*t, 3) for t in zip(p, g, m, v)]
        pkg.adamw_step(p, g, m, v, step=3, **HYPER)
        for i, o in enumerate(want):
            near(p[i], o["p"], o["p_mag"], 32)
    torch.cuda.synchronize()


def test_graph_capture(pkg, dev):
    """Router, norm and optimizer step captured with their backward: each replay on new inputs
    gives what the eager calls give, the step counting on; eager work between the replays."""
    torch.manual_seed(0)
    T, d, E, k = 600, 192, 8, 2
    x, y = torch.randn(T, d, device=dev), torch.randn(T, d, device=dev)
    tau = torch.tensor(0.5, device=dev)

    def params():
        g = torch.Generator().manual_seed(4)
        return [torch.nn.Parameter((torch.randn(s, generator=g) * 0.1 + 1).to(dev)) for s in ((d,), (d,), (d, E))]

    def body(ps, opt):
        gamma, w, router = ps
        r, h = pkg.fused_block_norm(x, y, gamma=gamma, next_weight=w)
        q = pkg.fused_router(h @ router, k, tau)
        loss = (q.weights * q.weights).sum() / T + q.lb_loss + q.z_loss + (r * r).mean()
        grads = torch.autograd.grad(loss, ps)
        for p, g in zip(ps, grads):
            p.grad = g
        opt.step()
        return q.idx, q.counts, loss.detach()
    ps, ref = params(), params()
    opt = pkg.FusedAdamW(ps, state_bits=8, capturable=True, lr=1e-2)
    ropt = pkg.FusedAdamW(ref, state_bits=8, lr=1e-2)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        body(ps, opt)
    torch.cuda.synchronize()
    body(ref, ropt)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out = body(ps, opt)
    for i in range(4):
        x.copy_(torch.randn(T, d, device=dev))
        tau.fill_(0.5 + 0.3 * i)
        graph.replay()
        want = body(ref, ropt)
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b), i
        for a, b in zip(ps, ref):
            # lr / (1 - beta^t): the device's pow and the host's may differ in the last place
            assert (a - b).abs().max() <= 1e-2 * 16 * U + 8 * U * b.abs().max(), i
        with torch.no_grad():
            for a, b in zip(ref, ps):
                a.copy_(b)
    assert opt.state[ps[0]]["step"].item() == 5 == ropt.state[ref[0]]["step"]


def test_capture_refuses_leaves_of_a_living_eager_graph(pkg, dev):
    """A capture whose leaves an eager graph of another stream still holds is refused when the
    operator is called; once that graph is gone it is captured and replayed."""
    x = torch.randn(64, 32, device=dev)
    w = torch.ones(32, device=dev, requires_grad=True)
    raw = torch.randn(64, 8, device=dev, requires_grad=True)
    for leaf, call in ((w, lambda: pkg.fused_block_norm(y=x, post_weight=w)[0]),
                       (raw, lambda: pkg.fused_router(raw, 2, 0.5).z_loss)):
        living = call()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="outside this capture"):
            with torch.cuda.graph(g, stream=s):
                call()
        del living
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out = call()
            grad, = torch.autograd.grad(out, leaf, torch.ones_like(out))
        want, = torch.autograd.grad(call().sum(), leaf)
        for _ in range(3):
            grad.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(grad, want)


def test_step_in_capture_needs_capturable(pkg, dev):
    p = torch.nn.Parameter(torch.ones(8, device=dev))
    p.grad = torch.ones_like(p)
    opt = pkg.FusedAdamW([p])
    opt.step()
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="capturable"):
        with torch.cuda.graph(g):
            opt.step()
    torch.cuda.synchronize()
    assert opt.state[p]["step"] == 1


def test_capturable_state_is_loaded_shared(pkg, dev):
    ps = [torch.nn.Parameter(torch.ones(8, device=dev)) for _ in range(3)]
    for p in ps:
        p.grad = torch.ones_like(p)
    opt = pkg.FusedAdamW(ps, capturable=True)
    opt.step()
    opt.step()
    opt2 = pkg.FusedAdamW(ps, capturable=True)
    opt2.load_state_dict(opt.state_dict())
    steps = [opt2.state[p]["step"] for p in ps]
    assert all(s is steps[0] for s in steps) and steps[0].dtype == torch.int64
    opt2.step()
    assert steps[0].item() == 3 and opt.state[ps[0]]["step"].item() == 2


def test_second_derivatives_are_refused(pkg, dev):
    raw = _logits(4, 8, torch.float32, 0).to(dev).requires_grad_()
    g, = torch.autograd.grad(pkg.fused_router(raw, 2, 0.5).z_loss, raw, create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        g.sum().backward()
    x = torch.randn(4, 8, device=dev, requires_grad=True)
    g, = torch.autograd.grad(pkg.fused_block_norm(y=x, post_weight=torch.ones(8, device=dev))[0].sum(), x,
                             create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        g.sum().backward()


def test_saved_inputs_are_guarded(pkg, dev):
    """A tensor that the backward needs and that was written to in between is an error."""
    raw = _logits(40, 8, torch.float32, 0).to(dev).requires_grad_()
    r = pkg.fused_router(raw, 2, 0.5)
    r.counts.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        r.lb_loss.backward()
    w = torch.ones(8, device=dev, requires_grad=True)
    x = torch.randn(4, 8, device=dev)
    out, _ = pkg.fused_block_norm(y=x, post_weight=w)
    p = [w]
    pkg.adamw_step(p, [torch.ones_like(w)], [torch.zeros(8, device=dev)], [torch.zeros(8, device=dev)], step=1, lr=1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        out.sum().backward()


# ---- the layers that call them ----------------------------------------------------

def _latent_torch(xs, G, idx, p):
    out = 0
    for j in range(idx.shape[1]):
        on = (idx[:, j:j + 1] >= 0).to(p.dtype)
        out = out + on * p[:, j:j + 1] * torch.einsum("bs,bsq->bq", xs, G[idx[:, j].clamp(min=0)])
    return out


def _router64(raw, k, tau, scale, mask):
    """train_ops.fused_router as float64 torch expressions."""
    from test_train_ops import _router_torch
    w, lb, z = _router_torch(raw, k, float(tau), scale, mask)
    idx = torch.sort(raw.detach(), dim=-1, descending=True, stable=True).indices[:, :k]
    if mask is not None:
        idx = torch.where(mask[:, None], idx, -1)
    return idx, w, lb, z, None


def _norm64(x=None, y=None, gate=None, post_weight=None, gamma=None, next_weight=None, eps=1e-5):
    from test_train_ops import _norm_torch
    if y is None:
        return x, _norm_torch(y=x, next_weight=next_weight, eps=eps)[1]
    return _norm_torch(x, y, gate, post_weight, gamma, next_weight, eps)


@pytest.mark.parametrize("padded", [False, True])
def test_block_train_gradients(pkg, dev, monkeypatch, padded):
    """TuckerFFNTrain: output, losses and every parameter's gradient against the same module in
    float64 on the CPU with plain expressions in the operators' places."""
    import mamba_tuckermoe_amd.block_train as bt
    import mamba_tuckermoe_amd.latent as lat
    cfg = pkg.TuckerMoEConfig(kmoe_num_experts=8, kmoe_r1=4, kmoe_r2=64, kmoe_r3=64, ffn_expand=2)
    torch.manual_seed(0)
    m = pkg.TuckerFFNTrain(64, cfg).train()
    ref = pkg.TuckerFFNTrain(64, cfg).double().train()
    with torch.no_grad():
        for l in (m.ffn_gate, m.ffn_up, m.ffn_down):
            l.router.weight.mul_(30)
            l.core.mul_(6)
    ref.load_state_dict({k: v.double() for k, v in m.state_dict().items()})
    x = torch.randn(3, 50, 64)
    mask = torch.rand(3, 50) > 0.3 if padded else None
    with monkeypatch.context() as mp:
        mp.setattr(lat.FusedLatentMoE, "apply", staticmethod(_latent_torch))
        mp.setattr(lat, "fused_router", _router64)
        mp.setattr(bt, "fused_block_norm", _norm64)
        xr = x.double().requires_grad_()
        o_ref, lb_ref, z_ref = ref(xr, step=700, mask=mask)
        (o_ref.square().mean() + 0.1 * lb_ref + 0.01 * z_ref).backward()
    m = m.to(dev)
    xg = x.to(dev).requires_grad_()
    o, lb, z = m(xg, step=700, mask=None if mask is None else mask.to(dev))
    (o.square().mean() + 0.1 * lb + 0.01 * z).backward()
    assert onp.rel_l2(f64(o), f64(o_ref)) <= 1e-5
    assert abs(lb.item() - lb_ref.item()) <= 1e-4 and abs(z.item() - z_ref.item()) <= 1e-4 * z_ref.item()
    n = 150 if mask is None else int(mask.sum())
    assert m.ffn_gate.expert_counts.sum().item() == 2 * n
    assert onp.rel_l2(f64(xg.grad), f64(xr.grad)) <= 1e-4
    for (name, p), (_, q) in zip(m.named_parameters(), ref.named_parameters()):
        assert onp.rel_l2(f64(p.grad), f64(q.grad)) <= 1e-4, name


def test_training_layer_fused_router_is_the_plain_one(pkg, dev):
    """fused_router=True against the torch expressions in float32: the same routing, outputs
    and gradients to float32 rounding."""
    torch.manual_seed(1)
    a = pkg.TuckerMoETrain(128, 96, num_experts=8, r2=128, r3=64).to(dev).train()
    b = pkg.TuckerMoETrain(128, 96, num_experts=8, r2=128, r3=64, fused_router=True).to(dev).train()
    b.load_state_dict(a.state_dict())
    x = torch.randn(300, 128, device=dev)
    for step in (None, 700, torch.tensor(700.0, device=dev)):
        outs = []
        for m in (a, b):
            m.zero_grad()
            o, lb, z = m(x, step=step)
            (o.square().mean() + lb + z).backward()
            outs.append((o, lb, z))
        for u, v in zip(*outs):
            assert onp.rel_l2(f64(v), f64(u)) <= 1e-5
        for (n, p), (_, q) in zip(a.named_parameters(), b.named_parameters()):
            assert onp.rel_l2(f64(q.grad), f64(p.grad)) <= 1e-4, n
    b.eval()
    assert b(x)[1:] == (0.0, 0.0)


@pytest.mark.parametrize("bits,dtype", [(32, torch.float32), (8, torch.float32), (8, torch.bfloat16)])
def test_training_steps_run_together(pkg, dev, bits, dtype):
    """Norms, routers, contraction and optimizer over a few steps: all finite, every parameter
    moved, and by no more than AdamW's bound of its steps."""
    cfg = pkg.TuckerMoEConfig(kmoe_num_experts=8, kmoe_r1=4, kmoe_r2=128, kmoe_r3=128, ffn_expand=2)
    torch.manual_seed(0)
    m = pkg.TuckerFFNTrain(128, cfg).to(dev, dtype).train()
    opt = pkg.FusedAdamW(m.parameters(), lr=1e-2, betas=(0.9, 0.95), weight_decay=0.0, state_bits=bits)
    start = [p.detach().clone() for p in m.parameters()]
    x = torch.randn(400, 128, device=dev).to(dtype)
    mask = torch.arange(400, device=dev) < 350
    for step in range(3):
        opt.zero_grad()
        out, lb, z = m(x, step=step, mask=mask)
        (out.float().square().mean() + 0.01 * lb + 0.001 * z).backward()
        opt.step()
        assert out.isfinite().all() and lb.isfinite() and z.isfinite()
    for (n, p), q in zip(m.named_parameters(), start):
        moved = (p.detach().float() - q.float()).abs()
        # |m / sqrt(v)| after bias correction is at most sqrt(3 steps); a code is off by 1/8
        assert p.isfinite().all() and moved.max() > 0, n
        assert moved.max() <= 3 * 1e-2 * 2.5 + 2.0 ** -7 * q.float().abs().max(), n


def test_adamw_8_decays_to_zero(pkg, dev):
    """A first moment whose scale's reciprocal fp32 does not hold (decayed over hundreds of steps
    without a gradient) becomes zero, not something else; v far below 1 keeps its codes."""
    p, g, mq, ms, rq, rs = _inputs8(dev, torch.float32, 2, [(512,)])
    g[0].zero_()
    ms[0].fill_(1e-39)
    rs[0].fill_(1e-15)
    old = tn.decode8(rq[0].view(torch.uint8).cpu().numpy(), f64(rs[0]))
    q = p[0].clone()
    pkg.adamw_step_8bit(p, g, mq, ms, rq, rs, step=5, seed=1, **HYPER)
    assert not ms[0].any() and (mq[0].view(torch.uint8) & 127 == 0).all()
    assert torch.allclose(p[0], q * (1 - 2e-4), rtol=1e-6, atol=0)
    new = tn.decode8(rq[0].view(torch.uint8).cpu().numpy(), f64(rs[0]))
    # one code up or down, and sqrt(0.97) of it
    assert np.all(np.abs(new - old * np.sqrt(0.97)) <= old / 7.9)


def test_adamw_8_odd_views(pkg, dev):
    """Views that begin anywhere, of parameters and of codes: as aligned copies; what lies beside
    them stays."""
    for dtype in DTYPES.values():
        n = 1031
        p, g, mq, ms, rq, rs = _inputs8(dev, dtype, 6, [(n,)])
        wide = {k: torch.zeros(n + 8, dtype=t.dtype, device=dev) for k, t in (("p", p[0]), ("g", g[0]))}
        wide.update({k: torch.zeros(n + 8, dtype=torch.uint8, device=dev) for k in ("m", "r")})
        v = {"p": wide["p"][3:n + 3], "g": wide["g"][1:n + 1], "m": wide["m"][1:n + 1], "r": wide["r"][3:n + 3]}
        for k, t in (("p", p[0]), ("g", g[0]), ("m", mq[0].view(torch.uint8)), ("r", rq[0].view(torch.uint8))):
            v[k].copy_(t)
        ms2, rs2 = ms[0].clone(), rs[0].clone()
        pkg.adamw_step_8bit(p, g, mq, ms, rq, rs, step=4, seed=9, **HYPER)
        pkg.adamw_step_8bit([v["p"]], [v["g"]], [v["m"]], [ms2], [v["r"]], [rs2], step=4, seed=9, **HYPER)
        assert torch.equal(v["p"], p[0]) and torch.equal(v["m"], mq[0].view(torch.uint8))
        assert torch.equal(v["r"], rq[0].view(torch.uint8)) and torch.equal(ms2, ms[0]) and torch.equal(rs2, rs[0])
        for k, a in (("p", 3), ("m", 1), ("r", 3)):
            assert not wide[k][:a].any() and not wide[k][n + a:].any()


@pytest.mark.parametrize("T,d", [(5, 2), (9, 3), (6, 4), (6, 5), (40, 129), (7, 513), (3, 1025), (3, 4097), (3, 8193)])
def test_norm_odd_widths_leave_the_rest(pkg, dev, T, d):
    """Rows whose width is no multiple of a load, their outputs in the middle of larger buffers
    (through the C ABI): the elements beside them stay as they were."""
    lib = pkg._lib
    L = lib.lib()
    for dtype in DTYPES.values():
        n, dr, dh = norm_inputs(NORM_FORMS[-1], T, d, T + d, dtype)
        n = {k: v.to(dev) for k, v in n.items()}
        dr, dh = dr.to(dev), dh.to(dev)
        names = ("x", "y", "gate", "post_weight", "gamma", "next_weight")
        a = lib.TmoeBlockNorm(*[n[k].data_ptr() for k in names[:3]], d, d, d, *[n[k].data_ptr() for k in names[3:]],
                              T, d, lib.dtype_code(dtype), 1e-5)
        es = dr.element_size()

        def out(rows):
            return torch.full((rows * d + 16,), 7.0, dtype=dtype, device=dev)
        r, h, dx, dy, dg = (out(T) for _ in range(5))
        dp, dga, dn = (out(1) for _ in range(3))
        inv = torch.zeros(2, T, device=dev)
        nws = L.tmoe_block_norm_workspace_bytes(T, d, lib.dtype_code(dtype))
        ws = torch.empty(max(nws, 1), dtype=torch.uint8, device=dev)
        st = torch.cuda.current_stream().cuda_stream
        at = lambda t: t.data_ptr() + 5 * es
        lib.check(L.tmoe_block_norm_forward(a, at(r), at(h), inv.data_ptr(), st))
        lib.check(L.tmoe_block_norm_backward(a, inv.data_ptr(), dr.data_ptr(), d, dh.data_ptr(), d, at(dx), at(dy),
                                             at(dg), at(dp), at(dga), at(dn), ws.data_ptr(), nws, st))
        o = tn.block_norm(**{k: f64(v) for k, v in n.items()}, dr=f64(dr), dh=f64(dh))
        for k, t, rows in (("r", r, T), ("h", h, T), ("dx", dx, T), ("dy", dy, T), ("dgate", dg, T),
                           ("dpost_weight", dp, 1), ("dgamma", dga, 1), ("dnext_weight", dn, 1)):
            assert (t[:5] == 7).all() and (t[5 + rows * d:] == 7).all(), k
            got = t[5:5 + rows * d]
            near(got, o[k].reshape(-1), o[k + "_mag"].reshape(-1), 400, k)


@pytest.mark.parametrize("shape", [(2048, 8, 2, 256, 256), (300, 8, 2, 64, 128)])
def test_masked_tokens_select_nothing_in_the_contraction(pkg, dev, shape):
    """The contraction of a masked routing (idx -1, weights 0) is that of the tokens that are left,
    in both of its forms: zero rows, and the same dG to the rounding of sums in another order."""
    B, E, k, r3, r2 = shape
    g = torch.Generator().manual_seed(B)
    raw = _logits(B, E, torch.float32, 1).to(dev)
    mask = (torch.rand(B, generator=g) > 0.4).to(dev)
    x = torch.randn(B, r3, generator=g).bfloat16().to(dev)
    G = (torch.randn(E, r3, r2, generator=g) * r3 ** -0.5).bfloat16().to(dev)
    dout = torch.randn(B, r2, generator=g).bfloat16().to(dev)

    def run(raw, x, dout, mask):
        leaves = [t.detach().requires_grad_() for t in (raw, x, G)]
        q = pkg.fused_router(leaves[0], k, 0.5, mask=mask)
        out = pkg.FusedLatentMoE.apply(leaves[1], leaves[2], q.idx, q.weights)
        return [out.detach()] + list(torch.autograd.grad(out, leaves, dout))
    a = run(raw, x, dout, mask)
    b = run(raw[mask], x[mask], dout[mask], None)
    for i in range(3):
        assert not a[i][~mask].any()
        assert onp.rel_l2(f64(a[i][mask]), f64(b[i])) <= 1e-2
    assert onp.rel_l2(f64(a[3]), f64(b[3])) <= 1e-2


def test_router_top1_weights_gradient(pkg, dev):
    """k = 1: the weight is P / (P + 1e-6), its gradient the 1e-6 that it lacks to one. Taken as
    the difference of two sums next to each other it would be 1e-2 off in float32; here within
    the rounding of its own terms, as every other k's."""
    raw = _logits(5000, 16, torch.float32, 8).to(dev).requires_grad_()
    dw = torch.randn(5000, 1, device=dev)
    r = pkg.fused_router(raw, 1, 0.5)
    draw, = torch.autograd.grad(r.weights, raw, dw)
    o = tn.router(f64(raw), 1, 0.5, 10.0, None, f64(dw))
    # 16 cap / tau + 128 roundings of each factor, in the 2-norm
    assert onp.rel_l2(f64(draw), o["draw"]) <= 4 * (16 * 10 / 0.5 + 128) * U


def test_router_nan_row_gradient_is_its_own(pkg, dev):
    """One NaN logit: that token's gradients are NaN, the others' what they are without it."""
    for E in (8, 64):
        raw = _logits(40, E, torch.float32, E).to(dev)
        dw = torch.randn(40, 3, device=dev)
        bad = raw.clone()
        bad[11, E - 3] = float("nan")
        d = [torch.autograd.grad(pkg.fused_router(t, 3, 0.5).weights, t, dw)[0]
             for t in (raw.requires_grad_(), bad.requires_grad_())]
        assert d[1][11].isnan().all()
        d[1][11] = d[0][11]
        assert torch.equal(d[0], d[1])


def _free_gib():
    return torch.cuda.mem_get_info()[0] / 2 ** 30


def test_offsets_past_32_bits(pkg, dev):
    """The last rows and elements of tensors of more than 2^31 elements, as by themselves."""
    if _free_gib() < 80:
        pytest.skip("needs 80 GiB of free memory")
    T, d, last = 2 ** 17 + 3, 16384, 5
    n, dr, dh = norm_inputs(("x", "y", "gamma", "next"), last, d, 1, torch.bfloat16)
    n = {k: v.to(dev) for k, v in n.items()}
    dr, dh = dr.to(dev), dh.to(dev)

    def long(t):
        z = torch.zeros(T, d, dtype=t.dtype, device=dev)
        z[-last:] = t
        return z
    big = {k: (long(v) if v.dim() == 2 else v).requires_grad_() for k, v in n.items()}
    r, h = pkg.fused_block_norm(**big)
    gx, gy = torch.autograd.grad((r, h), (big["x"], big["y"]), (long(dr), long(dh)))
    small = {k: v.requires_grad_() for k, v in n.items()}
    rs, hs = pkg.fused_block_norm(**small)
    sx, sy = torch.autograd.grad((rs, hs), (small["x"], small["y"]), (dr, dh))
    for a, b in ((r, rs), (h, hs), (gx, sx), (gy, sy)):
        assert torch.equal(a[-last:], b) and not a[:-last].any()
    del r, h, gx, gy, big
    B, E = 2 ** 23 + 3, 256
    raw = torch.zeros(B, E, device=dev)
    tail = _logits(last, E, torch.float32, 4).to(dev).requires_grad_()
    raw[-last:] = tail.detach()
    raw.requires_grad_()
    dw = torch.randn(last, 8, device=dev)
    a, b = pkg.fused_router(raw, 8, 0.5), pkg.fused_router(tail, 8, 0.5)
    assert torch.equal(a.idx[-last:], b.idx) and torch.equal(a.weights[-last:], b.weights)
    assert a.counts.sum().item() == 8 * B
    dwl = torch.zeros(B, 8, device=dev)
    dwl[-last:] = dw
    assert torch.equal(torch.autograd.grad(a.weights, raw, dwl)[0][-last:], torch.autograd.grad(b.weights, tail, dw)[0])
    del raw, a, dwl
    N, keep = 2 ** 31 + 517, 773        # keep: from a block's begin on
    pl, gl = (torch.zeros(N, dtype=torch.bfloat16, device=dev) for _ in range(2))
    p, g = ((torch.randn(keep, device=dev) * s).bfloat16() for s in (0.05, 0.01))
    N0 = N - keep
    assert N0 % 256 == 0
    pl[N0:], gl[N0:] = p, g
    for bits in (32, 8):
        st, sl = [], []
        for size, out in ((keep, st), (N, sl)):
            if bits == 32:
                out += [[torch.zeros(size, device=dev)] for _ in range(2)]
            else:
                for _ in range(2):
                    out += [[torch.zeros(size, dtype=torch.uint8, device=dev)],
                            [torch.zeros(-(-size // 256), device=dev)]]
        step = pkg.adamw_step if bits == 32 else pkg.adamw_step_8bit
        step([p], [g], *st, step=3, **HYPER)
        step([pl], [gl], *sl, step=3, **HYPER)
        assert torch.equal(pl[N0:], p) and not pl[:N0].any()
        for a, b in zip(sl, st):
            if a[0].dtype == torch.float32:        # (codes are rounded by the element's place)
                assert torch.equal(a[0][-b[0].numel():], b[0])
    del pl, gl, sl, a, b
    torch.cuda.empty_cache()


def test_capturable_counts_of_resting_parameters(pkg, dev):
    """Parameters that rest for some steps: the updates of the count on the device are those of
    the count on the host, eager and replayed."""
    def params():
        g = torch.Generator().manual_seed(7)
        return [torch.nn.Parameter((torch.randn(300, generator=g) * 0.1).to(dev)) for _ in range(3)]
    ps, ref = params(), params()
    opt = pkg.FusedAdamW(ps, capturable=True, lr=1e-2)
    ropt = pkg.FusedAdamW(ref, lr=1e-2)
    grads = torch.randn(3, 300, device=dev) * 0.01

    def step(o, qs, on):
        for q, g, use in zip(qs, grads, on):
            q.grad = g.clone() if use else None
        o.step()

    def same():
        for a, b in zip(ps, ref):
            # as in test_graph_capture: the device's pow against the host's, per step
            assert (a - b).abs().max() <= 10 * (1e-2 * 16 * U + 8 * U * b.abs().max())
        assert [opt.state[p]["step"].item() for p in ps] == [ropt.state[p]["step"] for p in ref]
    for on in ((1, 1, 1), (0, 1, 1), (0, 1, 1), (1, 1, 1), (1, 0, 1)):
        step(opt, ps, on)
        step(ropt, ref, on)
        same()
    for q, g in zip(ps, grads):
        q.grad = g.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for _ in range(3):
        graph.replay()
        step(ropt, ref, (1, 1, 1))
        torch.cuda.synchronize()
        same()


@pytest.mark.parametrize("capturable,bits", [(True, 32), (True, 8), (False, 8)])
def test_first_step_in_a_capture_is_refused(pkg, dev, capturable, bits):
    """... and leaves no state; the eager steps after it are those of an optimizer that never
    saw the capture."""
    def make():
        p = torch.nn.Parameter(torch.linspace(-1, 1, 700).to(dev))
        p.grad = torch.linspace(-0.01, 0.02, 700).to(dev)
        return p, pkg.FusedAdamW([p], state_bits=bits, capturable=capturable, lr=1e-2)
    (p, opt), (q, ropt) = make(), make()
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="first step" if capturable else "capturable"):
        with torch.cuda.graph(g):
            opt.step()
    torch.cuda.synchronize()
    assert not opt.state
    for _ in range(3):
        opt.step()
        ropt.step()
    assert torch.equal(p, q)


def test_forward_mode_is_refused_on_the_device(pkg, dev):
    """With and without reverse gradients wanted; in the layer too."""
    import torch.autograd.forward_ad as fw
    x = torch.randn(40, 64, device=dev)
    w = torch.ones(64, device=dev)
    layer = pkg.TuckerMoETrain(64, 48, num_experts=8, r2=64, r3=64, fused_router=True).to(dev)
    for grad in (False, True):
        w.requires_grad_(grad)
        layer.requires_grad_(grad)
        with fw.dual_level():
            t = fw.make_dual(x, torch.ones_like(x))
            for call in (lambda: pkg.fused_router(t[:, :8], 2, 0.5), lambda: pkg.fused_block_norm(y=t, post_weight=w),
                         lambda: pkg.fused_block_norm(x, t, gamma=w), lambda: layer(t)):
                with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                    call()
        assert pkg.fused_block_norm(y=x, post_weight=w)[0].isfinite().all()


@pytest.mark.parametrize("capturable", [False, True])
def test_optimizer_goes_on_from_torchs(pkg, dev, capturable):
    """torch's AdamW for three steps, FusedAdamW from its state for three more: as torch's for
    six, in float64."""
    torch.manual_seed(5)
    ps = [torch.nn.Parameter(torch.randn(s, device=dev) * 0.05) for s in ((70, 40), (300,))]
    ref = [torch.nn.Parameter(p.detach().double()) for p in ps]
    topt, ropt = torch.optim.AdamW(ps, **HYPER), torch.optim.AdamW(ref, **HYPER)
    opt = pkg.FusedAdamW(ps, capturable=capturable)
    for step in range(6):
        for p, r in zip(ps, ref):
            p.grad = torch.randn(p.shape, device=dev) * 0.01
            r.grad = p.grad.double()
        if step == 3:
            sd = topt.state_dict()
            sd["param_groups"][0]["capturable"] = capturable
            opt.load_state_dict(sd)
        (topt if step < 3 else opt).step()
        ropt.step()
    for p, r in zip(ps, ref):      # six steps of 32 roundings of p and of updates of lr
        assert (p.double() - r).abs().max() <= 6 * 32 * U * (r.abs().max() + 10 * HYPER["lr"])


@dtypes
def test_adamw_8_roots_of_subnormals(pkg, dev, dtype):
    """Gradients whose second moment is under 2^-126, with eps = 0: the step is lr in the first
    step and the formula's in the next, and the scales are the roots'. v, in steps of 2^-149, is
    off by half a one of each of r r (by 0.97), its product with 0.97, g g (by 0.03) and its
    product: 1.5 (the sum is exact), and its root r by that over 2 r^2 of itself."""
    g = torch.Generator().manual_seed(3)
    n, hyper = 1500, dict(lr=2e-3, betas=(0.9, 0.97), eps=0.0, weight_decay=0.0)
    mag = torch.exp(torch.empty(n).uniform_(np.log(2e-20), np.log(4e-18), generator=g))
    mag[256:512] *= 1e3                                       # a block of ordinary ones
    mag[700] = 1.0                                            # a block with one large element
    grad = (mag * torch.where(torch.rand(n, generator=g) < 0.5, -1.0, 1.0)).to(dtype)
    p = [(torch.randn(n, generator=g) * 0.05).to(dtype).to(dev)]
    q8 = lambda: [torch.zeros(n, dtype=torch.uint8, device=dev)]
    sc = lambda: [torch.zeros(-(-n // 256), device=dev)]
    mq, ms, rq, rs = q8(), sc(), q8(), sc()
    for step in (1, 2):
        old = [tn.decode8(c[0].cpu().numpy(), f64(s[0])) for c, s in ((mq, ms), (rq, rs))]
        o = tn.adamw(f64(p[0]), f64(grad), old[0], old[1] ** 2, step, 2e-3, 0.9, 0.97, 0.0, 0.0)
        pkg.adamw_step_8bit(p, [grad.to(dev)], mq, ms, rq, rs, step=step, seed=4, **hyper)
        v = o["v"]
        off = 1.5 * 2.0 ** -149 / (2 * v)                         # of the root, relative
        upd = np.abs(o["p_mag"]) * 40 * U + 2e-3 / (1 - 0.9 ** step) * np.abs(o["m"]) / np.sqrt(v) * off * 1.1
        tol = upd + (2.0 ** -8 * (np.abs(o["p"]) + upd) if dtype == torch.bfloat16 else 0)
        assert (np.abs(f64(p[0]) - o["p"]) <= tol).all(), step
        root = np.pad(np.sqrt(v), (0, -n % 256)).reshape(-1, 256)
        at = np.pad(off, (0, -n % 256)).reshape(-1, 256)[np.arange(root.shape[0]), root.argmax(1)]
        want = root.max(1) / 448
        assert (np.abs(f64(rs[0]) - want) <= want * (12 * U + 1.1 * at)).all(), step


def test_adamw_8_square_that_overflows(pkg, dev):
    """A finite gradient whose square is not: v is infinite and the element's step zero, as with
    32-bit states; its block's second scale is not finite from then on."""
    out = []
    for bits in (32, 8):
        p, g, mq, ms, rq, rs = _inputs8(dev, torch.float32, 2, [(700,)])
        m, v = ([torch.zeros(700, device=dev)] for _ in range(2))
        for t in mq + rq:
            t.view(torch.uint8).zero_()
        g[0][300] = 3e25
        g[0][:256] *= 1e15
        if bits == 32:
            pkg.adamw_step(p, g, m, v, step=1, **HYPER)
        else:
            pkg.adamw_step_8bit(p, g, mq, ms, rq, rs, step=1, **HYPER)
        out.append(p[0])
    assert out[1].isfinite().all() and not rs[0][1].isfinite() and rs[0][[0, 2]].isfinite().all()
    assert (out[0] - out[1]).abs().max() <= 40 * U * (out[0].abs().max() + 10 * HYPER["lr"])


@pytest.mark.parametrize("E,k", [(64, 1), (200, 2), (256, 1), (256, 2), (256, 16)])
def test_router_gradient_of_nearly_flat_logits(pkg, dev, E, k):
    """Many experts with hardly any difference, few of them selected: the weights' gradient has
    the selected probabilities' sum twice in its denominator, which is a hundredth of all.

    Steps of 2^-24, of a term, at most: an exponential 5 (its argument 2: a difference of two
    exponentials near 1, 3 each, times cap / (2 tau) = 1/4; itself 3). A sum of them 13 more
    (8 in a lane, 5 exchanges); 1 / sum over all 5 + 13 + 1 + 2 = 21; 1 / s 18 + 21 + 1 + 2 = 42.
    sum_i w_i (dw_i - dw_0): 18 + 2, the two and 2 products, 85; the term that has it times
    1 / s 128; with its exponential 5, 1 / (sum tau) 24, Q R^2 9 and 4 more roundings 170."""
    g = torch.Generator().manual_seed(E + k)
    B = 400
    raw = (torch.randn(B, E, generator=g) * 0.03).to(dev).requires_grad_()
    dw = torch.randn(B, k, generator=g).to(dev)
    r = pkg.fused_router(raw, k, 2.0, 1.0)
    draw, = torch.autograd.grad(r.weights, raw, dw)
    o = tn.router(f64(raw), k, 2.0, 1.0, None, f64(dw))
    near(draw, o["draw"], o["draw_mag"], 170, "draw")


def _router_large_cap(raw, k, tau, cap, dw, dlb, dz):
    """tn.router where exp(a - cap) is 0: the same by a's own maximum."""
    B, E = raw.shape
    th = np.tanh(raw / cap)
    a = cap * th
    top = a.max(-1, keepdims=True)
    soft = np.exp(a - top)
    lse = (top + np.log(soft.sum(-1, keepdims=True)))[:, 0]
    soft /= soft.sum(-1, keepdims=True)
    P = np.exp((a - top) / tau)
    P /= P.sum(-1, keepdims=True)
    idx = np.argsort(-raw, axis=-1, kind="stable")[:, :k]
    sel = np.zeros((B, E))
    np.put_along_axis(sel, idx, 1.0, -1)
    pk = np.take_along_axis(P, idx, -1)
    s = pk.sum(-1, keepdims=True) + 1e-6
    w = pk / s
    n = sel.sum(0)
    G, gs, gm = dlb * E * n / B ** 2, np.zeros((B, E)), np.zeros((B, E))
    np.put_along_axis(gs, idx, (dw - (dw * w).sum(-1, keepdims=True)) / s, -1)
    np.put_along_axis(gm, idx, (np.abs(dw) + (np.abs(dw) * w).sum(-1, keepdims=True)) / s, -1)
    g, gm = G + gs, np.abs(G) + gm
    z = dz * 2 * lse[:, None] * soft / B
    return {"idx": idx, "w": w, "lb": E * (n / B * P.mean(0)).sum(), "z": (lse ** 2).mean(),
            "draw": (P * (g - (P * g).sum(-1, keepdims=True)) / tau + z) * (1 - th * th),
            "draw_mag": P * (gm + (P * gm).sum(-1, keepdims=True)) / tau + np.abs(z)}


@dtypes
@pytest.mark.parametrize("cap,spread", [(15.9, 1.0), (16.1, 1.0), (100.0, 1.0), (100.0, 20.0), (1e3, 1.0),
                                        (1e6, 0.01), (1e8, 1.0), (3e38, 1.0)])
@pytest.mark.parametrize("E,k", [(4, 2), (33, 5)])
def test_router_large_caps(pkg, dev, E, k, cap, spread, dtype):
    """A cap that caps little or nothing, to that of a plain softmax. The bounds are those of
    _check_router with what its capped logits reach in the cap's place: cap tanh(raw / cap) is off
    by 8 steps of itself."""
    g = torch.Generator().manual_seed(E)
    raw = (_logits(500, E, torch.float32, E) * spread).to(dtype).to(dev).requires_grad_()
    dw, dlb, dz, tau = torch.randn(500, k, generator=g), 0.7, 0.05, 1.25
    cap = float(np.float32(cap))
    r = pkg.fused_router(raw, k, tau, cap)
    draw, = torch.autograd.grad((r.weights, r.lb_loss, r.z_loss), raw,
                                (dw.to(dev), torch.tensor(dlb, device=dev), torch.tensor(dz, device=dev)))
    o = _router_large_cap(f64(raw), k, tau, cap, f64(dw), dlb, dz)
    if cap < 300:
        for key, v in tn.router(f64(raw), k, tau, cap, None, f64(dw), dlb, dz).items():
            assert key == "counts" or np.allclose(o[key], v, rtol=1e-9, atol=1e-13), key
    most = cap * np.tanh(np.abs(f64(raw)).max() / cap)
    n = 16 * most / tau + 128
    assert np.array_equal(r.idx.cpu().numpy(), o["idx"])
    near(r.weights, o["w"], o["w"], n, "w")
    near(r.lb_loss, o["lb"], o["lb"], n, "lb")
    near(r.z_loss, o["z"], 2 * np.sqrt(o["z"]) * (8 * most + 32) + 16 * o["z"], 1, "z")
    near(draw, o["draw"], o["draw_mag"], 4 * n, "draw")


@dtypes
@pytest.mark.parametrize("cap", [0.01, 64.0])
def test_router_extremes_of_other_caps(pkg, dev, cap, dtype):
    """Infinities, logits far past the cap and next to zero, equal ones, with a cap far below the
    logits and with one above most; a NaN spoils its own row."""
    inf = float("inf")
    raw = torch.tensor([[1.0, 3, 3, 2, 3, 3, -1, 3], [500.0, 400, 900, 800, 1e30, 3e38, 2, 1],
                        [-inf, -inf, 5, -inf, 4, -inf, -inf, -inf], [inf, 0, inf, 1, 2, 3, 4, 5], [-inf] * 8,
                        [1e-30, -1e-30, 1e-3, -1e-3, 0, 15.9, 16.1, -16], [-1e30] * 7 + [-2e30]]).to(dtype).to(dev)
    _check_router(pkg, raw, 3, 0.5, cap, None, 1)
    bad = raw.clone()
    bad[0, 2] = float("nan")
    r, b = pkg.fused_router(raw, 3, 0.5, cap), pkg.fused_router(bad, 3, 0.5, cap)
    assert b.weights[0].isnan().all() and b.idx[0, 0] == 2 and torch.equal(r.weights[1:], b.weights[1:])


@dtypes
@pytest.mark.parametrize("capturable", [False, True])
def test_optimizer_8bit_is_the_functional_call(pkg, dev, capturable, dtype):
    """FusedAdamW(state_bits=8) over steps with a parameter that gets its gradients late, a
    transposed one and two groups, bit for bit adamw_step_8bit of the same tensors, codes, scales
    and counts: one call for the parameters of a group that have taken as many steps."""
    torch.manual_seed(0)
    shapes = [(70, 40), (300,), (9,), (33, 5)]
    ps = [torch.nn.Parameter((torch.randn(s, device=dev) * 0.05).to(dtype)) for s in shapes]
    ps[3] = torch.nn.Parameter(ps[3].detach().t().contiguous().t())
    groups = [[0, 1, 2], [3]]
    opt = pkg.FusedAdamW([{"params": ps[:3]}, {"params": ps[3:], "lr": 5e-3}], state_bits=8, seed=3,
                         capturable=capturable, **HYPER)
    q = [p.detach().clone(memory_format=torch.preserve_format) for p in ps]
    names = ("exp_avg_codes", "exp_avg_scales", "exp_avg_sq_codes", "exp_avg_sq_scales")
    st = [[torch.zeros(p.numel() if "codes" in k else -(-p.numel() // 256), device=dev,
                       dtype=torch.uint8 if "codes" in k else torch.float32) for k in names] for p in ps]
    count = [0] * 4
    for step in range(1, 6):
        for i, p in enumerate(ps):
            p.grad = None if i == 2 and step < 3 else (torch.randn(p.shape, device=dev) * 0.01).to(dtype)
        opt.step()
        for g, group in enumerate(groups):
            live = [i for i in group if ps[i].grad is not None]
            for i in live:
                count[i] += 1
            for n in sorted({count[i] for i in live}, reverse=True):
                ids = [i for i in live if count[i] == n]
                at = torch.tensor(n, device=dev) if capturable else n
                pkg.adamw_step_8bit([q[i] for i in ids], [ps[i].grad for i in ids],
                                    *[[st[i][k] for i in ids] for k in range(4)], step=at, seed=3,
                                    **{**HYPER, "lr": 5e-3 if g else HYPER["lr"]})
        for i, p in enumerate(ps):
            if not count[i]:
                assert p not in opt.state
                continue
            assert torch.equal(p.detach(), q[i]) and int(opt.state[p]["step"]) == count[i], (step, i)
            for k, t in zip(names, st[i]):
                assert torch.equal(opt.state[p][k].view(t.dtype), t), (step, i, k)
    assert count == [5, 5, 3, 5]


@pytest.mark.parametrize("E,k,tau", [(64, 2, 2.0), (256, 2, 2.0), (256, 2, 0.3), (256, 16, 2.0)])
def test_router_gradient_of_saturated_logits(pkg, dev, E, k, tau):
    """Most logits past the cap, so that many experts' probabilities are next to equal: the
    gradient of the weights in the 2-norm, by the bound of test_router_top1_weights_gradient."""
    g = torch.Generator().manual_seed(E * 7 + k)
    raw = (torch.randn(300, E, generator=g) * 30).to(dev).requires_grad_()
    dw = torch.randn(300, k, generator=g).to(dev)
    draw, = torch.autograd.grad(pkg.fused_router(raw, k, tau).weights, raw, dw)
    o = tn.router(f64(raw), k, tau, 10.0, None, f64(dw))
    assert onp.rel_l2(f64(draw), o["draw"]) <= 4 * (16 * 10 / tau + 128) * U
