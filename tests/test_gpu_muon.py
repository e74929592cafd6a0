"""The Muon step on the GPU against the float64 oracle (oracle/muon_np.py), whose `off` is what X may
be off in the Frobenius norm by the roundings of the products and what the polynomial makes of
them; a result in bfloat16 adds half a step, 2^-8 of itself, and one in float32 2^-24 for each of
the update's three operations. Momenta are off by two roundings."""
import numpy as np
import pytest
import torch

from oracle import muon_np as mn
from test_gpu_train_ops import DTYPES, dtypes, f64

pytestmark = pytest.mark.gpu


def norm(x):
    return np.sqrt((x * x).sum((-1, -2)))


def matrices(shape, seed, rank=None):
    g = torch.Generator().manual_seed(seed)
    u = torch.randn(shape, generator=g)
    if rank:        # a few directions and a thousandth of noise
        u = (torch.randn(*shape[:-1], rank, generator=g) @ torch.randn(*shape[:-2], rank, shape[-1], generator=g)
             + 1e-3 * u)
    return u


def near(got, want, off, what=""):
    e = norm(f64(got) - want)
    half = 2.0 ** -8 if got.dtype == torch.bfloat16 else 2.0 ** -22
    assert np.all(e <= off * 1.01 + half * norm(want) + 1e-30), (what, float((e / (off + half * norm(want))).max()))


SHAPES = [(1, 1), (1, 37), (64, 64), (65, 64), (37, 1), (128, 200), (257, 33), (3, 65, 129), (2, 3, 40, 30),
          (1001, 77), (129, 4097), (300, 300), (512, 128), (256, 1024)]


@dtypes
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_orthogonalize(pkg, dev, shape, dtype):
    for rank, scale in ((None, 1.0), (2, 1e-4), (None, 1e4)):
        u = (matrices(shape, sum(shape), rank) * scale).to(dtype)
        X, off = mn.orthogonalize(f64(u))
        got = pkg.orthogonalize(u.to(dev))
        assert got.shape == u.shape and got.dtype == dtype
        near(got, X, off, (rank, scale))
    for steps, c in ((1, mn.COEFFICIENTS), (3, (1.875, -1.25, 0.375)), (16, (1.5, -0.5, 0.0))):
        X, off = mn.orthogonalize(f64(u), steps, c)
        near(pkg.orthogonalize(u.to(dev), steps, c), X, off, steps)


@dtypes
def test_many_at_once_and_alone(pkg, dev, dtype):
    """A list in one call is each of its matrices by itself, with tiles of both sizes."""
    us = [matrices(s, i).to(dtype).to(dev) for i, s in enumerate(SHAPES)]
    alone = [pkg.orthogonalize(u) for u in us]
    for u, x, y in zip(us, alone, pkg.orthogonalize(us)):
        assert torch.equal(x, y), u.shape
    more = us * 6 + [matrices((40, 256, 512), 3).to(dtype).to(dev)]      # wide tiles, several tables
    for i, (u, y) in enumerate(zip(more, pkg.orthogonalize(more))):
        X, off = mn.orthogonalize(f64(u))
        near(y, X, off, i)
    strided = [us[5][::2], us[5].t(), us[9][:, 5:], us[8][:, 1], us[0].expand(5, 3)]
    for u, y in zip(strided, pkg.orthogonalize(strided)):
        X, off = mn.orthogonalize(f64(u))
        near(y, X, off)


def test_zero_empty_and_not_finite(pkg, dev):
    z = torch.zeros(3, 20, 30, device=dev)
    z[1] = matrices((20, 30), 1).to(dev)
    x = pkg.orthogonalize(z)
    assert (x[0] == 0).all() and (x[2] == 0).all() and (x[1] != 0).any()
    outs = pkg.orthogonalize([z[:0], z[:, :0], z, z[:, :, :0]])
    assert [tuple(o.shape) for o in outs] == [(0, 20, 30), (3, 0, 30), (3, 20, 30), (3, 20, 0)]
    assert torch.equal(outs[2], x)
    for bad in (float("nan"), float("inf")):
        y = z.clone()
        y[0, 3, 4] = bad
        got = pkg.orthogonalize(y)
        assert not torch.isfinite(got[0]).any() and torch.equal(got[1:], x[1:])


def _lists(shapes, dtype, dev, seed=0):
    p = [(matrices(s, seed + i) * 0.03).to(dtype).to(dev) for i, s in enumerate(shapes)]
    g = [(matrices(s, seed + 50 + i, 4) * 1e-3).to(dtype).to(dev) for i, s in enumerate(shapes)]
    m = [(matrices(s, seed + 90 + i, 4) * 5e-3).to(dev) for i, s in enumerate(shapes)]
    return p, g, m


@dtypes
@pytest.mark.parametrize("nesterov", [True, False])
def test_step(pkg, dev, dtype, nesterov):
    p, g, m = _lists(SHAPES, dtype, dev)
    want = [mn.muon(f64(a), f64(b), f64(c), 0.02, nesterov=nesterov) for a, b, c in zip(p, g, m)]
    mag = [0.95 * np.abs(f64(c)) + np.abs(f64(b)) for b, c in zip(g, m)]
    versions = [t._version for t in p + m]
    pkg.muon_step(p, g, m, lr=0.02, nesterov=nesterov)
    assert all(t._version > v for t, v in zip(p + m, versions))
    for a, c, o, s, q in zip(p, m, want, SHAPES, mag):
        near(a, o["p"], o["off"], s)
        assert np.all(np.abs(f64(c) - o["m"]) <= 2.0 ** -23 * q + 1e-37), s
    # gradients in another order of memory, and offsets that no wide load is aligned to
    p, g, m = _lists([(33, 65), (65, 33)], dtype, dev, 7)
    base = torch.zeros(2 * 33 * 65 + 1, dtype=dtype, device=dev)
    p2 = [base[1:1 + 33 * 65].view(33, 65), base[1 + 33 * 65:].view(65, 33)]
    for x, y in zip(p2, p):
        x.copy_(y)
    m2 = [x.clone() for x in m]
    pkg.muon_step(p, g, m, lr=0.1)
    pkg.muon_step(p2, [x.t().contiguous().t() for x in g], m2, lr=0.1)
    for x, y in zip(p + m, p2 + m2):
        assert torch.equal(x, y)


def test_no_decay_and_full_decay(pkg, dev):
    p, g, m = _lists([(40, 70)], torch.float32, dev)
    for lr, wd in ((0.0, 0.1), (0.5, 0.0), (0.5, 2.0)):
        q, n = [p[0].clone()], [m[0].clone()]
        o = mn.muon(f64(p[0]), f64(g[0]), f64(m[0]), lr, wd=wd)
        pkg.muon_step(q, g, n, lr=lr, weight_decay=wd)
        e = norm(f64(q[0]) - o["p"])
        assert e <= 1.01 * o["off"] + 2.0 ** -22 * (norm(f64(p[0])) + norm(o["p"]))


def test_captured_streams_and_repeats(pkg, dev):
    """The same bits each time: on another stream, captured and replayed with eager steps between."""
    shapes = [(512, 128), (256, 1024), (4, 128, 256), (33, 65)]
    p, g, m = _lists(shapes, torch.bfloat16, dev)
    q, n = [x.clone() for x in p], [x.clone() for x in m]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        pkg.muon_step(q, g, n, lr=0.02)
    torch.cuda.current_stream().wait_stream(side)
    pkg.muon_step(p, g, m, lr=0.02)
    for x, y in zip(p + m, q + n):
        assert torch.equal(x, y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pkg.muon_step(p, g, m, lr=0.02)
    for seed in range(4):
        for x, y in zip(g, _lists(shapes, torch.bfloat16, dev, 100 + seed)[1]):
            x.copy_(y)
        graph.replay()
        pkg.muon_step(q, g, n, lr=0.02)
        torch.cuda.synchronize()
        for x, y in zip(p + m, q + n):
            assert torch.equal(x, y)


@pytest.mark.parametrize("shape", [(256, 512), (512, 128), (3, 300, 200), (64, 64)], ids=lambda s: "x".join(map(str, s)))
def test_single_elements_of_a_step(pkg, dev, shape):
    """One step, element by element: a few elements' parts of 11 bits that do not belong together hide
    in a norm (each is off by 2^-11 of itself). The result is a polynomial of fifth degree in X, of
    magnitude a |X| + |b| |X||X|^T|X| + |c| (|X||X|^T)^2 |X|. X, A (three times) and B are held to 2^-23 of
    themselves, five factors X in a term; products of two low parts, 2^-24 of the whole, are left out of
    four products, and each adds as many terms as its axis is long: with Gram products over the long axis L
    (twice) and two over the short one S, at most (2 L + 2 S + 2 (5 + 3 + 1) + 4) 2^-24, here + 40. What
    is smaller than fp16's smallest numbers, 2^-25 / 2048 of X's elements, is below 1e-9."""
    a, b, c = 3.4445, -4.7750, 2.0315
    for seed in range(4):
        u = matrices(shape, seed).to(dev)
        x = u.double()
        x = x / (x.flatten(-2).norm(dim=-1)[..., None, None] + 1e-7)
        t = x if shape[-2] <= shape[-1] else x.transpose(-1, -2)
        m = t.abs()
        A, M = t @ t.transpose(-1, -2), m @ m.transpose(-1, -2)
        want, mag = a * t + (b * A + c * (A @ A)) @ t, a * m + (abs(b) * M + c * (M @ M)) @ m
        if t is not x:
            want, mag = want.transpose(-1, -2), mag.transpose(-1, -2)
        off = (pkg.orthogonalize(u, steps=1).double() - want).abs()
        n = 2 * max(shape[-2:]) + 2 * min(shape[-2:]) + 40
        assert (off <= n * 2.0 ** -24 * mag + 1e-9).all(), (seed, float((off / mag).max()))


def test_optimizer(pkg, dev):
    """FusedMuon's steps are the functional call's, through its state dict and in a capture."""
    shapes = [(40, 70), (3, 65, 33), (128, 64)]
    p, g, m = _lists(shapes, torch.float32, dev)
    m = [torch.zeros_like(x) for x in m]
    params = [torch.nn.Parameter(x.clone()) for x in p]
    half = torch.nn.Parameter(matrices((20, 30), 5).bfloat16().to(dev))
    idle = torch.nn.Parameter(torch.ones(3, 3, device=dev))
    opt = pkg.FusedMuon([{"params": params + [idle]}, {"params": [half], "lr": 0.1, "nesterov": False}])
    hp, hm = half.detach().clone(), torch.zeros(20, 30, device=dev)

    def step(o, ps, h, seed):
        for x, y in zip(ps, _lists(shapes, torch.float32, dev, seed)[1]):
            x.grad = y
        h.grad = matrices((20, 30), seed + 1).bfloat16().to(dev)
        o.step()
    for seed in (1, 2):
        step(opt, params, half, seed)
        pkg.muon_step(p, [x.grad for x in params], m, lr=2e-2)
        pkg.muon_step([hp], [half.grad], [hm], lr=0.1, nesterov=False)
    for x, y in zip(params, p):
        assert torch.equal(x.detach(), y)
    assert torch.equal(half.detach(), hp) and (idle == 1).all() and idle not in opt.state
    again = [torch.nn.Parameter(x.detach().clone()) for x in params]
    half2, idle2 = torch.nn.Parameter(half.detach().clone()), torch.nn.Parameter(torch.ones(3, 3, device=dev))
    other = pkg.FusedMuon([{"params": again + [idle2]}, {"params": [half2]}])
    other.load_state_dict(opt.state_dict())
    step(opt, params, half, 3)
    step(other, again, half2, 3)
    for x, y in zip(params + [half], again + [half2]):
        assert torch.equal(x.detach(), y.detach())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    graph.replay()
    other.step()
    torch.cuda.synchronize()
    for x, y in zip(params + [half], again + [half2]):
        assert torch.equal(x.detach(), y.detach())
    fresh = torch.nn.Parameter(torch.ones(4, 4, device=dev))
    fresh.grad = torch.ones(4, 4, device=dev)
    first = pkg.FusedMuon([fresh])
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="first step"):
        with torch.cuda.graph(graph):
            first.step()
    assert fresh not in first.state or not first.state[fresh]


@dtypes
@pytest.mark.parametrize("scale", [1e15, 1e20, 3e30, 1e-18, 1e-25, 3e-36])
def test_squares_past_float32(pkg, dev, scale, dtype):
    """Finite matrices the sum of whose squares leaves float32 at either end are orthogonalised as any
    others are, and matrices of zeros beside them stay zeros with the smallest eps."""
    us = [(matrices(s, 9) * scale).to(dtype) for s in ((40, 70), (130, 64), (3, 20, 33))]
    us[2][1] = 0
    eps = 1e-37 if scale < 1 else 1e-7
    for u, got in zip(us, pkg.orthogonalize([u.to(dev) for u in us], eps=eps)):
        X, off = mn.orthogonalize(f64(u), eps=eps)
        near(got, X, off, scale)
    assert (got[1] == 0).all()
    p, _, m = _lists([(40, 70)], dtype, dev)
    o = mn.muon(f64(p[0]), f64(us[0]), f64(m[0]) * scale, 0.02, eps=eps)
    q = [m[0] * scale]
    pkg.muon_step(p, [us[0].to(dev)], q, lr=0.02, eps=eps)
    near(p[0], o["p"], o["off"], scale)


def test_wide_tiles_element_by_element(pkg, dev):
    """test_single_elements_of_a_step's bound in the kernels of 128 x 128 tiles: many matrices at once,
    wide and tall, with ragged edges and with Gram products cut into slices."""
    a, b, c = 3.4445, -4.7750, 2.0315
    shapes = [(40, 256, 512), (512, 128), (300, 200), (129, 4097), (257, 33), (4097, 130), (1001, 77)]
    us = [matrices(s, i).to(dev) for i, s in enumerate(shapes)]
    for u, got in zip(us, pkg.orthogonalize(us, steps=1)):
        x = u.double()
        x = x / (x.flatten(-2).norm(dim=-1)[..., None, None] + 1e-7)
        t = x if u.shape[-2] <= u.shape[-1] else x.mT
        m = t.abs()
        A, M = t @ t.mT.contiguous(), m @ m.mT.contiguous()
        want, mag = a * t + (b * A + c * (A @ A)) @ t, a * m + (abs(b) * M + c * (M @ M)) @ m
        if t is not x:
            want, mag = want.mT, mag.mT
        off = (got.double() - want).abs()
        n = 2 * max(u.shape[-2:]) + 2 * min(u.shape[-2:]) + 40
        assert (off <= n * 2.0 ** -24 * mag + 1e-9).all(), (u.shape, float((off / mag).max()))


def test_a_refused_step_changes_nothing(pkg, dev):
    """Of two groups the second is refused: parameters, momenta and states are as they were."""
    def build(extra, **kw):
        a = torch.nn.Parameter(matrices((40, 70), 1).to(dev))
        b = torch.nn.Parameter(matrices((20, 30), 2).bfloat16().to(dev))
        return [a, b, extra], pkg.FusedMuon([{"params": [a, b]}, {"params": [extra], **kw}], lr=0.1)

    def grads(ps):
        for i, p in enumerate(ps):
            p.grad = torch.ones_like(p) * (i + 1)
    good = lambda: torch.nn.Parameter(matrices((6, 9), 3).to(dev))  # noqa: E731
    base = torch.zeros(200, device=dev)
    cases = [(torch.nn.Parameter(matrices((9, 6), 3).to(dev).t()), "contiguous"),
             (torch.nn.Parameter(matrices((6, 9), 3).half().to(dev)), "dtype"),
             (torch.nn.Parameter(matrices((6, 9), 3)), "HIP devices only")]
    for extra, text in cases:
        ps, opt = build(extra)
        grads(ps)
        before = [p.detach().clone() for p in ps]
        for _ in range(2):
            with pytest.raises(RuntimeError, match=text):
                opt.step()
            assert all(torch.equal(p.detach(), q) for p, q in zip(ps, before))
            assert not any(opt.state.get(p) for p in ps)
    for key, bad in (("lr", -1.0), ("momentum", 1.0), ("lr", float("inf")), ("steps", 99), ("coefficients", (5.0, 0.0, 0.0))):
        ps, opt = build(good())
        grads(ps)
        opt.step()
        before = [t.clone() for p in ps for t in (p.detach(), opt.state[p]["momentum_buffer"])]
        keep = opt.param_groups[1][key]
        opt.param_groups[1][key] = bad
        with pytest.raises((ValueError, RuntimeError)):
            opt.step()
        after = [t for p in ps for t in (p.detach(), opt.state[p]["momentum_buffer"])]
        assert all(torch.equal(x, y) for x, y in zip(before, after))
        opt.param_groups[1][key] = keep
        opt.step()
        assert not any(torch.equal(x, y) for x, y in zip(before, after))
    # a run by itself whose tensors share memory, and a state that is not float32
    one, two = (torch.nn.Parameter(base[i:i + 100].view(10, 10)) for i in (0, 50))
    opt = pkg.FusedMuon([one, two])
    grads([one, two])
    with pytest.raises(RuntimeError, match="share"):
        opt.step()
    assert (base == 0).all() and not opt.state.get(one) and not opt.state.get(two)
    ps, opt = build(good())
    grads(ps)
    opt.state[ps[2]]["momentum_buffer"] = torch.zeros(6, 9, device=dev, dtype=torch.bfloat16)
    before = [p.detach().clone() for p in ps]
    with pytest.raises(RuntimeError, match="momentum of float32"):
        opt.step()
    assert all(torch.equal(p.detach(), q) for p, q in zip(ps, before)) and not opt.state.get(ps[0])
