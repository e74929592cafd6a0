"""The expert router on the GPU against the float64 oracle (oracle/expert_router_np.py).

Selections and counts are equal. Tolerances: a float32 evaluation of n rounded steps is off by at
most n 2^-24 times the sum of its terms' magnitudes. A weight is an exponential (4 steps with its
argument's), a quotient (3), a sum over at most 256 terms in a tree with 8 in a row (13), and
twice that for the renormalised quotient: 48. A gradient adds a sum over 16 weights and a few
products: 128. bf16 gradients add half a step, 2^-8 of themselves."""
import numpy as np
import pytest
import torch

from oracle import expert_router_np as er
from test_gpu_train_ops import DTYPES, dtypes, f64, near

pytestmark = pytest.mark.gpu


def logits(B, E, dtype, seed, std=2.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(B, E, generator=g) * std + torch.randn(E, generator=g)).to(dtype)


def biases(E, score, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(E, generator=g) * (0.1 if score == "sigmoid" else 0.3 / E)


def check(pkg, raw, k, seed=0, mask=None, bias=None, call=None, grad=True, **kw):
    B = raw.shape[0]
    dw = torch.randn(B, k, generator=torch.Generator().manual_seed(seed + 1))
    leaf = raw.detach().requires_grad_()
    args = dict(kw, bias=None if bias is None else bias.to(raw.device), mask=mask)
    r = call(leaf, args) if call else pkg.fused_expert_router(leaf, k, **args)
    o = er.route(f64(raw), k, bias=None if bias is None else f64(bias),
                 mask=None if mask is None else mask.cpu().numpy(), dw=dw.numpy(), **kw)
    assert r.idx.dtype == r.counts.dtype == torch.int64 and r.weights.dtype == torch.float32
    assert np.array_equal(r.idx.cpu().numpy(), o["idx"])
    assert np.array_equal(r.counts.cpu().numpy(), o["counts"])
    near(r.weights, o["w"], o["w"], 48, "w")
    if grad:
        draw, = torch.autograd.grad(r.weights, leaf, dw.to(raw.device))
        assert draw.dtype == raw.dtype and draw.shape == raw.shape
        near(draw, o["draw"], o["draw_mag"], 128, "draw")
    return r


@dtypes
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("B,E,k,groups,top,padded", [
    (1, 1, 1, 1, 1, 0), (1, 16, 2, 1, 1, 0), (5, 3, 3, 1, 1, 0), (257, 8, 2, 1, 1, 0.3), (1000, 33, 5, 1, 1, 0.5),
    (4096, 64, 6, 1, 1, 0), (333, 64, 16, 8, 3, 0.1), (129, 100, 4, 20, 7, 0), (70, 256, 8, 8, 4, 0.2),
    (2001, 60, 6, 6, 2, 0.25), (300, 255, 16, 5, 2, 0), (65, 128, 4, 128, 9, 0), (41, 64, 4, 64, 7, 0.1),
    (90, 24, 6, 12, 3, 0), (50, 256, 3, 2, 1, 0), (64, 40, 4, 4, 4, 0)])
def test_route(pkg, dev, B, E, k, groups, top, padded, score, dtype):
    mask = None
    if padded:
        mask = (torch.rand(B, generator=torch.Generator().manual_seed(B)) >= padded).to(dev)
    raw = logits(B, E, dtype, B + E).to(dev)
    for bias in (None, biases(E, score, E)):
        for renorm in (True, False):
            check(pkg, raw, k, B, mask, bias, score=score, groups=groups, top_groups=top, renormalize=renorm,
                  scale=2.5 if renorm else 1.0)


def test_strides_and_no_grad(pkg, dev):
    wide = logits(77, 40, torch.float32, 3).to(dev)
    mask = (torch.arange(154, device=dev) % 3 > 0)[::2]
    b = biases(80, "sigmoid", 1).to(dev)
    for raw in (wide[:, 8:24], wide[:, 1:12], wide.t()[:, :30], wide[::3, :16], wide[:1].expand(9, 40)):
        check(pkg, raw, 2, 5, bias=b[::2][:raw.shape[1]], score="sigmoid")
    check(pkg, wide, 3, 5, mask, score="softmax", groups=4, top_groups=2)
    with torch.no_grad():
        x = pkg.fused_expert_router(wide.requires_grad_(), 2)
    y = pkg.fused_expert_router(wide, 2)
    assert not x.weights.requires_grad and y.weights.requires_grad and not y.idx.requires_grad
    for p, q in zip(x, y):
        assert torch.equal(p, q)


def test_no_tokens(pkg, dev):
    raw = torch.empty(0, 8, device=dev, requires_grad=True)
    r = pkg.fused_expert_router(raw, 2, score="sigmoid", bias=torch.zeros(8, device=dev))
    assert r.idx.shape == r.weights.shape == (0, 2) and r.counts.tolist() == [0] * 8
    r.weights.sum().backward()
    assert raw.grad.shape == (0, 8)
    off = torch.zeros(5, dtype=torch.bool, device=dev)
    raw = torch.full((5, 8), float("nan"), device=dev, requires_grad=True)
    r = pkg.fused_expert_router(raw, 2, score="sigmoid", mask=off)
    r.weights.sum().backward()
    assert (r.idx == -1).all() and (r.weights == 0).all() and (raw.grad == 0).all() and r.counts.sum() == 0


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_ties_and_extremes(pkg, dev, score):
    """Equal scores: the lowest index; infinities, NaN, and sigmoids that are 0 or 1 in float64."""
    inf, nan = float("inf"), float("nan")
    raw = torch.tensor([[1.0, 3, 3, 2, 3, 3, -1, 3], [0.0, -0.0, 0, 0, -0.0, 0, 0, 0],
                        [500.0, 400, 900, 800, 1e30, 3e38, 2, 1], [-inf, -inf, 5, -inf, 4, -inf, -inf, -inf],
                        [-30.0, -31, -29, -28, -40, -50, -27, -35], [40, 41, 39, 38, 36, 50, 37, 35],
                        [-1e30] * 7 + [-2e30], [-100, -90, -95, -99, -97, -120, -130, -99]], device=dev)
    for dt in DTYPES.values():
        for kw in (dict(), dict(bias=torch.zeros(8)), dict(groups=4, top_groups=2), dict(groups=2, top_groups=1),
                   dict(bias=torch.tensor([0.1, 0, 0.1, 0, 0, 0, 0.3, -0.2]), groups=8, top_groups=3)):
            rows = raw if score == "softmax" else raw[:, :8]
            # (sigmoids past 87 below zero are no float32 numbers: their weights lose places)
            rows = rows[:6] if score == "sigmoid" else rows
            check(pkg, rows.to(dt), 2, 1, score=score, **kw)
    for kw in (dict(), dict(bias=torch.zeros(8)), dict(groups=4, top_groups=2)):
        odd = torch.tensor([[1.0, nan, 3, 2, nan, 0, -1, 3], [inf, 0, inf, 1, 2, 3, 4, 5], [-inf] * 8], device=dev)
        o = er.route(f64(odd), 2, score=score, groups=kw.get("groups", 1), top_groups=kw.get("top_groups"),
                     bias=None if "bias" not in kw else np.zeros(8))
        a = {k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in kw.items()}
        r = pkg.fused_expert_router(odd, 2, score=score, **a)
        assert np.array_equal(r.idx.cpu().numpy(), o["idx"]), kw


@dtypes
@pytest.mark.parametrize("E,k,groups,top", [(4, 4, 1, 1), (11, 11, 1, 1), (64, 6, 8, 3), (96, 16, 8, 2),
                                            (256, 16, 32, 5), (256, 4, 4, 2), (64, 6, 1, 1)])
def test_near_ties(pkg, dev, E, k, groups, top, dtype):
    """Scores, and sums of two of them, that differ in float64 and not in float32; equal ones; and
    tokens of one wave without any."""
    g = torch.Generator().manual_seed(E)
    B = 200
    raw = logits(B, E, torch.float32, E)
    close = (torch.full((B, E), 1.0).view(torch.int32) + torch.randint(0, 400, (B, E), generator=g).int()).view(torch.float32)
    raw[::2] = close[::2]
    raw[1::6] = torch.randint(0, 3, (B, E), generator=g).float()[1::6]
    raw[3::16] += 20.0                    # sigmoids a few 2^-53 below one
    for score in ("softmax", "sigmoid"):
        # biases that put the scores of every other token's logits next to each other
        even = torch.randint(-3, 4, (E,), generator=g) * 2.0 ** -22
        for bias in (None, even, biases(E, score, 2), torch.full((E,), 1e6)):
            check(pkg, raw.to(dtype).to(dev), k, 4, bias=bias, score=score, groups=groups, top_groups=top)


def test_wild_biases(pkg, dev):
    """Biases of infinity and of no number, and of a size that leaves the scores no places."""
    raw = logits(64, 16, torch.float32, 1).to(dev)
    inf, nan = float("inf"), float("nan")
    for v in ([inf, -inf] + [0.0] * 14, [nan] + [0.1] * 15, [1e30, -1e30, 3e38, -3e38] + [0.0] * 12,
              [-inf] * 16):
        b = torch.tensor(v)
        for groups, top in ((1, 1), (4, 2)):
            check(pkg, raw, 3, 2, bias=b, score="sigmoid", groups=groups, top_groups=top)


def test_dominant_weight(pkg, dev):
    """One weight next to all: the gradient is what is left of two equal terms."""
    raw = torch.full((64, 8), -12.0, device=dev)
    raw[torch.arange(64), torch.arange(64) % 8] = 6.0
    raw += logits(64, 8, torch.float32, 7, 0.3).to(dev)
    for score in ("softmax", "sigmoid"):
        check(pkg, raw, 3, 1, score=score)
        check(pkg, raw, 1, 1, score=score)


def test_second_derivative_and_tangent_are_refused(pkg, dev):
    raw = logits(8, 8, torch.float32, 1).to(dev).requires_grad_()
    w = pkg.fused_expert_router(raw, 2, score="sigmoid").weights
    d, = torch.autograd.grad(w.square().sum(), raw, create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        d.sum().backward()


def test_captured_and_streams(pkg, dev):
    """A captured forward and backward replayed on new logits, eager calls in between, and a call
    on another stream."""
    B, E, k = 3000, 64, 6
    kw = dict(score="sigmoid", groups=8, top_groups=4, scale=2.0)
    bias = biases(E, "sigmoid", 3).to(dev)
    raw = logits(B, E, torch.float32, 1).to(dev).requires_grad_()
    dw = torch.randn(B, k, device=dev)

    def step(x):
        r = pkg.fused_expert_router(x, k, bias=bias, **kw)
        return (*r, torch.autograd.grad(r.weights, x, dw)[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(raw)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(raw)
    for seed in range(4):
        new = logits(B, E, torch.float32, 10 + seed).to(dev)
        with torch.no_grad():
            raw.copy_(new)
        graph.replay()
        want = step(new.requires_grad_())
        torch.cuda.synchronize()
        for p, q in zip(out, want):
            assert torch.equal(p, q)
    with torch.cuda.stream(side):
        other = step(new)
    side.synchronize()
    for p, q in zip(other, want):
        assert torch.equal(p, q)


@dtypes
@pytest.mark.parametrize("E,k,groups,top", [(4, 2, 1, 1), (8, 1, 1, 1), (64, 6, 8, 3), (256, 16, 1, 1)])
def test_small_selected_scores(pkg, dev, E, k, groups, top, dtype):
    """A bias that selects experts whose softmax scores lie 20 to 80 below another's: 1e-20 is a part,
    or all, of what a weight is divided by, and the other expert has a gradient too.

    Logits T apart have a difference that float32 rounds by 2^-24 T, and an exponential takes that as it
    is: T steps for a score and for a sum of them, 2 T for a weight (beside its 48). A selected gradient is
    w (g - top - D + top r): 2 T of w, 2 T of D's weights and T of r, another's s r (D + ...) less than that:
    5 T beside the 128. The kernel leaves r out below 2^-20: 16 steps, and as many of its sum's. A score
    below float32's normal numbers may be lost: 2^-126 over the 1e-20 in a weight."""
    g = torch.Generator().manual_seed(E)
    B = 200
    raw = torch.randn(B, E, generator=g)
    raw[:, E - 1] += torch.linspace(20, 80, B)
    bias = torch.zeros(E)
    bias[:E - E // groups] = 3.0            # (never the last group)
    if groups == 1:
        bias[:E - 1] = 3.0
    bias += 0.1 * torch.randn(E, generator=g)
    raw = raw.to(dtype).to(dev)
    T = float((raw.amax(-1) - raw.amin(-1)).max())
    dw = torch.randn(B, k, generator=g)
    some = (torch.rand(B, generator=g) < 0.7).to(dev)
    for mask, scale, renorm in ((None, 1.0, True), (None, 2.5, True), (some, 2.5, True), (some, 1.0, False)):
        kw = dict(groups=groups, top_groups=top, scale=scale, renormalize=renorm)
        leaf = raw.clone().requires_grad_()
        r = pkg.fused_expert_router(leaf, k, bias=bias.to(dev), mask=mask, **kw)
        o = er.route(f64(raw), k, bias=f64(bias), mask=None if mask is None else mask.cpu().numpy(),
                     dw=dw.numpy(), **kw)
        assert np.array_equal(r.idx.cpu().numpy(), o["idx"]) and not (r.idx == E - 1).any()
        lost = scale * 2.0 ** -126 / (1e-20 if renorm else 1.0)
        n, m = 48 + 2 * T, 128 + 5 * T + 32
        near(r.weights, o["w"], o["w"] + lost / (n * 2.0 ** -24), n, "w")
        draw, = torch.autograd.grad(r.weights, leaf, dw.to(dev))
        far = 4 * float(dw.abs().max())
        near(draw, o["draw"], o["draw_mag"] + far * lost / (m * 2.0 ** -24), m, "draw")


@dtypes
@pytest.mark.parametrize("E,k,groups,top", [(4, 2, 1, 1), (8, 1, 1, 1), (64, 6, 8, 3)])
def test_small_sigmoids(pkg, dev, E, k, groups, top, dtype):
    """Sigmoids of 20 to 80 below zero: 1e-20 is a part, or all, of what a weight is divided by."""
    raw = torch.randn(200, E, generator=torch.Generator().manual_seed(E)) - torch.linspace(20, 80, 200)[:, None]
    raw = raw.to(dtype).to(dev)
    for bias in (None, biases(E, "sigmoid", 1)):
        check(pkg, raw, k, 3, bias=bias, score="sigmoid", groups=groups, top_groups=top, scale=2.5)
