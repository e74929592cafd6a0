"""Performance cases of the training layer's wider operators: which experts, in how many bits,
and what update.

  route   fused_expert_router: softmax or sigmoid scores, a balancing bias, groups of experts,
          top-k, renormalised weights and per-expert counts, and the gradient of the logits
  fp8     fp8_matmul (products in 8-bit floating point, a scale for each block of 128, forward
          and both gradients) and fp8_block_matmul (on weights held in 8 bits)
  muon    muon_step: momentum, orthogonalisation by Newton-Schulz products and the update of
          all matrices of a model

prepare() makes a case's inputs on the GPU from its seed, run() makes one pass: with
`own` false in elementary torch operations in 32 bits (a router's ranks in 64), with `own`
true through this framework's entry points. exact() gives the same outputs in 64 bits. Sizes
are those of the workloads C1..C5, F1 / F2 and the reference model's layers, or generic.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_PKG = "mamba_tuckermoe_amd"
_DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
_RENORM_EPS = 1e-20
_ROUTE_SCALE = 2.5
_BLOCK = 128           # elements that share a scale
_E4M3_MAX = 448.0
_TINY = 2.0 ** -100    # blocks of no larger magnitude than this are stored as zeros
_LR, _MOMENTUM, _DECAY, _RMS, _STEPS, _NORM_EPS = 0.02, 0.95, 0.1, 0.2, 5, 1e-7
_NS = (3.4445, -4.7750, 2.0315)


def _package():
    """The package, whose folder's name is no Python identifier."""
    if _PKG not in sys.modules:
        d = os.path.join(_ROOT, "mamba-tuckermoe_amd")
        spec = importlib.util.spec_from_file_location(
            _PKG, os.path.join(d, "__init__.py"), submodule_search_locations=[d])
        sys.modules[_PKG] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules[_PKG])
    return sys.modules[_PKG]


# ---- cases ---------------------------------------------------------------------

def _route(B, E, k, score, bias=True, groups=1, top_groups=1, dtype="fp32", padded=0.0, renorm=True):
    return dict(kind="route", B=B, E=E, k=k, score=score, bias=bias, groups=groups,
                top_groups=top_groups, dtype=dtype, padded=padded, renorm=renorm)


def _linear(M, K, N, dtype="bf16"):
    return dict(kind="linear", M=M, K=K, N=N, dtype=dtype)


def _held(M, K, N, dtype="bf16"):
    return dict(kind="held", M=M, K=K, N=N, dtype=dtype)


def _muon(model, layers=1, dtype="fp32"):
    return dict(kind="muon", model=model, layers=layers, dtype=dtype)


def listed():
    return [
        # one token's routing in serving or an online update: launch and host latency
        dict(_route(1, 16, 2, "sigmoid"), name="route_B1_E16_sigmoid"),
        # the training batch's router under autocast, experts in groups, no bias yet
        dict(_route(16384, 64, 6, "softmax", bias=False, groups=8, top_groups=3, dtype="bf16"),
             name="route_B16384_E64_softmax_groups"),
        # a wide router (C4's experts and top-8), balanced by its bias within half of the groups
        dict(_route(4096, 256, 8, "sigmoid", groups=8, top_groups=4),
             name="route_B4096_E256_sigmoid_groups"),
        # a large batch of padded sequences: three tokens in ten are padding
        dict(_route(131072, 64, 6, "sigmoid", padded=0.3), name="route_B131072_E64_sigmoid_padded"),
        # one token through a projection whose weights are held in 8 bits (d_in to the widest d_out)
        dict(_held(1, 1536, 6144), name="fp8_held_M1_K1536_N6144"),
        # a prompt through the same form of weights (C3's output side)
        dict(_held(16384, 1024, 2304), name="fp8_held_M16384_K1024_N2304"),
        # a ragged batch's in-projection to rank 256, with its gradients
        dict(_linear(5003, 1536, 256, "fp32"), name="fp8_linear_M5003_K1536_N256"),
        # the training batch's widest products (F1's widths), with their gradients
        dict(_linear(16384, 768, 4608), name="fp8_linear_M16384_K768_N4608"),
        # the matrices of one small layer (C1): latency
        dict(_muon("c1"), name="muon_c1"),
        # matrices of odd sizes, tall and wide, and a vector's worth
        dict(_muon("odd"), name="muon_odd"),
        # the FFN sub-block in bf16
        dict(_muon("ffn", dtype="bf16"), name="muon_ffn"),
        # all 66 layers of the reference model
        dict(_muon("reference"), name="muon_reference"),
    ]


def _log_int(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["route", "linear", "held", "muon"])
    if kind == "route":
        groups = rng.choice([1, 1, 2, 4, 8, rng.randint(3, 16)])
        E = groups * _log_int(rng, 2, 256 // groups)
        top = rng.randint(1, groups)
        k = rng.randint(1, min(top * (E // groups), 8))
        # (one renormalised weight is a constant: nobody trains that)
        return _route(_log_int(rng, 1, min(262144, 2 ** 23 // E)), E, k, rng.choice(["softmax", "sigmoid"]),
                      rng.random() < 0.6, groups, top, rng.choice(["fp32", "bf16"]),
                      rng.choice([0.0, 0.0, rng.uniform(0.0, 0.9)]), k > 1 and rng.random() < 0.7)
    if kind == "muon":
        return _muon(rng.choice(["c1", "c3", "ffn", "odd"]), rng.randint(1, 12), rng.choice(["fp32", "bf16"]))
    M = _log_int(rng, 1, 16384)
    K, N = (rng.choice([_log_int(rng, 64, 4608), 128 * _log_int(rng, 1, 36)]) for _ in range(2))
    while M * K * N > 16384 * 768 * 4608:
        M //= 2
    return (_linear if kind == "linear" else _held)(M, K, N, rng.choice(["bf16", "bf16", "fp32"]))


# ---- inputs --------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, shape, std=1.0):
    return torch.randn(shape, generator=g, device="cuda") * std


def _route_inputs(case, seed):
    g, dt = _gen(seed), _DT[case["dtype"]]
    B, E, k = case["B"], case["E"], case["k"]
    # logits of a trained router: some experts likelier than others
    raw = (_normal(g, (B, E), 1.5) + _normal(g, (E,), 0.7)).to(dt)
    bias = None
    if case["bias"]:
        bias = _normal(g, (E,), 0.1 if case["score"] == "sigmoid" else 0.3 / E)
    mask = None
    if case["padded"]:
        mask = torch.rand(B, generator=g, device="cuda") >= case["padded"]
    return {"raw": raw, "bias": bias, "mask": mask, "dw": _normal(g, (B, k))}


def _activations(g, M, K, dtype):
    """A normed hidden state: a few channels much larger than the others."""
    wide = 1 + 20 * (torch.rand(K, generator=g, device="cuda") < 0.01)
    return (_normal(g, (M, K)) * wide).to(dtype)


def _linear_inputs(case, seed):
    g, dt = _gen(seed), _DT[case["dtype"]]
    M, K, N = case["M"], case["K"], case["N"]
    return (_activations(g, M, K, dt), _normal(g, (K, N), K ** -0.5).to(dt),
            (_normal(g, (M, N)) * torch.exp(_normal(g, (M, 1)))).to(dt))


def _muon_shapes(case):
    def layer(d_in, d_out, r1, r2, r3):     # U_in, U_out and the core's matrices
        return [(d_in, r3), (r2, d_out), (r1, r3, r2)]
    up, out = layer(1536, 6144, 32, 512, 256), layer(768, 768, 32, 512, 256)
    wide, down = layer(768, 4608, 32, 512, 256), layer(4608, 768, 32, 512, 256)
    shapes = {"c1": layer(512, 1024, 4, 256, 128), "c3": layer(1536, 2304, 4, 1024, 256),
              "odd": [(1, 37), (257, 33), (3, 65, 129), (1001, 77), (255, 511), (31, 31)],
              "ffn": wide + wide + down,
              "reference": 24 * (up + out) + 6 * (wide + wide + down)}[case["model"]]
    return shapes * case["layers"]


def _muon_inputs(case, seed):
    """Parameters, gradients and momenta, a flat buffer each, and the tensors' shapes."""
    g, dt = _gen(seed), _DT[case["dtype"]]
    shapes = _muon_shapes(case)
    p = _normal(g, (sum(math.prod(s) for s in shapes),), 0.03).to(dt)
    grad, m = torch.empty_like(p), torch.empty_like(p, dtype=torch.float32)
    for s, gv, mv in zip(shapes, _views(grad, shapes), _views(m, shapes)):
        # gradients of a low rank and noise about it, as a projection's are
        a, b = _normal(g, (*s[:-1], 8)), _normal(g, (*s[:-2], 8, s[-1]))
        low = a @ b
        gv.copy_(1e-3 * (low + _normal(g, s)))
        mv.copy_(5e-3 * (low + _normal(g, s)))
    return p, grad, m, shapes


def _views(flat, shapes):
    at, out = 0, []
    for s in shapes:
        n = math.prod(s)
        out.append(flat[at:at + n].view(s))
        at += n
    return out


def _blocks(x, rows):
    """x (R, K) in blocks of `rows` x 128, padded with zeros: (R', rows, K', 128)."""
    R, K = x.shape
    x = torch.nn.functional.pad(x, (0, -K % _BLOCK, 0, -R % rows))
    return x.view(-1, rows, x.shape[1] // _BLOCK, _BLOCK)


def _quantised(x, rows):
    """(codes (R, K padded to 128), scales) of x in blocks of `rows` x 128, 32-bit arithmetic."""
    b = _blocks(x.float(), rows)
    top = b.abs().amax((1, 3))
    on = top > _TINY
    safe, most = torch.where(on, top, 1.0), torch.full_like(top, _E4M3_MAX)
    # quotients of two tensors: torch makes a product of one by a number
    inv = torch.where(on, torch.div(most, safe), 0.0)
    q = (b * inv[:, None, :, None]).to(torch.float8_e4m3fn)
    q = q.view(-1, b.shape[2] * _BLOCK)[:x.shape[0]].contiguous()
    return q, torch.where(on, torch.div(safe, most), 0.0)


def prepare(case, seed):
    if case["kind"] == "route":
        s = _route_inputs(case, seed)
        s["raw"].requires_grad_()
        return {**case, **s}
    if case["kind"] == "linear":
        x, w, dy = _linear_inputs(case, seed)
        return {"kind": "linear", "x": x.requires_grad_(), "w": w.requires_grad_(), "dy": dy}
    if case["kind"] == "held":
        x, w, _ = _linear_inputs(case, seed)
        codes, scales = _quantised(w.t().contiguous(), _BLOCK)
        return {"kind": "held", "x": x, "codes": codes, "scales": scales, "K": case["K"]}
    p, g, m, shapes = _muon_inputs(case, seed)
    return {"kind": "muon", "p": p, "m": m, "params": _views(p, shapes), "grads": _views(g, shapes),
            "momenta": _views(m, shapes)}


# ---- a pass --------------------------------------------------------------------

def _plain_route(s):
    raw, k, mask, groups = s["raw"].detach().float(), s["k"], s["mask"], s["groups"]
    B, E = raw.shape
    if mask is not None:
        raw = torch.where(mask[:, None], raw, 0.0)
    softmax = s["score"] == "softmax"
    fine = torch.softmax(raw.double(), -1) if softmax else torch.sigmoid(raw.double())
    rank = fine if s["bias"] is None else fine + s["bias"].double()
    if groups > 1:
        by = rank.view(B, groups, -1)
        best = torch.sort(by, dim=-1, descending=True).values[..., :2].sum(-1)
        kept = torch.sort(best, dim=-1, descending=True, stable=True).indices[:, :s["top_groups"]]
        open_ = torch.zeros(B, groups, dtype=torch.bool, device=raw.device).scatter_(1, kept, True)
        rank = torch.where(open_[..., None], by, -math.inf).view(B, E)
    elif s["bias"] is None:
        rank = raw                       # both scores are monotone
    idx = torch.sort(rank, dim=-1, descending=True, stable=True).indices[:, :k]
    p = torch.softmax(raw, -1) if softmax else torch.sigmoid(raw)
    top = p.gather(-1, idx)
    total = top.sum(-1, keepdim=True) + _RENORM_EPS
    w = _ROUTE_SCALE * (top / total if s["renorm"] else top)
    # the gradient: of the selected scores, then of the logits
    dw = s["dw"]
    dt = _ROUTE_SCALE * dw
    if s["renorm"]:
        dt = _ROUTE_SCALE / total * (dw - (dw * top).sum(-1, keepdim=True) / total)
    dp = torch.zeros_like(p).scatter_(1, idx, dt)
    draw_ = p * (dp - (dp * p).sum(-1, keepdim=True)) if softmax else dp * p * (1 - p)
    keep = torch.ones(B, dtype=torch.int64, device=raw.device) if mask is None else mask.to(torch.int64)
    counts = torch.zeros(E, dtype=torch.int64, device=raw.device)
    counts = counts.index_add(0, idx.reshape(-1), keep.repeat_interleave(k))
    if mask is not None:
        idx, w = torch.where(mask[:, None], idx, -1), torch.where(mask[:, None], w, 0.0)
        draw_ = torch.where(mask[:, None], draw_, 0.0)
    return {"idx": idx, "w": w, "counts": counts, "draw": draw_.to(s["raw"].dtype)}


def _values(codes, scales, rows, K):
    v = _blocks(codes.float(), rows) * scales[:, None, :, None]
    return v.view(-1, v.shape[2] * _BLOCK)[:codes.shape[0], :K]


def _rounded(x, rows):
    """The values that x's codes and scales stand for."""
    return _values(*_quantised(x, rows), rows, x.shape[1])


def _plain_linear(x, w, dy):
    wv = _rounded(w.t(), _BLOCK)                                    # (N, K)
    y = _rounded(x, 1) @ wv.t()
    dx = _rounded(dy, 1) @ wv
    dw = _rounded(x.t(), 1) @ _rounded(dy.t(), 1).t()
    return {"y": y.to(x.dtype), "dx": dx.to(x.dtype), "dw": dw.to(x.dtype)}


def _plain_orthogonal(u):
    wide = u.shape[-2] > u.shape[-1]
    X = u.transpose(-1, -2) if wide else u
    X = X / (torch.sqrt((X * X).sum((-2, -1), keepdim=True)) + _NORM_EPS)
    a, b, c = _NS
    for _ in range(_STEPS):
        A = X @ X.transpose(-1, -2).contiguous()
        X = a * X + (b * A + c * (A @ A)) @ X
    return X.transpose(-1, -2) if wide else X


def _plain_muon(p, g, m):
    g = g.float()
    m.mul_(_MOMENTUM).add_(g)
    o = _plain_orthogonal(g + _MOMENTUM * m)
    s = _RMS * math.sqrt(max(p.shape[-2:]))
    p.copy_(p.float() * (1 - _LR * _DECAY) - _LR * s * o)


def run(state):
    kind = state["kind"]
    if kind == "route":
        if not own:
            return _plain_route(state)
        r = _package().fused_expert_router(
            state["raw"], state["k"], score=state["score"], bias=state["bias"], groups=state["groups"],
            top_groups=state["top_groups"], renormalize=state["renorm"], scale=_ROUTE_SCALE,
            mask=state["mask"])
        draw_, = torch.autograd.grad(r.weights, state["raw"], state["dw"])
        return {"idx": r.idx, "w": r.weights.detach(), "counts": r.counts, "draw": draw_}
    if kind == "linear":
        x, w, dy = state["x"], state["w"], state["dy"]
        if not own:
            with torch.no_grad():
                return _plain_linear(x, w, dy)
        y = _package().fp8_matmul(x, w)
        dx, dw = torch.autograd.grad(y, (x, w), dy)
        return {"y": y.detach(), "dx": dx, "dw": dw}
    if kind == "held":
        x = state["x"]
        if not own:
            wv = _values(state["codes"], state["scales"], _BLOCK, state["K"])
            return (_rounded(x, 1) @ wv.t()).to(x.dtype)
        held = _package().BlockFp8(state["codes"], state["scales"], state["K"])
        return _package().fp8_block_matmul(x, held)
    with torch.no_grad():
        if not own:
            for p, g, m in zip(state["params"], state["grads"], state["momenta"]):
                _plain_muon(p, g, m)
        else:
            _package().muon_step(state["params"], state["grads"], state["momenta"], lr=_LR,
                                 momentum=_MOMENTUM, weight_decay=_DECAY, update_rms=_RMS, steps=_STEPS)
    return {"p": state["p"], "m": state["m"]}


# ---- what a pass cannot do without ---------------------------------------------

def work(case):
    es = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "route":
        B, E, k = case["B"], case["E"], case["k"]
        # logits in and their gradient out; indices and weights out, the weights' gradient in
        return {"bytes": B * (2 * E * es + 16 * k) + 8 * E + (4 * E if case["bias"] else 0)
                + (B if case["padded"] else 0), "flops": 20 * B * E}
    if case["kind"] == "muon":
        n = flops = 0
        for s in _muon_shapes(case):
            batch, lo, hi = math.prod(s[:-2]), min(s[-2:]), max(s[-2:])
            n += batch * lo * hi
            # X X^T and A A are symmetric: half of each
            flops += batch * _STEPS * (3 * lo * lo * hi + lo * lo * lo)
        return {"bytes": n * (3 * es + 8), "flops": flops}
    M, K, N = case["M"], case["K"], case["N"]
    if case["kind"] == "held":
        return {"bytes": es * (M * K + M * N) + N * K + 4 * -(-N // _BLOCK) * -(-K // _BLOCK),
                "flops": 2 * M * K * N}
    return {"bytes": es * 2 * (M * K + K * N + M * N), "flops": 6 * M * K * N}


# ---- the same outputs in 64 bits -----------------------------------------------

def _exact_route(case, seed):
    s = _route_inputs(case, seed)
    B, E, k, G = case["B"], case["E"], case["k"], case["groups"]
    x = s["raw"].double()
    on = torch.ones(B, dtype=torch.bool, device="cuda") if s["mask"] is None else s["mask"]
    if case["score"] == "softmax":
        e = torch.exp(x - x.amax(-1, keepdim=True))
        p = e / e.sum(-1, keepdim=True)
    else:
        p = 1 / (1 + torch.exp(-x))
    left = p.clone() if s["bias"] is None else p + s["bias"].double()
    if s["bias"] is None and G == 1:
        left = x.clone()                 # both scores grow with the logit

    def take(v):
        """The first of the largest in each row, struck out for the next."""
        top = v.amax(-1, keepdim=True)
        first = torch.where(v == top, torch.arange(v.shape[1], device="cuda"), v.shape[1]).amin(-1)
        v[torch.arange(v.shape[0], device="cuda"), first] = -math.inf
        return top[:, 0], first
    if G > 1:
        per = left.reshape(B * G, E // G).clone()
        worth = take(per)[0]
        if E // G > 1:
            worth = worth + take(per)[0]
        worth, open_ = worth.view(B, G), torch.zeros(B, G, dtype=torch.bool, device="cuda")
        for _ in range(case["top_groups"]):
            open_[torch.arange(B, device="cuda"), take(worth)[1]] = True
        left[~open_.repeat_interleave(E // G, 1)] = -math.inf
    idx = torch.stack([take(left)[1] for _ in range(k)], 1)
    t = p.gather(1, idx)
    dw = s["dw"].double()
    if case["renorm"]:
        total = t.sum(-1, keepdim=True) + _RENORM_EPS
        w = t / total
        dt = (dw - (dw * w).sum(-1, keepdim=True)) / total
    else:
        w, dt = t, dw
    w, dt = w * _ROUTE_SCALE, dt * _ROUTE_SCALE
    full = torch.zeros_like(p).scatter_(1, idx, dt)
    if case["score"] == "softmax":
        d = p * full - p * (full * p).sum(-1, keepdim=True)
    else:
        d = full * p / (1 + torch.exp(x))
    cnt = torch.zeros_like(p).scatter_(1, idx, 1.0)[on].sum(0).to(torch.int64)
    return {"idx": torch.where(on[:, None], idx, -1), "w": w * on[:, None], "counts": cnt,
            "draw": torch.where(on[:, None], d, 0.0)}


def _to_e4m3(v):
    """v (64 bits) to the nearest e4m3 value, even ones on ties."""
    _, e = torch.frexp(v.abs())
    step = torch.ldexp(torch.ones_like(v), (e - 1).clamp(min=-6) - 3)
    return (torch.round(v / step) * step).clamp(-_E4M3_MAX, _E4M3_MAX)


def _exact_rounded(x, rows):
    """x (R, K) as its codes in blocks of rows x 128 stand for it: the scale and its inverse are
    32-bit numbers, and so is the product that is rounded."""
    R, K = x.shape
    x = x.double()
    out = torch.zeros(R + -R % rows, K + -K % _BLOCK, dtype=torch.float64, device="cuda")
    out[:R, :K] = x
    b = out.view(out.shape[0] // rows, rows, out.shape[1] // _BLOCK, _BLOCK)
    top = b.abs().amax(3, keepdim=True).amax(1, keepdim=True)
    some = top > _TINY
    safe = torch.where(some, top, 1.0)
    scale, inv = (safe / _E4M3_MAX).float().double(), (_E4M3_MAX / safe).float().double()
    v = _to_e4m3((b * inv).float().double()) * scale
    return torch.where(some, v, 0.0).view_as(out)[:R, :K]


def _exact_linear(case, seed):
    x, w, dy = _linear_inputs(case, seed)
    wv = _exact_rounded(w.t(), _BLOCK)
    y = _exact_rounded(x, 1).matmul(wv.t())
    if case["kind"] == "held":
        return y
    return {"y": y, "dx": _exact_rounded(dy, 1).matmul(wv),
            "dw": _exact_rounded(x.t(), 1).matmul(_exact_rounded(dy.t(), 1).t())}


def _exact_muon(case, seed):
    flat_p, flat_g, flat_m, shapes = _muon_inputs(case, seed)
    ps, ms = [], []
    a, b, c = _NS
    for p, g, m in zip(*(_views(t.double(), shapes) for t in (flat_p, flat_g, flat_m))):
        m = _MOMENTUM * m + g
        u = g + _MOMENTUM * m
        tall = u.shape[-2] > u.shape[-1]
        x = u.mT if tall else u
        x = x / (x.square().sum((-1, -2), keepdim=True).sqrt() + _NORM_EPS)
        for _ in range(_STEPS):
            s = x.matmul(x.mT)
            sx = s.matmul(x)
            x = a * x + b * sx + c * s.matmul(sx)
        x = x.mT if tall else x
        ms.append(m.reshape(-1))
        ps.append((p - _LR * (_DECAY * p + _RMS * max(p.shape[-2:]) ** 0.5 * x)).reshape(-1))
    return {"p": torch.cat(ps), "m": torch.cat(ms)}


def exact(case, seed):
    with torch.no_grad():
        f = {"route": _exact_route, "linear": _exact_linear, "held": _exact_linear,
             "muon": _exact_muon}[case["kind"]]
        return f(case, seed)
