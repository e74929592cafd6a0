"""Performance cases of the training step's operators around the expert contraction.

  route   fused_router: capped router, top-k, balance and z losses and per-expert counts
          of a batch of tokens, and the gradient of its logits
  norm    fused_block_norm: gate, norm after a block, residual with its scale, norm
          before the next block, and the gradients of all of them
  adamw   adamw_step / adamw_step_8bit: one AdamW step over all tensors of a model

prepare() makes a case's inputs on the GPU from its seed, run() makes one pass: with
`own` false in elementary torch operations in 32 bits, with `own` true through this
framework's entry points. exact() gives the same outputs in 64 bits. Sizes are those of
the workloads C1..C5, F1 / F2 and the reference model's layers, or generic.
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
_CAP = 10.0            # the router's cap
_EPS = 1e-5            # of the norms
_BETA1, _BETA2, _ADAM_EPS, _DECAY, _LR = 0.9, 0.95, 1e-8, 0.1, 3e-4
_BLOCK = 256           # elements that share a scale in 8-bit states
_E4M3_MAX = 448.0


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

def _route(B, E, k, dtype="fp32", tau=0.5, padded=0.0):
    return dict(kind="route", B=B, E=E, k=k, dtype=dtype, tau=tau, padded=padded)


def _norm(T, d, dtype="bf16", residual=True, gate=False, post=False, gamma=True, nxt=True):
    return dict(kind="norm", T=T, d=d, dtype=dtype, residual=residual, gate=gate, post=post,
                gamma=gamma, next=nxt)


def _adamw(model, layers=1, bits=32, dtype="fp32"):
    return dict(kind="adamw", model=model, layers=layers, bits=bits, dtype=dtype)


def listed():
    return [
        # one token's routing in an online update: launch and host latency
        dict(_route(1, 8, 2), name="route_B1_E8"),
        # the training layer's batch (the contraction's own case), early in the schedule
        dict(_route(16384, 8, 2, tau=2.0), name="route_B16384_E8"),
        # a wide router's top-8 under autocast (C4)
        dict(_route(4096, 256, 8, "bf16"), name="route_B4096_E256"),
        # a large batch of padded sequences: three tokens in ten are padding
        dict(_route(131072, 64, 6, tau=1.25, padded=0.3), name="route_B131072_E64_padded"),
        # one token through a sub-block's end: residual scale and the next block's norm
        dict(_norm(1, 768), name="norm_T1_d768"),
        # the transformer block's FFN output on a training batch
        dict(_norm(16384, 768), name="norm_T16384_d768"),
        # the Mamba block's gated norm on a ragged batch, y and gate halves of one projection
        dict(_norm(5003, 1536, "fp32", residual=False, gate=True, post=True, gamma=False, nxt=False),
             name="norm_gated_T5003_d1536"),
        # rows of an odd width: no row but the first is aligned
        dict(_norm(2049, 1001, "fp32"), name="norm_T2049_d1001"),
        # norms on both sides of a gated block, all operands (C3's output width)
        dict(_norm(16384, 2304, gate=True, post=True), name="norm_sandwich_T16384_d2304"),
        # the seven tensors of one small layer (C1): latency
        dict(_adamw("c1"), name="adamw_c1_32bit"),
        # the FFN sub-block in bf16 with 8-bit states
        dict(_adamw("ffn", bits=8, dtype="bf16"), name="adamw_ffn_8bit"),
        # all 66 layers of the reference model
        dict(_adamw("reference", layers=66), name="adamw_reference_32bit"),
    ]


def _log_int(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["route", "norm", "norm", "adamw"])
    if kind == "route":
        E = _log_int(rng, 2, 256)
        return _route(_log_int(rng, 1, min(262144, 2 ** 23 // E)), E, rng.randint(1, min(E, 8)),
                      rng.choice(["fp32", "bf16"]), rng.uniform(0.5, 2.0),
                      rng.choice([0.0, 0.0, rng.uniform(0.0, 0.9)]))
    if kind == "norm":
        d = rng.choice([_log_int(rng, 33, 6144), 64 * _log_int(rng, 1, 96)])
        gamma, residual = rng.random() < 0.7, rng.random() < 0.8
        return _norm(_log_int(rng, 1, min(65536, 2 ** 25 // d)), d, rng.choice(["bf16", "bf16", "fp32"]),
                     residual, rng.random() < 0.4, rng.random() < 0.4, gamma,
                     rng.random() < 0.7 or not residual)
    return _adamw(rng.choice(["c1", "c3", "ffn", "odd"]), rng.randint(1, 24), rng.choice([32, 8]),
                  rng.choice(["fp32", "bf16"]))


# ---- inputs --------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, shape, std=1.0):
    return torch.randn(shape, generator=g, device="cuda") * std


def _route_inputs(case, seed):
    g, dt = _gen(seed), _DT[case["dtype"]]
    B, E, k = case["B"], case["E"], case["k"]
    # logits of a trained router: some experts likelier than others, a few tokens far into the cap
    raw = (_normal(g, (B, E), 2.0) + _normal(g, (E,)) + _normal(g, (B, 1), 3.0)).to(dt)
    mask = None
    if case["padded"]:
        mask = torch.rand(B, generator=g, device="cuda") >= case["padded"]
    return {"raw": raw, "mask": mask, "dw": _normal(g, (B, k)), "dlb": _normal(g, (), 0.01).abs(),
            "dz": _normal(g, (), 0.001).abs()}


def _norm_inputs(case, seed):
    g, dt = _gen(seed), _DT[case["dtype"]]
    T, d = case["T"], case["d"]
    n = {}
    if case["residual"]:
        # a residual stream: a few channels much larger than the others
        wide = 1 + 20 * (torch.rand(d, generator=g, device="cuda") < 0.01)
        n["x"] = (_normal(g, (T, d), 2.0) * wide).to(dt)
    if case["gate"]:
        both = _normal(g, (T, 2 * d)).to(dt)         # one projection's two halves
        n["y"], n["gate"] = both[:, :d], both[:, d:]
    else:
        n["y"] = _normal(g, (T, d)).to(dt)
    if case["post"]:
        n["post_weight"] = (1 + _normal(g, (d,), 0.1)).to(dt)
    if case["gamma"]:
        n["gamma"] = (0.5 + _normal(g, (d,), 0.1)).to(dt)
    if case["next"]:
        n["next_weight"] = (1 + _normal(g, (d,), 0.1)).to(dt)
    return n, _normal(g, (T, d)).to(dt), _normal(g, (T, d)).to(dt) if case["next"] else None


def _layer_shapes(d_in, d_out, E, r1, r2, r3):
    """A training layer's parameters: router, U_expert, U_in, U_out, core, bias, norm."""
    return [(E, d_in), (E, r1), (d_in, r3), (r2, d_out), (r1, r3, r2), (d_out,), (r3,)]


def _tensor_sizes(case):
    ref = (8, 32, 512, 256)
    up, out = _layer_shapes(1536, 6144, *ref), _layer_shapes(768, 768, *ref)
    wide, down = _layer_shapes(768, 4608, *ref), _layer_shapes(4608, 768, *ref)
    shapes = {"c1": _layer_shapes(512, 1024, 8, 4, 256, 128),
              "c3": _layer_shapes(1536, 2304, 16, 4, 1024, 256),
              "odd": [(1,), (7,), (257, 3), (255,), (511, 129), (33, 65, 17)],
              "ffn": wide + wide + down,
              "reference": 24 * (up + out) + 6 * (wide + wide + down)}[case["model"]]
    if case["model"] != "reference":
        shapes = shapes * case["layers"]
    return [math.prod(s) for s in shapes]


def _offsets(sizes):
    """Where each tensor begins in one buffer whose tensors begin on whole blocks; its length."""
    at, offs = 0, []
    for n in sizes:
        offs.append(at)
        at += -(-n // _BLOCK) * _BLOCK
    return offs, at


def _quantised(v):
    """(e4m3 codes, one scale a block) of non-negative or signed values, to nearest."""
    b = v.view(-1, _BLOCK)
    s = b.abs().amax(1) / _E4M3_MAX
    q = (b / torch.where(s > 0, s, 1.0)[:, None]).clamp(-_E4M3_MAX, _E4M3_MAX)
    return q.to(torch.float8_e4m3fn).view(-1), s


def _adamw_inputs(case, seed):
    g, dt = _gen(seed), _DT[case["dtype"]]
    sizes = _tensor_sizes(case)
    offs, n = _offsets(sizes)
    # gradients of a few sizes along the buffer, the moments of earlier steps about them
    size = 1e-3 * torch.exp(_normal(g, (n // _BLOCK, 1)))
    keep = torch.ones(n, device="cuda")    # what fills a tensor's last block stays zero
    for o, m in zip(offs, sizes):
        keep[o + m:o + -(-m // _BLOCK) * _BLOCK] = 0
    size = size * keep.view(-1, _BLOCK)
    p = _normal(g, (n,), 0.03) * keep
    del keep
    grad = (_normal(g, (n // _BLOCK, _BLOCK)) * size).view(-1).to(dt)
    m = (_normal(g, (n // _BLOCK, _BLOCK)) * size * 0.3).view(-1)
    v = ((0.5 + torch.rand((n // _BLOCK, _BLOCK), generator=g, device="cuda")) * size * size).view(-1)
    return {"p": p.to(dt), "g": grad, "m": m, "v": v, "sizes": sizes, "offs": offs}


def _views(flat, offs, sizes):
    return [flat[o:o + n] for o, n in zip(offs, sizes)]


def prepare(case, seed):
    if case["kind"] == "route":
        s = _route_inputs(case, seed)
        s["raw"].requires_grad_()
        return dict(s, kind="route", k=case["k"], tau=case["tau"])
    if case["kind"] == "norm":
        n, dr, dh = _norm_inputs(case, seed)
        return {"kind": "norm", "in": {k: v.detach().requires_grad_() for k, v in n.items()},
                "dr": dr, "dh": dh}
    s = _adamw_inputs(case, seed)
    offs, sizes = s["offs"], s["sizes"]
    st = {"kind": "adamw", "bits": case["bits"], "step": 100, "seed": 20 + seed, "p": s["p"], "g": s["g"]}
    st["params"], st["grads"] = _views(s["p"], offs, sizes), _views(s["g"], offs, sizes)
    if case["bits"] == 32:
        st["m"], st["v"] = s["m"], s["v"]
        st["ms"], st["vs"] = _views(s["m"], offs, sizes), _views(s["v"], offs, sizes)
        return st
    st["mq"], st["mscale"] = _quantised(s["m"])
    st["rq"], st["rscale"] = _quantised(s["v"].sqrt())
    soffs, ssizes = [o // _BLOCK for o in offs], [-(-n // _BLOCK) for n in sizes]
    st["mqs"], st["mscales"] = _views(st["mq"], offs, sizes), _views(st["mscale"], soffs, ssizes)
    st["rqs"], st["rscales"] = _views(st["rq"], offs, sizes), _views(st["rscale"], soffs, ssizes)
    # each element's number among its tensor's, with the tensor's own mixed in: what its random bits go by
    key = torch.empty(st["p"].numel(), dtype=torch.int64, device="cuda")
    for i, (o, n) in enumerate(zip(offs, sizes)):
        m = -(-n // _BLOCK) * _BLOCK
        key[o:o + m] = (torch.arange(m, device="cuda") + i * 0x9E3779B9) & 0xFFFFFFFF
    st["key"] = key
    return st


# ---- a pass --------------------------------------------------------------------

def _plain_router(raw, k, tau, mask):
    E = raw.shape[1]
    a = raw.float()
    if mask is not None:
        a = torch.where(mask[:, None], a, 0.0)
    order = torch.sort(a.detach(), dim=-1, descending=True, stable=True).indices[:, :k]
    cap = _CAP * torch.tanh(a / _CAP)
    lse = cap.logsumexp(-1)
    probs = torch.softmax(cap / tau, -1)
    top = probs.gather(-1, order)
    w = top / (top.sum(-1, keepdim=True) + 1e-6)
    keep = torch.ones_like(lse) if mask is None else mask.float()
    n = keep.sum().clamp(min=1.0)
    counts = torch.zeros(E, device=a.device, dtype=torch.int64)
    counts = counts.index_add(0, order.reshape(-1), keep.to(torch.int64).repeat_interleave(k))
    lb = E * ((counts.float() / n) * ((probs * keep[:, None]).sum(0) / n)).sum()
    z = (lse * lse * keep).sum() / n
    if mask is not None:
        w = torch.where(mask[:, None], w, 0.0)
        order = torch.where(mask[:, None], order, -1)
    return order, w, lb, z, counts


def _plain_norm(x=None, y=None, gate=None, post_weight=None, gamma=None, next_weight=None):
    dt = y.dtype
    u = y.float()
    if gate is not None:
        g = gate.float()
        u = u * (g * torch.sigmoid(g))
    if post_weight is not None:
        u = u / torch.sqrt((u * u).mean(-1, keepdim=True) + _EPS) * post_weight.float()
    if gamma is not None:
        u = gamma.float() * u
    r = u if x is None else x.float() + u
    h = None
    if next_weight is not None:
        h = (r / torch.sqrt((r * r).mean(-1, keepdim=True) + _EPS) * next_weight.float()).to(dt)
    return r.to(dt), h


def _corrections(step):
    return 1.0 - _BETA1 ** step, math.sqrt(1.0 - _BETA2 ** step)


def _moments(m, v, g):
    return m * _BETA1 + g * (1.0 - _BETA1), v * _BETA2 + g * g * (1.0 - _BETA2)


def _updated(p, m, v, step):
    c1, c2 = _corrections(step)
    return p * (1.0 - _LR * _DECAY) - (m / (torch.sqrt(v) / c2 + _ADAM_EPS)) * (_LR / c1)


def _mix(h):
    """32 bits in 64, every bit of the input in every bit of the output."""
    h = ((h ^ (h >> 16)) * 0x85EBCA6B) & 0xFFFFFFFF
    h = ((h ^ (h >> 13)) * 0xC2B2AE35) & 0xFFFFFFFF
    return h ^ (h >> 16)


def _grid(a):
    """(code, value, step to the next) of the largest e4m3 value that is no larger than a."""
    e = ((a.view(torch.int32) >> 23) - 127).clamp(min=-6)
    step = ((e + 124) << 23).view(torch.float32)
    q = torch.floor(a / step)
    return q.to(torch.int32) + ((e + 6) << 3), q * step, step


def _encode(v, root, u):
    """(e4m3 codes, scales) of v (signed), or of the roots of v where `root`, rounded up where
    the chance to (unbiased in v) is more than u."""
    b = (torch.sqrt(v) if root else v.abs()).view(-1, _BLOCK)
    s = b.amax(1) / _E4M3_MAX
    a = (b / torch.where(s > 0, s, 1.0)[:, None]).clamp(max=_E4M3_MAX).view(-1)
    code, lo, step = _grid(a)
    chance = (a - lo) / step
    if root:
        chance = chance * ((a + lo) / (lo + lo + step))
    code = code + (u < chance)
    if root:
        code = torch.where((code == 0) & (a > 0), 1, code)
    else:
        code = torch.where(v < 0, code + 128, code)
    return code.to(torch.uint8).view(torch.float8_e4m3fn), s


def _decode(q, s):
    return (q.float().view(-1, _BLOCK) * s[:, None]).view(-1)


def _random(key, seed, step):
    """Two uniform numbers in (0, 1) for each key, of 16 bits each."""
    h = _mix(key ^ _mix((seed + step * 0x9E3779B1) & 0xFFFFFFFF))
    return ((h >> 16).float() + 0.5) / 65536.0, ((h & 0xFFFF).float() + 0.5) / 65536.0


def _plain_adamw(st):
    step = st["step"]
    g, p = st["g"].float(), st["p"].float()
    if st["bits"] == 32:
        m, v = _moments(st["m"], st["v"], g)
        st["p"].copy_(_updated(p, m, v, step))
        st["m"].copy_(m)
        st["v"].copy_(v)
        return
    r = _decode(st["rq"], st["rscale"])
    m, v = _moments(_decode(st["mq"], st["mscale"]), r * r, g)
    um, uv = _random(st["key"], st["seed"], step)
    st["p"].copy_(_updated(p, m, v, step))
    for q, s, new in (("mq", "mscale", _encode(m, False, um)), ("rq", "rscale", _encode(v, True, uv))):
        st[q].view(torch.uint8).copy_(new[0].view(torch.uint8))
        st[s].copy_(new[1])


def run(state):
    if state["kind"] == "route":
        raw, mask = state["raw"], state["mask"]
        if own:
            idx, w, lb, z, counts = _package().fused_router(raw, state["k"], state["tau"], mask=mask)
        else:
            idx, w, lb, z, counts = _plain_router(raw, state["k"], state["tau"], mask)
        draw_, = torch.autograd.grad((w, lb, z), raw, (state["dw"], state["dlb"], state["dz"]))
        return {"idx": idx, "w": w.detach(), "lb": lb.detach(), "z": z.detach(), "counts": counts,
                "draw": draw_}
    if state["kind"] == "norm":
        n, dh = state["in"], state["dh"]
        if own:
            r, h = _package().fused_block_norm(**n, eps=_EPS)
        else:
            r, h = _plain_norm(**n)
        outs, seeds = ((r,), (state["dr"],)) if dh is None else ((r, h), (state["dr"], dh))
        grads = torch.autograd.grad(outs, list(n.values()), seeds)
        got = dict(zip(("d" + k for k in n), grads))
        got.update(r=r.detach())
        if h is not None:
            got.update(h=h.detach())
        return got
    state["step"] += 1
    with torch.no_grad():
        if not own:
            _plain_adamw(state)
        elif state["bits"] == 32:
            _package().adamw_step(state["params"], state["grads"], state["ms"], state["vs"],
                                  step=state["step"], lr=_LR, betas=(_BETA1, _BETA2), eps=_ADAM_EPS,
                                  weight_decay=_DECAY)
        else:
            _package().adamw_step_8bit(state["params"], state["grads"], state["mqs"], state["mscales"],
                                       state["rqs"], state["rscales"], step=state["step"], lr=_LR,
                                       betas=(_BETA1, _BETA2), eps=_ADAM_EPS, weight_decay=_DECAY,
                                       seed=state["seed"])
    names = ("p", "m", "v") if state["bits"] == 32 else ("p", "mq", "mscale", "rq", "rscale")
    return {n: state[n] for n in names}


# ---- what a pass cannot do without ---------------------------------------------

def work(case):
    es = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "route":
        B, E, k = case["B"], case["E"], case["k"]
        # logits in and their gradient out; indices and weights out, the weights' gradient in
        return {"bytes": B * (2 * E * es + 16 * k) + 8 * E + 16 + (B if case["padded"] else 0),
                "flops": 30 * B * E}
    if case["kind"] == "norm":
        T, d = case["T"], case["d"]
        acts = 1 + case["residual"] + case["gate"]             # in; their gradients out
        outs = 1 + case["next"]                                # out; their gradients in
        rows = case["post"] + case["gamma"] + case["next"]     # weights in, their gradients out
        return {"bytes": es * (2 * (acts + outs) * T * d + 2 * rows * d), "flops": 40 * T * d}
    n = sum(_tensor_sizes(case))
    state = 16 if case["bits"] == 32 else 4 + 16 / _BLOCK
    return {"bytes": n * (3 * es + state), "flops": 15 * n}


# ---- the same outputs in 64 bits -----------------------------------------------

def _exact_route(case, seed):
    s = _route_inputs(case, seed)
    B, E, k, tau = case["B"], case["E"], case["k"], case["tau"]
    raw = s["raw"].double()
    on = torch.ones(B, dtype=torch.bool, device="cuda") if s["mask"] is None else s["mask"]
    # an expert's rank: how many are larger, or as large and come first
    idx = torch.empty(B, k, dtype=torch.int64, device="cuda")
    left = raw.clone()
    for j in range(k):
        top = left.amax(-1, keepdim=True)
        first = torch.where(left == top, torch.arange(E, device="cuda"), E).amin(-1)
        idx[:, j] = first
        left[torch.arange(B, device="cuda"), first] = -math.inf
    th = torch.tanh(raw / _CAP)
    a = _CAP * th
    ez = torch.exp(a - _CAP)
    lse = _CAP + torch.log(ez.sum(-1))
    soft = ez / ez.sum(-1, keepdim=True)
    ep = torch.exp((a - _CAP) / tau)
    P = ep / ep.sum(-1, keepdim=True)
    sel = torch.zeros(B, E, dtype=torch.float64, device="cuda").scatter_(1, idx, 1.0) * on[:, None]
    N = max(1, int(on.sum()))
    cnt = sel.sum(0)
    lb = E * (cnt / N * (P[on].sum(0) / N)).sum()
    z = (lse[on] ** 2).sum() / N
    pk = P.gather(1, idx)
    tot = pk.sum(-1, keepdim=True) + 1e-6
    w = pk / tot
    dw, dlb, dz = s["dw"].double(), s["dlb"].double(), s["dz"].double()
    g = (dlb * E / N / N) * cnt[None, :].expand(B, E).clone()
    g = g.scatter_add(1, idx, (dw - (dw * w).sum(-1, keepdim=True)) / tot)
    da = P * (g - (P * g).sum(-1, keepdim=True)) / tau + dz * 2 / N * lse[:, None] * soft
    draw_ = da * (1 - th * th) * on[:, None]
    return {"idx": torch.where(on[:, None], idx, -1), "w": w * on[:, None], "lb": lb, "z": z,
            "counts": cnt.to(torch.int64), "draw": draw_}


def _exact_norm(case, seed):
    n, dr, dh = _norm_inputs(case, seed)
    n = {k: v.double() for k, v in n.items()}
    y, out = n["y"], {}
    sg = torch.sigmoid(n["gate"]) if "gate" in n else None
    u = y if sg is None else y * n["gate"] * sg
    f, iu = u, None
    if "post_weight" in n:
        iu = (u.square().mean(-1, keepdim=True) + _EPS).rsqrt()
        f = u * iu * n["post_weight"]
    r = n["gamma"] * f if "gamma" in n else f
    r = r + n["x"] if "x" in n else r
    D = dr.double()
    out["r"] = r
    if "next_weight" in n:
        ir = (r.square().mean(-1, keepdim=True) + _EPS).rsqrt()
        nr, dhd = r * ir, dh.double()
        out["h"] = nr * n["next_weight"]
        out["dnext_weight"] = (dhd * nr).sum(0)
        q = dhd * n["next_weight"]
        D = D + ir * (q - nr * (q * nr).mean(-1, keepdim=True))
    if "x" in n:
        out["dx"] = D
    df = D
    if "gamma" in n:
        out["dgamma"] = (D * f).sum(0)
        df = D * n["gamma"]
    if iu is not None:
        nu = u * iu
        out["dpost_weight"] = (df * nu).sum(0)
        q = df * n["post_weight"]
        df = iu * (q - nu * (q * nu).mean(-1, keepdim=True))
    if sg is not None:
        gt = n["gate"]
        out["dgate"] = df * y * sg * (1 + gt * (1 - sg))
        df = df * gt * sg
    out["dy"] = df
    return out


def _exact_adamw(case, seed):
    st = prepare(case, seed)
    step = st["step"] + 1
    bits8 = case["bits"] == 8
    c1, c2 = 1 - _BETA1 ** step, 1 - _BETA2 ** step
    g = st["g"].double()
    if bits8:
        m = (st["mq"].double().view(-1, _BLOCK) * st["mscale"].double()[:, None]).view(-1)
        v = (st["rq"].double().view(-1, _BLOCK) * st["rscale"].double()[:, None]).view(-1) ** 2
    else:
        m, v = st["m"].double(), st["v"].double()
    m = m + (1 - _BETA1) * (g - m)
    v = v + (1 - _BETA2) * (g.square() - v)
    p = st["p"].double()
    p = p - _LR * _DECAY * p - _LR * (m / c1) / ((v / c2).sqrt() + _ADAM_EPS)
    if not bits8:
        return {"p": p, "m": m, "v": v}
    # the states that come of random rounding: their scales alone have a value of their own
    out = {"p": p, "mq": None, "rq": None}
    for name, t in (("mscale", m.abs()), ("rscale", v.sqrt())):
        out[name] = t.view(-1, _BLOCK).amax(1) / _E4M3_MAX
    return out


def exact(case, seed):
    with torch.no_grad():
        return {"route": _exact_route, "norm": _exact_norm, "adamw": _exact_adamw}[case["kind"]](case, seed)
