"""AdamW over many tensors at once on MI355X (gfx950), with moments in 32 or in 8 bits.

The reference trains with torch's AdamW (pre-train/train.py:1263-1268):
    m = beta1 m + (1 - beta1) g;  v = beta2 v + (1 - beta2) g^2
    p = p (1 - lr wd) - lr / (1 - beta1^t) m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
Here a step is one launch for up to 56 tensors (tmoe_adamw_step): bfloat16 or float32
parameters on a HIP device with gradients of their dtype, computed in float32.

8-bit states hold m and sqrt(v) as OCP e4m3 codes (torch.float8_e4m3fn) with one float32
scale for each BLOCK elements of a tensor in its memory's order: value = code * scale.
Codes are rounded up or down at random (from seed, step, the tensor's place in the list and
the element's in the tensor), so that m and v are right in the mean; a moment that moves
by a thousandth a step would otherwise never leave its code. A gradient that is not finite, or
whose square is not in float32 (from 1.8e19 on), makes the moments of its whole block
non-finite.
"""
from __future__ import annotations

from typing import Sequence, Union

import torch

from . import _lib

BLOCK = 256
E4M3_MAX = 448.0


def _capturing(device: torch.device) -> bool:
    """Whether the current stream of a device records a graph."""
    if device.type != "cuda":
        return False
    if device.index == torch.cuda.current_device():
        return torch.cuda.is_current_stream_capturing()
    with torch.cuda.device(device):
        return torch.cuda.is_current_stream_capturing()


def _run(params, grads, m, v, ms, vs, step, lr, betas, eps, weight_decay, seed):
    if not 0.0 <= betas[0] < 1.0 or not 0.0 <= betas[1] < 1.0:
        raise ValueError(f"adamw_step: betas {betas}")
    if not lr >= 0.0 or not eps >= 0.0 or not weight_decay >= 0.0:
        raise ValueError(f"adamw_step: lr {lr}, eps {eps}, weight_decay {weight_decay}")
    dev = isinstance(step, torch.Tensor)
    _lib.native().adamw(params, grads, m, v, ms, vs, None if dev else int(step), step if dev else None,
                        float(lr), float(betas[0]), float(betas[1]), float(eps), float(weight_decay),
                        int(seed))


def adamw_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor],
               exp_avgs: Sequence[torch.Tensor], exp_avg_sqs: Sequence[torch.Tensor], *,
               step: Union[int, torch.Tensor], lr: float, betas=(0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 1e-2) -> None:
    """One step on lists of tensors of one dtype on one device, in place. The moments are
    float32, laid out as their parameters. step counts from 1: a number, or an int64 tensor
    of one value on the device, which is read when the kernels run. What is written may share
    no memory, nor may a gradient lie in what is written of another element."""
    _run(params, grads, exp_avgs, exp_avg_sqs, None, None, step, lr, betas, eps, weight_decay, 0)


def adamw_step_8bit(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor],
                    exp_avg_codes: Sequence[torch.Tensor], exp_avg_scales: Sequence[torch.Tensor],
                    exp_avg_sq_codes: Sequence[torch.Tensor],
                    exp_avg_sq_scales: Sequence[torch.Tensor], *, step: Union[int, torch.Tensor],
                    lr: float, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2,
                    seed: int = 0) -> None:
    """adamw_step with 8-bit moments: for a parameter of n elements n codes
    (torch.float8_e4m3fn or its uint8 bits) and ceil(n / BLOCK) scales of each moment, the
    second one's of sqrt(v)."""
    _run(params, grads, exp_avg_codes, exp_avg_sq_codes, exp_avg_scales, exp_avg_sq_scales, step, lr,
         betas, eps, weight_decay, seed)


def dequantize_state(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """The float32 values (n,) of a moment's codes and scales (of sqrt(v): square them)."""
    if codes.dtype == torch.uint8:
        codes = codes.view(torch.float8_e4m3fn)
    q = codes.reshape(-1).float()
    return q * scales.repeat_interleave(BLOCK)[:q.numel()]


class FusedAdamW(torch.optim.Optimizer):
    """AdamW whose step is one launch for up to 56 parameters of a group.

    state_bits 32 keeps float32 moments ("exp_avg", "exp_avg_sq"), 8 keeps codes and scales
    ("exp_avg_codes", "exp_avg_scales", "exp_avg_sq_codes", "exp_avg_sq_scales", of
    sqrt(v)). Parameters are bfloat16 or float32, dense, on HIP devices, with gradients of
    their dtype; bfloat16 ones are rounded to nearest.

    capturable=True holds the step counts on the device, so that a captured step counts on in
    its replays; without it a step inside a capture raises, and so does a parameter's first
    step, which makes its state. lr and the other numbers are those of the capture in each
    replay. Each parameter counts the steps that it took: those that step together share a
    count until a step that only some of them take, which is refused once a captured step
    advances that count."""

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, *, state_bits: int = 32, seed: int = 0,
                 capturable: bool = False):
        options = dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay,
                       state_bits=state_bits, seed=seed, capturable=capturable)
        self._check_options(options)
        self._captured = {}     # by id: the device counts that captured steps advance
        super().__init__(params, options)

    @staticmethod
    def _check_options(o) -> None:
        if not o["lr"] >= 0.0 or not o["eps"] >= 0.0 or not o["weight_decay"] >= 0.0:
            raise ValueError(f"FusedAdamW: lr {o['lr']}, eps {o['eps']}, weight_decay {o['weight_decay']}")
        if not 0.0 <= o["betas"][0] < 1.0 or not 0.0 <= o["betas"][1] < 1.0:
            raise ValueError(f"FusedAdamW: betas {o['betas']}")
        if o["state_bits"] not in (32, 8):
            raise ValueError(f"FusedAdamW: state_bits {o['state_bits']} is not 32 or 8")

    def add_param_group(self, param_group) -> None:
        self._check_options({**self.defaults, **param_group})
        super().add_param_group(param_group)

    def __setstate__(self, state) -> None:
        super().__setstate__(state)
        self._captured = {}

    def _init_state(self, p: torch.Tensor, group, count) -> dict:
        st = self.state[p]
        st["step"] = count
        if group["state_bits"] == 32:
            for k in ("exp_avg", "exp_avg_sq"):
                st[k] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format)
        else:
            for k in ("exp_avg", "exp_avg_sq"):
                st[k + "_codes"] = torch.zeros(p.numel(), dtype=torch.uint8,
                                               device=p.device).view(torch.float8_e4m3fn)
                st[k + "_scales"] = torch.zeros(-(-p.numel() // BLOCK), device=p.device)
        return st

    @torch.no_grad()
    def step(self, closure=None):
        """One step over every parameter that has a gradient; closure as in torch.optim."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        # what is refused is refused before anything changes
        work, captured = [], {}
        for group in self.param_groups:
            live, resting = [], []      # (parameter, gradient, device, state or None); parameters
            for p in group["params"]:
                g = p.grad
                if g is None:
                    resting.append(p)
                    continue
                if g.is_sparse:
                    raise RuntimeError("FusedAdamW: sparse gradients are not supported")
                live.append((p, g, p.device, self.state.get(p)))
            work.append((group, live, self._check_step(group, live, resting, captured)))
        self._captured.update(captured)
        for group, live, parted in work:
            on_device = group["capturable"]
            fresh = {}      # device: the count that parameters first met in this step share
            runs = {}       # (device, dtype, step): its parameters, one call each
            for p, g, dev, st in live:
                if not st:
                    if on_device and dev not in fresh:
                        fresh[dev] = torch.zeros((), dtype=torch.int64, device=dev)
                    st = self._init_state(p, group, fresh[dev] if on_device else 0)
                n = st["step"]
                if parted and id(n) in parted:      # those that step now count by themselves from here on
                    if parted[id(n)] is None:
                        parted[id(n)] = n.clone()
                    n = st["step"] = parted[id(n)]
                key = (dev, p.dtype, id(n) if on_device else n)
                run = runs.get(key)
                if run is None:
                    run = runs[key] = (n, [], [], [])
                run[1].append(p)
                run[2].append(g)
                run[3].append(st)
            counted = set()
            for n, ps, gs, sts in runs.values():
                first = on_device and id(n) not in counted
                if first:
                    counted.add(id(n))
                    n.add_(1)
                try:
                    self._run(group, n if on_device else n + 1, ps, gs, sts)
                except Exception:
                    if first:       # nothing was launched that this counts
                        n.sub_(1)
                    raise
                if not on_device:
                    for st in sts:
                        st["step"] = n + 1
        return loss

    def _check_step(self, group, live, resting, captured) -> dict:
        """Refuses what a step of a group cannot do; adds the device counts that it advances in a
        capture to `captured`, by id. {id: None} of the device counts of live parameters that
        resting ones hold too."""
        capturing = {d: _capturing(d) for d in {d for _, _, d, _ in live}}
        if not group["capturable"]:
            if True in capturing.values():
                raise RuntimeError("FusedAdamW: a step inside a graph capture needs "
                                   "capturable=True (its count would stand still)")
            return {}
        parted = {}
        if resting:
            mine = {id(st["step"]) for _, _, _, st in live if st}
            parted = {id(st["step"]): None for st in map(self.state.get, resting)
                      if st and id(st["step"]) in mine}
        if not parted and True not in capturing.values():
            return parted
        for p, _, dev, st in live:
            if not st:
                if capturing[dev]:      # each replay would clear it again
                    raise RuntimeError("FusedAdamW: a parameter's first step inside a graph capture: make "
                                       "one step with these gradients before the capture")
                continue
            n = st["step"]
            if id(n) not in parted:
                if capturing[dev]:
                    captured[id(n)] = n
            elif capturing[dev]:
                raise RuntimeError("FusedAdamW: a captured step of some of the parameters that have stepped "
                                   "together so far: make one step with these gradients before the capture")
            elif id(n) in self._captured:       # the graph counts for all of them
                raise RuntimeError("FusedAdamW: parameters whose step was captured together step together "
                                   "(where that graph is gone, opt.load_state_dict(opt.state_dict()) parts "
                                   "them)")
        return parted

    @staticmethod
    def _run(group, step, ps, gs, sts):
        def state(k):
            return [st[k] for st in sts]
        eight = group["state_bits"] == 8
        m, v = ("exp_avg_codes", "exp_avg_sq_codes") if eight else ("exp_avg", "exp_avg_sq")
        _run(ps, gs, state(m), state(v), state("exp_avg_scales") if eight else None,
             state("exp_avg_sq_scales") if eight else None, step, group["lr"], group["betas"],
             group["eps"], group["weight_decay"], group["seed"])

    def load_state_dict(self, state_dict) -> None:
        """As torch.optim's, but 8-bit states keep their dtypes and 32-bit moments are float32
        in their parameter's layout (torch casts states to their parameter's dtype). A
        torch.optim.AdamW's state is taken as 32-bit moments; what it lacks of this class's
        options stays as it is here. States of other kinds, and amsgrad's, maximize's or an L2
        decay's, are refused. 8-bit states lie in their parameter's order in memory: they are
        for parameters of the same strides."""
        saved, groups = state_dict["state"], state_dict["param_groups"]
        if len(groups) == len(self.param_groups):       # (torch refuses it otherwise)
            groups = [{**{k: mine[k] for k in self.defaults if k in mine}, **its}
                      for mine, its in zip(self.param_groups, groups)]
            for mine, its in zip(self.param_groups, groups):
                self._check_load(mine, its, saved)
        super().load_state_dict({**state_dict, "param_groups": groups})
        for mine, its in zip(self.param_groups, groups):
            counts = {}
            for p, i in zip(mine["params"], its["params"]):
                if i not in saved:
                    continue
                st = self.state[p] = {}
                for k, v in saved[i].items():
                    if k in ("exp_avg", "exp_avg_sq"):
                        st[k] = torch.empty_like(p, dtype=torch.float32, requires_grad=False,
                                                 memory_format=torch.preserve_format).copy_(v.detach())
                    elif isinstance(v, torch.Tensor):
                        st[k] = v.detach().to(p.device, copy=True)
                    else:
                        st[k] = v
                n = int(st["step"])
                if mine["capturable"]:
                    if (p.device, n) not in counts:
                        counts[p.device, n] = torch.full((), n, dtype=torch.int64, device=p.device)
                    st["step"] = counts[p.device, n]
                else:
                    st["step"] = n

    @staticmethod
    def _check_load(mine, its, saved) -> None:
        for k in ("amsgrad", "maximize"):
            if its.get(k):
                raise ValueError(f"FusedAdamW: a state of an optimizer with {k}")
        FusedAdamW._check_options(its)
        if its["weight_decay"] and not its.get("decoupled_weight_decay", True):
            raise ValueError("FusedAdamW: a state of an optimizer with an L2 decay")
        eight = its["state_bits"] == 8
        needed = {"step"} | {m + s for m in ("exp_avg", "exp_avg_sq")
                             for s in (("_codes", "_scales") if eight else ("",))}
        for p, i in zip(mine["params"], its["params"]):
            st = saved.get(i)
            if not st:
                continue
            if not needed <= set(st):
                raise ValueError(f"FusedAdamW: a state of {sorted(st)} for state_bits {its['state_bits']}")
            for k in needed - {"step"}:
                want = p.shape if not eight else \
                    (p.numel() if k.endswith("_codes") else -(-p.numel() // BLOCK),)
                if st[k].shape != want:
                    raise ValueError(f"FusedAdamW: {k} {tuple(st[k].shape)} for a parameter {tuple(p.shape)}")
