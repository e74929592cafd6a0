"""Muon on MI355X (gfx950): momentum whose update is orthogonalised by Newton-Schulz products,
over many matrices at once.

The reference trains with AdamW (adamw.py). For the matrices of its layers (U_in, U_out, the
core's (r3, r2) slices) this is the other step in use:
    m = momentum m + g;  u = g + momentum m (nesterov) or m
    X = u / (|u| + eps), and `steps` times X = a X + (b A + c A A) X with A = X X^T
    p = p (1 - lr wd) - lr update_rms sqrt(max(rows, cols)) X
X's singular values end near one, so that its root mean square is about 1 / sqrt(max(rows, cols))
and the update's is lr update_rms: with update_rms 0.2 that of an AdamW step of the same lr.

A step is one launch for each product of all tensors (tmoe_muon_step), and two before them:
bfloat16 or float32 parameters (..., rows, cols) on a HIP device, each of whose last two axes is a
matrix; float32 momenta, sums in float32 (|u|'s in float64), X held in 22 bits.
"""
from __future__ import annotations

from typing import List, Sequence, Union

import torch

from . import _lib
from .adamw import _capturing

COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def _coefficients(c):
    c = tuple(float(v) for v in c)
    if len(c) != 3:
        raise ValueError(f"muon: coefficients {c}: three expected")
    return c


def _check_numbers(who: str, o) -> None:
    if not 0.0 <= o["momentum"] < 1.0:
        raise ValueError(f"{who}: momentum {o['momentum']}")
    if not o["lr"] >= 0.0 or not o["weight_decay"] >= 0.0 or not o["update_rms"] >= 0.0 or not o["eps"] > 0.0:
        raise ValueError(f"{who}: lr {o['lr']}, weight_decay {o['weight_decay']}, update_rms "
                         f"{o['update_rms']}, eps {o['eps']}")


def _step(params, grads, momenta, o, check: bool = False) -> None:
    """muon_step with the options o, or (check) its refusals alone."""
    _lib.native().muon(params, grads, momenta, float(o["lr"]), float(o["momentum"]), float(o["weight_decay"]),
                       float(o["update_rms"]), float(o["eps"]), _coefficients(o["coefficients"]),
                       int(o["steps"]), bool(o["nesterov"]), False, check)


def muon_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor],
              momenta: Sequence[torch.Tensor], *, lr: float, momentum: float = 0.95,
              nesterov: bool = True, weight_decay: float = 0.1, update_rms: float = 0.2, steps: int = 5,
              coefficients=COEFFICIENTS, eps: float = 1e-7) -> None:
    """One step on lists of tensors of one dtype on one device, in place. Parameters and momenta
    (float32) are contiguous. What is written may share no memory, nor with a gradient. The
    coefficients have to keep singular values within [-2, 2]."""
    o = dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, update_rms=update_rms,
             steps=steps, coefficients=coefficients, eps=eps)
    _check_numbers("muon_step", o)
    _step(params, grads, momenta, o)


def orthogonalize(matrices: Union[torch.Tensor, Sequence[torch.Tensor]], steps: int = 5,
                  coefficients=COEFFICIENTS, eps: float = 1e-7) -> Union[torch.Tensor, List[torch.Tensor]]:
    """X of each matrix (..., rows, cols) after `steps`, in its dtype; a list for a list. No
    gradient."""
    one = isinstance(matrices, torch.Tensor)
    if not eps > 0.0:
        raise ValueError(f"orthogonalize: eps {eps}")
    out = _lib.native().muon(None, [matrices] if one else matrices, None, 0.0, 0.0, 0.0, 0.0, float(eps),
                             _coefficients(coefficients), int(steps), False, True, False)
    return out[0] if one else out


class FusedMuon(torch.optim.Optimizer):
    """Muon over parameters of two axes or more, each of whose last two is a matrix: dense,
    contiguous, bfloat16 or float32, on HIP devices, with gradients of their dtype. Vectors, and
    what is better left to it (embeddings, routers), go to a FusedAdamW beside it.

    The state is a float32 momentum of each parameter. It can be captured into a graph once each
    parameter has stepped; lr and the other numbers are those of the capture in each replay."""

    def __init__(self, params, lr: float = 2e-2, momentum: float = 0.95, *, nesterov: bool = True,
                 weight_decay: float = 0.1, update_rms: float = 0.2, steps: int = 5,
                 coefficients=COEFFICIENTS, eps: float = 1e-7):
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay,
                                      update_rms=update_rms, steps=steps,
                                      coefficients=_coefficients(coefficients), eps=eps))

    @staticmethod
    def _check_options(o) -> None:
        _check_numbers("FusedMuon", o)
        if not 1 <= o["steps"] <= 16:
            raise ValueError(f"FusedMuon: steps {o['steps']} (1 to 16)")
        try:
            _step([], [], [], o, True)      # whether the coefficients stay in range
        except RuntimeError as e:
            raise ValueError(f"FusedMuon: {e}") from None

    def add_param_group(self, param_group) -> None:
        self._check_options({**self.defaults, **param_group})
        params = param_group["params"]
        params = [params] if isinstance(params, torch.Tensor) else list(params)
        for p in params:
            q = p[1] if isinstance(p, tuple) else p
            if isinstance(q, torch.Tensor) and q.dim() < 2:
                raise ValueError(f"FusedMuon: a parameter {tuple(q.shape)} is no matrix")
        super().add_param_group({**param_group, "params": params})

    @torch.no_grad()
    def step(self, closure=None):
        """One step over every parameter that has a gradient; closure as in torch.optim. What is
        refused is refused before anything changes."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        work = []       # (group, parameters, gradients, momenta) of each group, device and dtype
        for group in self.param_groups:
            _check_numbers("FusedMuon", group)
            runs = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError("FusedMuon: sparse gradients are not supported")
                if not self.state.get(p) and _capturing(p.device):     # each replay would clear it again
                    raise RuntimeError("FusedMuon: a parameter's first step inside a graph capture: make "
                                       "one step with these gradients before the capture")
                runs.setdefault((p.device, p.dtype), []).append(p)
            for ps in runs.values():
                ms = [self.state[p]["momentum_buffer"] if self.state.get(p) else torch.zeros_like(
                    p, dtype=torch.float32, memory_format=torch.contiguous_format) for p in ps]
                work.append((group, ps, [p.grad for p in ps], ms))
        if len(work) > 1:                   # (a call by itself refuses before it launches)
            for group, ps, gs, ms in work:
                _step(ps, gs, ms, group, True)
        for group, ps, gs, ms in work:
            _step(ps, gs, ms, group)
            for p, m in zip(ps, ms):
                if not self.state[p]:
                    self.state[p]["momentum_buffer"] = m
        return loss

    def load_state_dict(self, state_dict) -> None:
        """As torch.optim's, with momenta kept in float32 (torch casts states to their
        parameter's dtype)."""
        saved, groups = state_dict["state"], state_dict["param_groups"]
        if len(groups) == len(self.param_groups):       # (torch refuses it otherwise)
            groups = [{**{k: mine[k] for k in self.defaults if k in mine}, **its}
                      for mine, its in zip(self.param_groups, groups)]
            for mine, its in zip(self.param_groups, groups):
                self._check_options(its)
                for p, i in zip(mine["params"], its["params"]):
                    if saved.get(i) and ("momentum_buffer" not in saved[i] or
                                         saved[i]["momentum_buffer"].shape != p.shape):
                        raise ValueError(f"FusedMuon: no momentum for a parameter {tuple(p.shape)} in its state")
        super().load_state_dict({**state_dict, "param_groups": groups})
        for mine, its in zip(self.param_groups, groups):
            for p, i in zip(mine["params"], its["params"]):
                if saved.get(i):
                    self.state[p] = {"momentum_buffer": torch.empty_like(
                        p, dtype=torch.float32, requires_grad=False,
                        memory_format=torch.contiguous_format).copy_(saved[i]["momentum_buffer"].detach())}
