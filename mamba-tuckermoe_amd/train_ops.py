"""The operators of a training step around the expert contraction, on MI355X (gfx950).

fused_router      the training layer's router with its balance and z losses and per-expert
                  counts (sft_cot_bundle/scripts/model.py:318-332), and its gradient
fused_block_norm  the norms before and after a block with the block's gate and the residual's
                  scale (pure_torch_mlx/model.py:258-260, :337-341), and their gradients

They take bfloat16 or float32 tensors on a HIP device (no fallback), compute in float32 and
round each output once. Both run on the current stream, allocate with torch's allocator and
wait for nothing, so that they can be captured into a HIP graph; a gradient of their
gradients is refused, and so is a forward-mode derivative.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import _lib


class Routing(NamedTuple):
    """What fused_router returns."""
    idx: torch.Tensor       # (B, k) int64, by descending logit; -1 for masked tokens
    weights: torch.Tensor   # (B, k) float32
    lb_loss: torch.Tensor   # float32
    z_loss: torch.Tensor    # float32
    counts: torch.Tensor    # (E) int64: how many tokens selected each expert


def fused_router(raw: torch.Tensor, top_k: int, temperature: Union[float, torch.Tensor],
                 scale: float = 10.0, mask: Optional[torch.Tensor] = None) -> Routing:
    """Routes tokens by their raw logits (B, E), E <= 256 and top_k <= 16:

        a = scale tanh(raw / scale);  P = softmax(a / temperature)
        idx = the top_k largest raw (the lowest index first on ties)
        weights = P[idx] / (sum P[idx] + 1e-6)
        lb_loss = E sum_e (counts[e] / N) (sum_b P[b, e] / N)
        z_loss = sum_b logsumexp(a[b])^2 / N

    over the N tokens that mask (B, bool; None: every token) does not leave out. A token
    that it leaves out selects nothing: idx -1, which FusedLatentMoE skips, weights 0 and no
    gradient, whatever its logits hold. With no token at all the losses are 0. Gradients
    flow from weights, lb_loss and z_loss to raw. temperature is a number (a tensor on the
    CPU is read as one), or a float32 tensor of one value on raw's device, which is read
    when the kernels run (its validity is the caller's) and gets no gradient."""
    tau = None
    if isinstance(temperature, torch.Tensor):
        if temperature.device.type == "cuda":
            tau = temperature
        else:
            temperature = float(temperature)
    return Routing(*_lib.native().router(raw, top_k, None if tau is not None else float(temperature),
                                         tau, float(scale), mask))


def fused_block_norm(x: Optional[torch.Tensor] = None, y: Optional[torch.Tensor] = None,
                     gate: Optional[torch.Tensor] = None,
                     post_weight: Optional[torch.Tensor] = None,
                     gamma: Optional[torch.Tensor] = None,
                     next_weight: Optional[torch.Tensor] = None,
                     eps: float = 1e-5) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """The end of one block and the beginning of the next, (r, h):

        u = y * silu(gate);  f = RMSNorm(u, post_weight);  r = x + gamma * f
        h = RMSNorm(r, next_weight),   RMSNorm(v, w) = v / sqrt(mean(v^2) + eps) * w

    x (the residual), y (the block's output) and gate are (..., d) of one shape, the weights
    (d), all of one dtype; what is None falls away (without next_weight h is None). Without y
    there is next_weight alone: r is x itself and h its norm. d <= 16384; rows may lie at any
    one stride. h is taken from the unrounded r."""
    r, h = _lib.native().block_norm(x, y, gate, post_weight, gamma, next_weight, float(eps))
    return (x if y is None else r), h
