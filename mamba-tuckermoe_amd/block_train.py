"""The TransformerBlock's FFN sub-block for training on MI355X (gfx950).

TuckerFFNTrain is TuckerFFN (block.py) with gradients: the same attribute and parameter
names, so that what it trained loads into a TuckerFFN (whose layers then want
set_router_mode("capped"), the router that training uses). Its three layers are
TuckerMoETrain with the fused router; what stands around them is fused_block_norm:
    x_f  = norm_ffn(x_res)
    h    = ffn_up(x_f) * silu(ffn_gate(x_f))
    out  = x_res + ls_ffn(ffn_down(h))          (pure_torch_mlx/model.py:337-341)
"""
from __future__ import annotations

import torch.nn as nn

from .block import LayerScale
from .latent import TuckerMoETrain
from .module import RMSNorm
from .train_ops import fused_block_norm


class TuckerFFNTrain(nn.Module):
    """forward(x_res, step=None, mask=None) -> (out, lb_loss, z_loss), the losses summed over
    the three layers. d and cfg as TuckerFFN's; mask (...) bool leaves tokens out (a
    left-out token's layers are their biases). norm_ffn and ls_ffn hold their parameters and
    are not called: hooks on them do not run."""

    def __init__(self, d: int, cfg):
        super().__init__()
        d_ff = getattr(cfg, "ffn_expand", 6) * d
        dims = dict(num_experts=cfg.kmoe_num_experts, top_k=cfg.kmoe_top_k, r1=cfg.kmoe_r1,
                    r2=cfg.kmoe_r2, r3=cfg.kmoe_r3, fused_router=True)
        self.norm_ffn = RMSNorm(d, eps=cfg.rms_norm_eps)
        self.ffn_gate = TuckerMoETrain(d, d_ff, **dims)
        self.ffn_up = TuckerMoETrain(d, d_ff, **dims)
        self.ffn_down = TuckerMoETrain(d_ff, d, **dims)
        self.ls_ffn = LayerScale(d)

    def forward(self, x_res, step=None, mask=None):
        _, x_f = fused_block_norm(x_res, next_weight=self.norm_ffn.weight, eps=self.norm_ffn.eps)
        gate, lb_g, z_g = self.ffn_gate(x_f, step, mask)
        up, lb_u, z_u = self.ffn_up(x_f, step, mask)
        h, _ = fused_block_norm(y=up, gate=gate)
        dn, lb_d, z_d = self.ffn_down(h, step, mask)
        out, _ = fused_block_norm(x_res, dn, gamma=self.ls_ffn.gamma)
        return out, lb_g + lb_u + lb_d, z_g + z_u + z_d
