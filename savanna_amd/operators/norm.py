"""Layer norm in front of the mixers, forward and backward, with the weight's and bias's gradient.

One kernel each way (and a small one that adds the gradient's partial sums): a row is read once and held in registers,
statistics and sums are fp32, every output is rounded once.  With ``save_8bit`` the backward reads the input from its
8-bit checkpoint (act8.py), which the forward writes in the same pass, instead of the input itself.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn

from .. import _lib


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b, eps, save_8bit):
        y, stats, codes, scales = _lib.layer_norm_fwd(x, w, b, eps, save_8bit)
        ctx.save_for_backward(*((None, codes, scales) if save_8bit else (x, None, None)), stats, w, b)
        return y

    @staticmethod
    def backward(ctx, dy):
        _, need_dw, need_db = ctx.needs_input_grad[:3]
        dx, dw, db = _lib.layer_norm_bwd(dy if dy.is_contiguous() else dy.contiguous(), *ctx.saved_tensors, need_dw, need_db)
        return dx, dw if need_dw else None, db if need_db else None, None, None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, eps: float = 1e-5,
               save_8bit: bool = False) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over x's last dimension (at most 16384 elements).

    x: float32, bfloat16 or float16; weight and bias: of x's dtype, or float32 with 16-bit x.  ``save_8bit``: the backward
    pass works on x's 8-bit checkpoint, which is all that is kept of x (1.03 bytes an element)."""
    x = x if x.is_contiguous() else x.contiguous()
    if not torch.is_grad_enabled() and not _lib.forward_mode():
        return _lib.layer_norm_fwd(x, weight, bias, eps, stats=False)[0]
    if _lib.native_nodes(x):
        return torch.ops.gcg.layer_norm(x, weight, bias, eps, save_8bit)
    return _LayerNorm.apply(x, weight, bias, eps, save_8bit)


class LayerNorm(nn.Module):
    """``layer_norm`` with its parameters: weight ones, bias zeros (None with ``bias=False``)."""

    def __init__(self, hidden_size: int, eps: float = 1e-5, bias: bool = True, save_8bit: bool = False, dtype=torch.float32,
                 device=None):
        super().__init__()
        self.hidden_size, self.eps, self.save_8bit = hidden_size, eps, save_8bit
        self.weight = nn.Parameter(torch.ones(hidden_size, dtype=dtype, device=device))
        self.bias = nn.Parameter(torch.zeros(hidden_size, dtype=dtype, device=device)) if bias else None

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        assert x.shape[-1] == self.hidden_size
        return layer_norm(x, self.weight, self.bias, self.eps, self.save_8bit)
