"""Norms in front of the mixers, forward and backward, with their parameters' gradients.

Layer norm, and root-mean-square norm, which also adds the residual and can write its output in the 8 bits that a dense layer's product
reads (float8.py).

One kernel each way (and a small one that adds the gradient's partial sums): a row is read once and held in registers,
statistics and sums are fp32, every output is rounded once.  With ``save_8bit`` the backward reads the input from its
8-bit checkpoint (act8.py), which the forward writes in the same pass, instead of the input itself.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from .. import _lib
from .float8 import Float8


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


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, w, eps):
        ctx.set_materialize_grads(False)
        y, r, rstd = _lib.rms_norm_fwd(x, residual, w, eps)
        ctx.added = residual is not None
        ctx.save_for_backward(r if ctx.added else x, rstd, w)
        return (y, r) if ctx.added else y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dr=None):
        r, rstd, w = ctx.saved_tensors
        need = ctx.needs_input_grad[2]
        dy = dy.contiguous() if dy is not None else torch.zeros_like(r)
        dx, dw = _lib.rms_norm_bwd(dy, r, dr.contiguous() if dr is not None else None, rstd, w, need)
        return dx, dx if ctx.added else None, dw if need else None, None


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: float = 1e-6, residual: Optional[torch.Tensor] = None):
    """r / sqrt(mean(r^2) + eps) * weight over the last dimension (at most 16384 elements) of r = x; with ``residual`` of r = x + residual, rounded
    to x's dtype, and (y, r) is returned: r is the residual stream after the addition.

    x, residual: float32, bfloat16 or float16; weight: of x's dtype, or float32 with 16-bit x."""
    x = x if x.is_contiguous() else x.contiguous()
    residual = residual if residual is None or residual.is_contiguous() else residual.contiguous()
    if not torch.is_grad_enabled() and not _lib.forward_mode():
        y, r, _ = _lib.rms_norm_fwd(x, residual, weight, eps, stats=False)
        return y if residual is None else (y, r)
    if _lib.native_nodes(x):
        out = torch.ops.gcg.rms_norm(x, residual, weight, eps)
        return out[0] if residual is None else tuple(out)
    return _RMSNorm.apply(x, residual, weight, eps)


class _StreamBeside8Bits(torch.autograd.Function):
    """rms_norm_float8 with a residual: r is a sum with a gradient, the 8 bits beside it have none."""

    @staticmethod
    def forward(ctx, x, residual, w, eps):
        ctx.set_materialize_grads(False)
        codes, scales, r, _ = _lib.rms_norm_float8(x, residual, w, eps)
        ctx.mark_non_differentiable(codes, scales)
        return codes, scales, r

    @staticmethod
    def backward(ctx, _codes, _scales, dr):
        return dr, dr, None, None


def rms_norm_float8(x: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: float = 1e-6, residual: Optional[torch.Tensor] = None):
    """``rms_norm`` with y as a ``Float8`` (float8.py), formed of y in float32: y, or (y, r).  y is not differentiable: no gradient reaches x, the
    residual or the weight through it (``norm_linear_float8`` is the differentiable form, with the product).  r is, as the sum that it is."""
    recorded = residual is not None and torch.is_grad_enabled() and (x.requires_grad or residual.requires_grad)
    if not recorded:
        _lib.refuse_lost_tangents("rms_norm_float8", x, residual, weight)
        x, residual, weight = (t.detach() if t is not None and t.requires_grad else t for t in (x, residual, weight))
    x = x if x.is_contiguous() else x.contiguous()
    residual = residual if residual is None or residual.is_contiguous() else residual.contiguous()
    if recorded:
        node = torch.ops.gcg.rms_norm_float8_stream if _lib.native_nodes(x) else _StreamBeside8Bits.apply
        codes, scales, r = node(x, residual, weight, eps)
    else:
        codes, scales, r, _ = _lib.rms_norm_float8(x, residual, weight, eps)
    y = Float8(codes, scales, x.shape[-1])
    return y if residual is None else (y, r)


class RMSNorm(nn.Module):
    """``rms_norm`` with its weight, ones."""

    def __init__(self, hidden_size: int, eps: float = 1e-6, dtype=torch.float32, device=None):
        super().__init__()
        self.hidden_size, self.eps = hidden_size, eps
        self.weight = nn.Parameter(torch.ones(hidden_size, dtype=dtype, device=device))

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None):
        assert x.shape[-1] == self.hidden_size
        return rms_norm(x, self.weight, self.eps, residual)
