"""Tensors in 8-bit floating point with a scale for each block of 128, and dense layers that multiply them.

A ``Float8`` holds codes (``torch.float8_e4m3fn`` or ``float8_e5m2``) and, for every 128 of them along a row, a power of two.  The matrix
instructions apply these powers by themselves, and because scaling by them is exact, a number is rounded once, to 4 (3) significant bits, however
often it changes the direction it is quantised along.

``linear_float8`` is a dense layer, y = x w^T, with all three products of a training step in 8 bits, each operand quantised along the
dimension that is summed over: y of x and w along their columns, dx of dy and w along w's rows, dw of dy and x along the
tokens.  ``norm_linear_float8`` puts a root-mean-square norm in front, whose kernel writes the 8 bits that the product reads.  What is kept
of the layer's input for the backward is those 8 bits.  For serving, the weight is quantised once (``to_float8``) and given in w's place.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Union

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from .. import _lib

E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2


class Float8(NamedTuple):
    """codes: (..., 128 * ceil(columns / 128)) of an 8-bit type, zero beyond ``columns``; scales: (..., 4 * ceil(columns / 512)) of
    ``torch.float8_e8m0fnu``, one beyond the last block; columns: the tensor's last dimension.  Both contiguous."""
    codes: torch.Tensor
    scales: torch.Tensor
    columns: int


def to_float8(x: torch.Tensor, dtype: torch.dtype = E4M3) -> Float8:
    """x (float32, bfloat16 or float16) in 8 bits: of each block of 128 along the last dimension the scale is the smallest power of two, 2^-127
    at least, that brings the largest magnitude to at most 448 (``float8_e5m2``: 57344), and a code the element over it, rounded to nearest even.  A block
    that holds an infinity or a NaN has the scale 2^120 (``float8_e5m2``: 2^113); they become NaN (in ``float8_e5m2`` an infinity stays one) and
    numbers below 2^110 (2^96) zero.  Not differentiable: x's own graph is left alone."""
    if x.requires_grad:
        _lib.refuse_lost_tangents("to_float8", x)
        x = x.detach()
    return Float8(*_lib.to_float8(x if x.is_contiguous() else x.contiguous(), dtype), x.shape[-1])


def from_float8(x: Float8, dtype: torch.dtype) -> torch.Tensor:
    """The tensor that a Float8 stands for (bfloat16 and float32 hold its numbers exactly, short of float32's smallest)."""
    return _lib.from_float8(*x, dtype)


def matmul_float8(a: Float8, b: Float8, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """a b^T (..., N) in bfloat16 or float16, of a (..., K) and a matrix b (N, K); sums in float32 between the matrix instructions, which cut what
    lies 2^-14.6 below the largest of eight products.  Not differentiable."""
    if a.columns != b.columns:
        raise ValueError(f"a has {a.columns} columns and b has {b.columns}")
    return _lib.matmul_float8(a.codes, a.scales, b.codes, b.scales, a.columns, dtype)


def _check_weight(x: torch.Tensor, w: torch.Tensor, *others: Optional[torch.Tensor]) -> None:
    """others: the norm's, whose gradients are formed of x's."""
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"products of 8-bit tensors are bfloat16 or float16; got {x.dtype}")
    if w.dim() != 2 or x.dim() < 1 or w.shape[1] != x.shape[-1] or w.dtype != x.dtype or w.device != x.device:
        raise ValueError("the weight must be a (out, in) matrix with the dtype and device of x")
    most = _lib.PRODUCT8_MAX_K
    if (x.numel() > most or w.shape[0] > most) and torch.is_grad_enabled():
        if w.requires_grad and x.shape[:-1].numel() > most:
            raise ValueError(f"the weight's gradient is a sum over {x.shape[:-1].numel()} rows; at most {most} are supported")
        if w.shape[0] > most and any(t is not None and t.requires_grad for t in (x, *others)):
            raise ValueError(f"x's gradient is a sum over {w.shape[0]} outputs; at most {most} are supported")


def _gradients(dy, x8, w, grad_dtype, need_dx, need_dw):
    """(dx, dw) of y = x w^T from x in 8 bits; dy contiguous (..., out)."""
    flat = dy.reshape(dy.shape[:-1].numel(), w.shape[0])
    dx = dw = rows = cols = None
    if need_dx and need_dw:
        *rows, codes, scales = _lib.to_float8_both(flat, grad_dtype)
        cols = codes, scales
    elif need_dx:
        rows = _lib.to_float8(flat, grad_dtype)
    elif need_dw:
        cols = _lib.to_float8_columns(flat, grad_dtype)
    if need_dx:
        dx = _lib.matmul_float8(*rows, *_lib.to_float8_columns(w, E4M3), w.shape[0], dy.dtype).reshape(*dy.shape[:-1], w.shape[1])
    if need_dw:
        codes, scales = (t.reshape(flat.shape[0], t.shape[-1]) for t in x8)
        dw = _lib.matmul_float8(*cols, *_lib.float8_columns(codes, scales, w.shape[1], E4M3), flat.shape[0], dy.dtype)
    return dx, dw


class _LinearFloat8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, grad_dtype):
        codes, scales = _lib.to_float8(x, E4M3)
        need_dw = ctx.needs_input_grad[1]
        ctx.save_for_backward(codes if need_dw else None, scales if need_dw else None, w)
        ctx.grad_dtype = grad_dtype
        return _lib.matmul_float8(codes, scales, *_lib.to_float8(w, E4M3), w.shape[1], x.dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        codes, scales, w = ctx.saved_tensors
        return *_gradients(dy.contiguous(), (codes, scales), w, ctx.grad_dtype, *ctx.needs_input_grad[:2]), None


class _NormLinearFloat8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, gain, w, eps, grad_dtype):
        ctx.set_materialize_grads(False)
        codes, scales, r, rstd = _lib.rms_norm_float8(x, residual, gain, eps)
        need_dw = ctx.needs_input_grad[3]
        ctx.save_for_backward(codes if need_dw else None, scales if need_dw else None, w, x if residual is None else r, rstd, gain)
        ctx.added, ctx.grad_dtype = residual is not None, grad_dtype
        y = _lib.matmul_float8(codes, scales, *_lib.to_float8(w, E4M3), w.shape[1], x.dtype)
        return (y, r) if ctx.added else y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dr=None):
        codes, scales, w, r, rstd, gain = ctx.saved_tensors
        need_x, need_residual, need_gain, need_w = ctx.needs_input_grad[:4]
        dy = dy.contiguous() if dy is not None else r.new_zeros(*r.shape[:-1], w.shape[0])
        need_norm = need_x or need_residual or need_gain
        dn, dw = _gradients(dy, (codes, scales), w, ctx.grad_dtype, need_norm, need_w)
        dx = dgain = None
        if need_norm:
            dx, dgain = _lib.rms_norm_bwd(dn, r, dr.contiguous() if dr is not None else None, rstd, gain, need_gain)
        return dx, dx if ctx.added else None, dgain if need_gain else None, dw, None, None


def _no_gradient(*tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError("a product with a weight in 8 bits is not differentiable; give the weight itself, or call it under torch.no_grad()")


def linear_float8(x: torch.Tensor, w: Union[torch.Tensor, Float8], grad_dtype: torch.dtype = E4M3) -> torch.Tensor:
    """x w^T (..., out) with both operands in 8 bits (``float8_e4m3fn``).

    x: (..., in) bfloat16 or float16.  w: (out, in) of x's dtype, differentiable as x is, or a ``Float8``, laid out once for inference.
    ``grad_dtype``: the 8-bit type of y's gradient in the backward's products; ``float8_e5m2`` trades a bit of each number for range within a block.
    Sums go over 2^22 numbers at most: in, out where x's gradient is wanted, the rows where w's is."""
    x = x if x.is_contiguous() else x.contiguous()
    if isinstance(w, Float8):
        _no_gradient(x)
        return _lib.linear_float8_infer(x, *w)
    _check_weight(x, w)
    _lib.format_code(grad_dtype)
    if not torch.is_grad_enabled() and not _lib.forward_mode():
        return _lib.linear_float8_infer(x, *_lib.to_float8(w.contiguous(), E4M3), w.shape[1])
    if _lib.native_nodes(x):
        return torch.ops.gcg.linear_float8(x, w, grad_dtype)
    return _LinearFloat8.apply(x, w.contiguous(), grad_dtype)


def norm_linear_float8(x: torch.Tensor, gain: Optional[torch.Tensor], w: Union[torch.Tensor, Float8], eps: float = 1e-6,
                       residual: Optional[torch.Tensor] = None, grad_dtype: torch.dtype = E4M3):
    """``linear_float8`` of the root-mean-square norm (norm.py) of x, or of r = x + residual: y, or (y, r) with a residual.  The norm's output
    is in 8 bits only; gradients pass its rounding as if it were not there.  gain: the norm's weight."""
    x = x if x.is_contiguous() else x.contiguous()
    residual = residual if residual is None or residual.is_contiguous() else residual.contiguous()
    ready = isinstance(w, Float8)
    if ready:
        _no_gradient(x, residual, gain)
    else:
        _check_weight(x, w, residual, gain)
        _lib.format_code(grad_dtype)
    if ready or (not torch.is_grad_enabled() and not _lib.forward_mode()):
        y, r = _lib.norm_linear_float8_infer(x, residual, gain, *(w if ready else to_float8(w)), eps)
        return y if residual is None else (y, r)
    if _lib.native_nodes(x):
        out = torch.ops.gcg.norm_linear_float8(x, residual, gain, w, eps, grad_dtype)
        return out[0] if residual is None else tuple(out)
    return _NormLinearFloat8.apply(x, residual, gain, w.contiguous(), eps, grad_dtype)


class LinearFloat8(nn.Module):
    """``linear_float8`` with its weight (out_features, in_features), initialised as ``nn.Linear``'s.

    ``lay_out()`` quantises the weight once for calls without gradients, as a serving program does after loading; until then, and after ``train()``,
    a move or cast of the module, ``load_state_dict`` or any change of the weight that torch counts, every call quantises it.  (It counts none that goes
    by ``weight.data``, a pointer or a replayed graph, of a weight made in inference mode, or inside a traced program: call it again then.)"""

    _laid_out_of = None             # the weight that was laid out, and torch's count of its modifications then

    def __init__(self, in_features: int, out_features: int, grad_dtype: torch.dtype = E4M3, dtype=torch.bfloat16, device=None):
        super().__init__()
        self.in_features, self.out_features, self.grad_dtype = in_features, out_features, grad_dtype
        self.weight = nn.Parameter(torch.empty(out_features, in_features, dtype=dtype, device=device))
        nn.init.kaiming_uniform_(self.weight, a=5 ** 0.5)
        self._laid_out = None

    def lay_out(self) -> "LinearFloat8":
        self._laid_out = to_float8(self.weight)
        self._note()
        return self

    def _note(self) -> None:
        # (in a tuple: an attribute of its own would be a second parameter)
        self._laid_out_of = self.weight, None if self.weight.is_inference() else self.weight._version

    def _current(self) -> bool:
        if self._laid_out is None or self._laid_out_of is None:
            return False
        weight, count = self._laid_out_of
        if self._parameters.get("weight") is not weight:
            return False
        return count is None or torch.compiler.is_compiling() or weight._version == count

    def __getstate__(self):
        """A copy's weight has a count of its own, so what a copy holds is either of its weight as it is, or not there."""
        return {**self.__dict__, "_laid_out": self._laid_out if self._current() else None, "_laid_out_of": None}

    def __setstate__(self, state):
        super().__setstate__(state)
        if "_laid_out_of" not in state:             # (written before it was noted what was laid out)
            self._laid_out = None
        if self._laid_out is not None:
            self._note()

    def _apply(self, fn, recurse=True):
        self._laid_out = None
        return super()._apply(fn, recurse)

    def train(self, mode: bool = True):
        if mode:
            self._laid_out = None
        return super().train(mode)

    def _load_from_state_dict(self, *args, **kwargs):
        self._laid_out = None
        super()._load_from_state_dict(*args, **kwargs)

    def operand(self) -> Union[torch.Tensor, Float8]:
        """The weight, or its 8 bits where they are laid out and no gradient is wanted."""
        return self._laid_out if not torch.is_grad_enabled() and self._current() else self.weight

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return linear_float8(x, self.operand(), self.grad_dtype)
