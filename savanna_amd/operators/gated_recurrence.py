"""Gated linear recurrence: a mixer whose every channel carries one number, with a decay that the data choose.

    a_t = sigmoid(f_t + bias),   h_t = a_t h_{t-1} + (1 - a_t) x_t,   y_t = gate_t h_t

``gated_recurrence`` is the form for prompts and training (differentiable in x, f, gate, bias and the initial state),
``gated_recurrence_features`` the training form on the projected features before their split, ``gated_recurrence_step`` the one for a token.
One kernel each way: time is cut into chunks that hand a state on to each other while their rows wait in registers.
"""
from __future__ import annotations

import math
from typing import Optional

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from .. import _lib


class _GatedRecurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, f, gate, bias, initial, lengths, final):
        ctx.set_materialize_grads(False)
        y, last, states = _lib.scan_fwd(x, f, gate, bias, initial, lengths, final, True)
        ctx.save_for_backward(x, f, gate, bias, states, lengths)
        return (y, last) if final else y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dfinal=None):
        x, f, gate, bias, states, lengths = ctx.saved_tensors
        need_bias, need_initial = ctx.needs_input_grad[3:5]
        dy = dy if dy is not None else torch.zeros_like(x)
        dfinal = dfinal.contiguous() if dfinal is not None else None
        dx, df, dg, db, di = _lib.scan_bwd(dy, x, f, gate, bias, states, lengths, dfinal, need_bias, need_initial)
        return dx, df, dg if gate is not None else None, db if need_bias else None, di if need_initial else None, None, None


class _PackedRecurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, features, bias):
        y, states = _lib.scan_packed_fwd(features, bias, True)
        ctx.save_for_backward(features, bias, states)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        features, bias, states = ctx.saved_tensors
        need = ctx.needs_input_grad[1]
        d, db = _lib.scan_packed_bwd(dy, features, bias, states, need)
        return d, db if need else None


def gated_recurrence(x: torch.Tensor, f: torch.Tensor, gate: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                     initial_state: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None, output_final_state: bool = False):
    """y (bs, L, D), or (y, final state) with ``output_final_state``.

    x, f, gate: (bs, L, D), float32, bfloat16 or float16, read where they lie if their last dimension is contiguous (views of one
    projection are not copied); without a gate y = h.  bias: (D,) float32.  initial_state and the final state: contiguous (bs, D) float32.
    lengths: (bs,) int32; rows of an entry from its length on are not read, their outputs and gradients are zero, and its final
    state is the one after its last row.  The state and all sums are float32, y and the gradients are rounded once."""
    if not torch.is_grad_enabled() and not _lib.forward_mode():
        y, last, _ = _lib.scan_fwd(x, f, gate, bias, initial_state, lengths, output_final_state, False)
        return (y, last) if output_final_state else y
    if _lib.native_nodes(x):
        out = torch.ops.gcg.scan(x, f, gate, bias, initial_state, lengths, output_final_state)
        return tuple(out) if output_final_state else out[0]
    return _GatedRecurrence.apply(x, f, gate, bias, initial_state, lengths, output_final_state)


def gated_recurrence_features(features: torch.Tensor, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y (bs, L, D) of the projected features (bs, L, 3 * D), laid out "(p d)" with p = x, f, gate: read in place, and their gradient
    written in the same layout."""
    features = features if features.is_contiguous() else features.contiguous()
    if not torch.is_grad_enabled() and not _lib.forward_mode():
        return _lib.scan_packed_fwd(features, bias, False)[0]
    if _lib.native_nodes(features):
        return torch.ops.gcg.scan_packed(features, bias)
    return _PackedRecurrence.apply(features, bias)


def gated_recurrence_step(x: torch.Tensor, f: torch.Tensor, state: torch.Tensor, gate: Optional[torch.Tensor] = None,
                          bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y (bs, D) of one token, x, f, gate: (bs, D).  ``state`` (bs, D) float32, contiguous, is moved on in place.  Not differentiable."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, f, gate, bias, state)):
        raise RuntimeError("gated_recurrence_step is not differentiable; use gated_recurrence, or call it under torch.no_grad()")
    return _lib.scan_step(x, f, gate, bias, state)


class GatedRecurrence(nn.Module):
    """The mixer on projected features (bs, L, 3 * hidden_size), laid out "(p d)" with p = x, f, gate -> (bs, L, hidden_size).

    ``decay_bias``: a parameter, log of the channels' memories, which start spaced over their logarithm from ``shortest`` tokens to ``longest``; it
    stays float32 when the module is cast.  ``prefill`` also returns the state after a prompt (of ``lengths``, if its entries
    differ), ``step`` takes one token's features (bs, 3 * hidden_size) and moves that state on in place."""

    def __init__(self, hidden_size: int, shortest: float = 8.0, longest: float = 4096.0, device=None):
        super().__init__()
        self.hidden_size = hidden_size
        spread = torch.linspace(0, 1, hidden_size, dtype=torch.float32, device=device)
        self.decay_bias = nn.Parameter(math.log(shortest) + math.log(longest / shortest) * spread)

    def _apply(self, fn, recurse=True):
        """Moves the bias with the module and leaves it in fp32 when it is cast: rounded to 16 bits, long memories would be others."""
        def keep(t):
            new = fn(t)
            return t.to(new.device) if t is not None and t.dtype == torch.float32 and new.dtype != t.dtype and new.is_floating_point() else new
        return super()._apply(keep, recurse)

    def _split(self, features: torch.Tensor):
        return features.unflatten(-1, (3, self.hidden_size)).unbind(-2)

    def forward(self, features: torch.Tensor) -> torch.Tensor:
        return gated_recurrence_features(features, self.decay_bias)

    def prefill(self, features: torch.Tensor, state: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None):
        x, f, gate = self._split(features)
        return gated_recurrence(x, f, gate, self.decay_bias, initial_state=state, lengths=lengths, output_final_state=True)

    def step(self, features: torch.Tensor, state: torch.Tensor) -> torch.Tensor:
        x, f, gate = self._split(features)
        return gated_recurrence_step(x, f, state, gate, self.decay_bias)
