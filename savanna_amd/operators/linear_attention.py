"""Linear attention with a decay for each head: a mixer that carries a state, beside the convolutional ones of hyena.py.

With f = exp(log_decay[h]) and a state S of dk x dv (fp32) for every batch entry and head

    S_t = f S_{t-1} + k_t v_t^T,    o_t = scale q_t S_t

``linear_attention`` is the chunked form for prompts and training (differentiable in q, k, v and the initial state),
``linear_attention_step`` the recurrent form for one token, ``linear_attention_features`` the training form on the
projected features before their split.  The decays are constants of the heads, as the decay of an explicit hyena filter is.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn

from .. import _lib
from .act8 import pack8, unpack8


class _LinearAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, initial, lengths, scale, final):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(q, k, v, log_decay, initial, lengths)
        ctx.scale = scale
        return _lib.linear_attn_fwd(q, k, v, log_decay, initial, lengths, scale, final)

    @staticmethod
    def backward(ctx, do, dfinal):
        q, k, v, log_decay, initial, lengths = ctx.saved_tensors
        do = do if do is not None else torch.zeros(v.shape, dtype=v.dtype, device=v.device)
        dfinal = dfinal.contiguous() if dfinal is not None else None
        need = initial is not None and ctx.needs_input_grad[4]
        dq, dk, dv, di = _lib.linear_attn_bwd(do, q, k, v, log_decay, initial, lengths, dfinal, ctx.scale, need)
        return dq, dk, dv, None, di, None, None, None


class _PackedLinearAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, features, heads, log_decay, scale, save_8bit):
        kept = pack8(features) if save_8bit else None
        ctx.save_for_backward(*((kept.codes, kept.scales) if save_8bit else (features, None)), log_decay)
        ctx.rest = heads, scale, features.dtype, save_8bit
        return _lib.linear_attn_packed_fwd(features, heads, log_decay, scale)

    @staticmethod
    def backward(ctx, do):
        kept, scales, log_decay = ctx.saved_tensors
        heads, scale, dtype, save_8bit = ctx.rest
        features = _lib.unpack8(kept, scales, dtype) if save_8bit else kept
        return _lib.linear_attn_packed_bwd(do, features, heads, log_decay, scale), None, None, None, None


def _constant(log_decay: torch.Tensor) -> None:
    if torch.is_grad_enabled() and log_decay.requires_grad:
        raise RuntimeError("log_decay is a constant of the heads and has no gradient; pass log_decay.detach()")


def linear_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, scale: Optional[float] = None,
                     initial_state: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                     output_final_state: bool = False):
    """o (bs, L, H, dv), or (o, final state) with ``output_final_state``.

    q, k: (bs, L, H, dk), v: (bs, L, H, dv), float32, bfloat16 or float16, head dimensions up to 256; read where they lie if
    their last dimension is contiguous (views of one projection are not copied).  log_decay: (H,) float32, at most 0.
    scale: dk ** -0.5 unless given.  initial_state and the final state: contiguous (bs, H, dk, dv) float32.  lengths: (bs,)
    int32; rows of an entry from its length on are not read, their outputs and gradients are zero, and its final state is
    the one after its last row.

    States and sums are float32.  With 16-bit tensors the matrix instructions take 16-bit operands, so scores and the state's
    read-out copy are rounded to the type once before the output is; where a state is a result, the rows it adds up are kept
    to more bits, and ``o`` may then round differently.  Infinities and NaN reach later rows only."""
    _constant(log_decay)
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    if not torch.is_grad_enabled() and not _lib.forward_mode():
        o, final = _lib.linear_attn_fwd(q, k, v, log_decay, initial_state, lengths, scale, output_final_state)
        return (o, final) if output_final_state else o
    if _lib.native_nodes(q) and v.numel() > 0:
        out = torch.ops.gcg.linear_attn(q, k, v, log_decay, initial_state, lengths, scale, output_final_state)
        return tuple(out) if output_final_state else out[0]
    o, final = _LinearAttention.apply(q, k, v, log_decay, initial_state, lengths, scale, output_final_state)
    return (o, final) if output_final_state else o


def linear_attention_features(features: torch.Tensor, num_heads: int, log_decay: torch.Tensor, scale: Optional[float] = None,
                              save_8bit: bool = False) -> torch.Tensor:
    """o (bs, L, H, d) of the projected features (bs, L, 3 * H * d), laid out "(p h d)" with p = q, k, v: read in place, and their
    gradient written in the same layout.  ``save_8bit``: only their 8-bit checkpoint (act8.py) is kept for the backward."""
    _constant(log_decay)
    features = features if features.is_contiguous() else features.contiguous()
    scale = (features.shape[-1] // (3 * num_heads)) ** -0.5 if scale is None else scale
    if not torch.is_grad_enabled() and not _lib.forward_mode():
        return _lib.linear_attn_packed_fwd(features, num_heads, log_decay, scale)
    if _lib.native_nodes(features):
        return torch.ops.gcg.linear_attn_packed(features, num_heads, log_decay, scale, save_8bit)
    return _PackedLinearAttention.apply(features, num_heads, log_decay, scale, save_8bit)


def linear_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, state: torch.Tensor,
                          scale: Optional[float] = None) -> torch.Tensor:
    """o (bs, H, dv) of one token, q, k: (bs, H, dk), v: (bs, H, dv).  ``state`` (bs, H, dk, dv) float32, contiguous, is moved
    on in place.  Not differentiable."""
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, log_decay, state)):
        raise RuntimeError("linear_attention_step is not differentiable; use linear_attention, or call it under torch.no_grad()")
    return _lib.linear_attn_step(q, k, v, log_decay, state, q.shape[-1] ** -0.5 if scale is None else scale)


class LinearAttention(nn.Module):
    """The mixer on projected features (bs, L, 3 * hidden_size), laid out "(p h d)" with p = q, k, v -> (bs, L, hidden_size).

    ``log_decay``: a buffer, rates spaced over the heads' logarithm from a memory of ``shortest`` tokens to one of ``longest``; it stays
    float32 when the module is cast.
    ``prefill`` also returns the state after a prompt (of ``lengths``, if its entries differ), ``step`` takes one token's
    features (bs, 3 * hidden_size) and moves that state on in place."""

    def __init__(self, hidden_size: int, num_heads: int, shortest: float = 8.0, longest: float = 4096.0, save_8bit: bool = False,
                 device=None):
        super().__init__()
        assert hidden_size % num_heads == 0
        self.hidden_size, self.num_heads, self.head_dim = hidden_size, num_heads, hidden_size // num_heads
        self.save_8bit = save_8bit
        spread = torch.linspace(0, 1, num_heads, dtype=torch.float32, device=device)
        self.register_buffer("log_decay", -1.0 / (shortest * (longest / shortest) ** spread))

    def _apply(self, fn, recurse=True):
        """Moves the decays with the module and leaves them in fp32 when it is cast: rounded to 16 bits they would be others."""
        decay = self.log_decay
        super()._apply(fn, recurse)
        if self.log_decay.dtype != decay.dtype:
            self.log_decay = decay.to(self.log_decay.device)
        return self

    def _split(self, features: torch.Tensor):
        return features.unflatten(-1, (3, self.num_heads, self.head_dim)).unbind(-3)

    def forward(self, features: torch.Tensor) -> torch.Tensor:
        return linear_attention_features(features, self.num_heads, self.log_decay, save_8bit=self.save_8bit).flatten(2)

    def prefill(self, features: torch.Tensor, state: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None):
        o, state = linear_attention(*self._split(features), self.log_decay, initial_state=state, lengths=lengths,
                                    output_final_state=True)
        return o.flatten(2), state

    def step(self, features: torch.Tensor, state: torch.Tensor) -> torch.Tensor:
        return linear_attention_step(*self._split(features), self.log_decay, state).flatten(1)
