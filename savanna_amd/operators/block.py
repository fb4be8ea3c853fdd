"""Pre-norm layers of a hybrid model around any of the mixers: x + out(mixer(projection(norm(x)))).

What the operators of this package are for when used together: ``LayerNorm`` (norm.py), the dense projection to three times
the width, ``HyenaMixer`` (hyena.py) or ``LinearAttention`` (linear_attention.py), the output projection and the residual.  With
``save_8bit`` the norm's input and the mixer's features are kept in 8 bits for the backward (act8.py).  A layer with linear
attention or a ``GatedRecurrence`` (gated_recurrence.py) also decodes: ``prefill`` takes a prompt and returns the state after it, ``step`` one token.

``MixerBlockFloat8`` is the same layer with a root-mean-square norm that adds the residual and dense layers in 8-bit floating point (float8.py).
"""
from __future__ import annotations

from typing import Optional, Union

import torch
import torch.nn as nn

from .float8 import E4M3, LinearFloat8, norm_linear_float8
from .gated_recurrence import GatedRecurrence
from .hyena import HyenaMixer
from .linear_attention import LinearAttention
from .norm import LayerNorm, RMSNorm

Mixer = Union[HyenaMixer, LinearAttention, GatedRecurrence]


def _with_state(mixer: Mixer):
    if not isinstance(mixer, (LinearAttention, GatedRecurrence)):
        raise RuntimeError(f"{type(mixer).__name__} carries no state; decoding needs a LinearAttention or GatedRecurrence mixer")
    return mixer


class MixerBlock(nn.Module):
    """x: (b, l, hidden_size).  ``mixer``: a HyenaMixer, a LinearAttention or a GatedRecurrence of that width; ``save_8bit`` sets the mixer's
    too (a mixer that keeps its features in 8 bits by itself goes on doing so without; a GatedRecurrence has no such form)."""

    def __init__(self, hidden_size: int, mixer: Mixer, eps: float = 1e-5, save_8bit: bool = False,
                 dtype=torch.float32, device=None):
        super().__init__()
        self.mixer = mixer
        if not isinstance(mixer, GatedRecurrence):
            mixer.save_8bit = mixer.save_8bit or save_8bit
        elif save_8bit:
            raise ValueError("a GatedRecurrence keeps its features in their own type; save_8bit is not for it")
        self.norm = LayerNorm(hidden_size, eps, save_8bit=save_8bit, dtype=dtype, device=device)
        self.projection = nn.Linear(hidden_size, 3 * hidden_size, bias=False, dtype=dtype, device=device)
        self.out = nn.Linear(hidden_size, hidden_size, bias=False, dtype=dtype, device=device)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return x + self.out(self.mixer(self.projection(self.norm(x))))

    @torch.no_grad()
    def prefill(self, x: torch.Tensor, state: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None):
        """(the layer's output, the state after each entry's last row); ``lengths`` as in linear_attention."""
        y, state = _with_state(self.mixer).prefill(self.projection(self.norm(x)), state, lengths)
        return x + self.out(y), state

    @torch.no_grad()
    def step(self, x: torch.Tensor, state: torch.Tensor) -> torch.Tensor:
        """The layer's output (b, hidden_size) for one token of every entry; ``state`` is moved on in place."""
        return x + self.out(_with_state(self.mixer).step(self.projection(self.norm(x)), state))


class MixerBlockFloat8(nn.Module):
    """The layer with its two dense layers in 8-bit floating point, on a residual stream that each layer's norm adds up: ``forward(x, residual)``
    takes what the layer before added to the stream (the embedding, without ``residual``, in front) and the stream before that addition, both
    (b, l, hidden_size), and returns the same two of this layer.  Behind the last layer, ``rms_norm(x, weight, residual=residual)`` or their sum.

    Parameters are of ``dtype``, bfloat16 or float16.  ``lay_out`` quantises the weights once, for serving."""

    def __init__(self, hidden_size: int, mixer: Mixer, eps: float = 1e-6, grad_dtype: torch.dtype = E4M3, dtype=torch.bfloat16, device=None):
        super().__init__()
        self.mixer, self.grad_dtype = mixer, grad_dtype
        self.norm = RMSNorm(hidden_size, eps, dtype=dtype, device=device)
        self.projection = LinearFloat8(hidden_size, 3 * hidden_size, grad_dtype, dtype=dtype, device=device)
        self.out = LinearFloat8(hidden_size, hidden_size, grad_dtype, dtype=dtype, device=device)

    def lay_out(self) -> "MixerBlockFloat8":
        self.projection.lay_out()
        self.out.lay_out()
        return self

    def _features(self, x: torch.Tensor, residual: Optional[torch.Tensor]):
        """(the projected features, the stream)"""
        y = norm_linear_float8(x, self.norm.weight, self.projection.operand(), self.norm.eps, residual, self.grad_dtype)
        return (y, x) if residual is None else y

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None):
        features, residual = self._features(x, residual)
        return self.out(self.mixer(features)), residual

    @torch.no_grad()
    def prefill(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None, state: Optional[torch.Tensor] = None,
                lengths: Optional[torch.Tensor] = None):
        """(x, residual, the state after each entry's last row)"""
        features, residual = self._features(x, residual)
        y, state = _with_state(self.mixer).prefill(features, state, lengths)
        return self.out(y), residual, state

    @torch.no_grad()
    def step(self, x: torch.Tensor, state: torch.Tensor, residual: Optional[torch.Tensor] = None):
        """(x, residual), both (b, hidden_size), for one token of every entry; ``state`` is moved on in place."""
        features, residual = self._features(x, residual)
        return self.out(_with_state(self.mixer).step(features, state)), residual
