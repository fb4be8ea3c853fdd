"""A pre-norm layer of a hybrid model around any of the mixers: x + out(mixer(projection(norm(x)))).

What the operators of this package are for when used together: ``LayerNorm`` (norm.py), the dense projection to three times
the width, ``HyenaMixer`` (hyena.py) or ``LinearAttention`` (linear_attention.py), the output projection and the residual.  With
``save_8bit`` the norm's input and the mixer's features are kept in 8 bits for the backward (act8.py).  A layer with linear
attention also decodes: ``prefill`` takes a prompt and returns the state after it, ``step`` one token.
"""
from __future__ import annotations

from typing import Optional, Union

import torch
import torch.nn as nn

from .hyena import HyenaMixer
from .linear_attention import LinearAttention
from .norm import LayerNorm


class MixerBlock(nn.Module):
    """x: (b, l, hidden_size).  ``mixer``: a HyenaMixer or a LinearAttention of that width; ``save_8bit`` sets the mixer's too
    (a mixer that keeps its features in 8 bits by itself goes on doing so without)."""

    def __init__(self, hidden_size: int, mixer: Union[HyenaMixer, LinearAttention], eps: float = 1e-5, save_8bit: bool = False,
                 dtype=torch.float32, device=None):
        super().__init__()
        self.mixer = mixer
        mixer.save_8bit = mixer.save_8bit or save_8bit
        self.norm = LayerNorm(hidden_size, eps, save_8bit=save_8bit, dtype=dtype, device=device)
        self.projection = nn.Linear(hidden_size, 3 * hidden_size, bias=False, dtype=dtype, device=device)
        self.out = nn.Linear(hidden_size, hidden_size, bias=False, dtype=dtype, device=device)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return x + self.out(self.mixer(self.projection(self.norm(x))))

    def _recurrent(self) -> LinearAttention:
        if not isinstance(self.mixer, LinearAttention):
            raise RuntimeError(f"{type(self.mixer).__name__} carries no state; decoding needs a LinearAttention mixer")
        return self.mixer

    @torch.no_grad()
    def prefill(self, x: torch.Tensor, state: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None):
        """(the layer's output, the state after each entry's last row); ``lengths`` as in linear_attention."""
        y, state = self._recurrent().prefill(self.projection(self.norm(x)), state, lengths)
        return x + self.out(y), state

    @torch.no_grad()
    def step(self, x: torch.Tensor, state: torch.Tensor) -> torch.Tensor:
        """The layer's output (b, hidden_size) for one token of every entry; ``state`` is moved on in place."""
        return x + self.out(self._recurrent().step(self.projection(self.norm(x)), state))
