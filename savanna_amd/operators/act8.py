"""Activation checkpoints in 8 bits: what a layer keeps of its activations for the backward pass, at about half of their
16-bit size (128 elements along the last dimension share an fp32 scale: 1.03 bytes an element).

``pack8`` and ``unpack8`` are the kernels by themselves.  The layers that use them: ``layer_norm(..., save_8bit=True)``
(norm.py) writes the checkpoint in the forward's own pass and reads it in the backward's; ``HyenaMixer(..., save_8bit=True)``
(hyena.py) and ``LinearAttention(..., save_8bit=True)`` (linear_attention.py) keep the projected features as one.  Forward
results do not change; a mixer's gradients are those at its features' 8-bit values, half a step (0.4 % of the largest magnitude
of 128 neighbours) at most from the exact ones, and the norm's are its formula's with those values about the exact row's mean and rstd.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from .. import _lib


class Packed8(NamedTuple):
    """codes: int8 of the tensor's shape; scales: float32, one for every 128 elements of a row; dtype: the tensor's."""
    codes: torch.Tensor
    scales: torch.Tensor
    dtype: torch.dtype


def pack8(x: torch.Tensor) -> Packed8:
    """The 8-bit checkpoint of x: scale = top * fp32(1 / 127), code = rint(x * (127 / top)), top the largest magnitude of a
    block.  A block that holds an infinity or a NaN comes back as NaN throughout; below 2^-100 as zeros.  Not
    differentiable: x's own graph is left alone."""
    x = x.detach()
    codes, scales = _lib.pack8(x if x.is_contiguous() else x.contiguous())
    return Packed8(codes, scales, x.dtype)


def unpack8(packed: Packed8) -> torch.Tensor:
    """The tensor a checkpoint stands for: code * scale, rounded once to the tensor's type."""
    return _lib.unpack8(packed.codes, packed.scales, packed.dtype)
