"""Definitions in 64 bits of the operators of a layer in 8-bit floating point: what their kernels' tests compare with."""
import torch

TOP = {torch.float8_e4m3fn: 448.0, torch.float8_e5m2: 57344.0}
BITS = {torch.float8_e4m3fn: (3, -6), torch.float8_e5m2: (2, -14)}          # of the fraction; the smallest normal number's exponent
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}      # half an f16 denormal


def two_to(e):
    """2^e in 64 bits, exactly."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def float8(x, fmt=torch.float8_e4m3fn):
    """(values, exponents) of finite x (..., D) in 8 bits, both in 64 bits: a block of 128 is divided by the smallest power of two, 2^-127 at
    least, that brings its largest magnitude to at most the format's largest number, and rounded to nearest even."""
    D, (bits, low) = x.shape[-1], BITS[fmt]
    v = torch.nn.functional.pad(x.double(), (0, -D % 128)).unflatten(-1, (-1, 128))
    part, power = torch.frexp(v.abs().amax(-1, keepdim=True))
    top = TOP[fmt]
    e = power - (9 if top == 448.0 else 16) + (part > 0.875).int()
    e = torch.where(part > 0, e, 0).clamp(min=-127)
    q = v / two_to(e)
    step = two_to((torch.frexp(q)[1] - 1).clamp(min=low) - bits)
    q = torch.round(q / step) * step
    return (q * two_to(e)).flatten(-2)[..., :D], e.squeeze(-1)


def values(q):
    """What a Float8 stands for, in 64 bits."""
    scale = q.scales.view(torch.uint8).int() - 127
    v = q.codes.double() * two_to(scale).repeat_interleave(128, -1)[..., :q.codes.shape[-1]]
    return v[..., :q.columns]


def check(got, ref, tol, what):
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    off = (got.double() - ref).abs() - tol
    assert (off <= 0).all(), f"{what}: {off.max().item():.3e} over a tolerance of {tol.expand_as(ref).flatten()[off.argmax()].item():.3e}"
