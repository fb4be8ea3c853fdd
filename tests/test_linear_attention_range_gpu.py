"""Linear attention in f16 at the ends of the type's range, against its recurrence in 64 bits.

Tolerances, by output element: as in test_linear_attention_gpu.py, U |ref| + (2 U + 2^-15) A with A the sum of its terms'
magnitudes, and 2^-25, half an f16 denormal, for the output's own rounding.  Operands that are scaled by a power of two before they are
rounded lose 2^-25 of the largest one beside them at most; the inputs here are such that this stays below 2^-15 A.  A state is off by
2^-17 of its A."""
import pytest
import torch

from savanna_amd.operators.linear_attention import linear_attention
from test_linear_attention_gpu import DEV, recurrence, step

pytestmark = pytest.mark.gpu
U16, U32 = 2.0 ** -11, 2.0 ** -24
NAMES = ("q", "k", "v", "do")


def reference(t, log_decay, scale, initial, dfinal):
    size = lambda x: x.abs() if x is not None else None                          # noqa: E731
    ref = recurrence(*(t[n] for n in NAMES), log_decay, scale, initial, dfinal)
    assert all(ref[i].abs().max() < 60000 for i in (0, 2, 3, 4)), "results that f16 holds"
    mag = recurrence(*(t[n].abs() for n in NAMES), log_decay, scale, size(initial), size(dfinal))
    return [(r, 2.0 ** -17 * a + U32 if i in (1, 5) else U16 * r.abs() + (2 * U16 + 2.0 ** -15) * a + 2.0 ** -25)
            for i, (r, a) in enumerate(zip(ref, mag))]


def check(got, want, what):
    for name, g, (ref, tol) in zip(("o", "final", "dq", "dk", "dv", "dinitial"), got, want):
        if g is None:
            continue
        off = (g.double() - ref).abs()
        assert bool((off <= tol).all()), f"{what} {name}: {int((~(off <= tol)).sum())} of {off.numel()} off, by up to {off.max().item():.3e}"


def data(L, H, dk, dv, seed, size):
    """Normal values of the given size, as f16."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return {n: (size * torch.randn(1, L, H, d, generator=gen, device=DEV)).half() for n, d in zip(NAMES, (dk, dk, dv, dv))}, gen


@pytest.mark.parametrize("states", [False, True])
@pytest.mark.parametrize("which", NAMES)
@pytest.mark.parametrize("L,H,dk,dv", [(150, 3, 64, 48), (2049, 2, 64, 64)])
def test_operands_near_the_largest(gcg_lib, L, H, dk, dv, which, states):
    """One operand between half the type's largest value and all of it, as loss-scaled gradients may be; results that fit."""
    t, gen = data(L, H, dk, dv, 1, 2.0 ** -4)
    big = t[which]
    size = 0.5 + 0.5 * torch.rand(big.shape, generator=gen, device=DEV)
    t[which] = (65504 * size * torch.where(big < 0, -1.0, 1.0)).half()
    ld = torch.tensor([-0.01, -0.003, -0.3], device=DEV)[:H].contiguous()
    initial, dfinal = (2.0 ** -8 * torch.randn(1, H, dk, dv, generator=gen, device=DEV) if states else None for _ in range(2))
    got = step(*(t[n] for n in NAMES), ld, 0.125, initial, dfinal)
    check(got, reference(t, ld, 0.125, initial, dfinal), f"large {which}")


@pytest.mark.parametrize("states", [False, True])
@pytest.mark.parametrize("which", NAMES)
def test_operands_near_the_smallest(gcg_lib, which, states):
    """One operand of a few denormals' size, the others large enough for results that are not."""
    t, gen = data(150, 3, 64, 48, 2, 8.0)
    t[which] = (2.0 ** -20 * torch.randn(t[which].shape, generator=gen, device=DEV)).half()
    ld = torch.tensor([-0.01, -0.003, -0.3], device=DEV)
    initial, dfinal = (2.0 ** -10 * torch.randn(1, 3, 64, 48, generator=gen, device=DEV) if states else None for _ in range(2))
    got = step(*(t[n] for n in NAMES), ld, 0.125, initial, dfinal)
    check(got, reference(t, ld, 0.125, initial, dfinal), f"small {which}")


@pytest.mark.parametrize("which", NAMES)
@pytest.mark.parametrize("L,H,dk,dv", [(200, 2, 64, 64), (200, 1, 256, 40), (2049, 2, 128, 64)])
def test_channels_of_different_size(gcg_lib, L, H, dk, dv, which):
    """Neighbouring channels of one operand 2^8 and 2^-11, the other operands 2^-3: each column of the result keeps its own precision."""
    t, gen = data(L, H, dk, dv, 3, 1.0)
    by = torch.where(torch.arange(t[which].shape[-1], device=DEV) % 3 == 0, 2.0 ** 8, 2.0 ** -11)
    for n in NAMES:
        t[n] = (t[n].float() * (by if n == which else 2.0 ** -3)).half()
    ld = torch.tensor([-0.01, -0.003], device=DEV)[:H].contiguous()
    got = step(*(t[n] for n in NAMES), ld, 0.125)
    check(got, reference(t, ld, 0.125, None, None), f"channels of {which}")


def test_a_column_without_finite_values_leaves_its_neighbours_alone(gcg_lib):
    """An infinity in one column of the given state, values beyond f16's largest in the others: those come out as without it."""
    t, gen = data(100, 2, 64, 64, 4, 2.0 ** -8)
    ld = torch.tensor([-0.01, -0.003], device=DEV)
    initial = 1e5 * torch.randn(1, 2, 64, 64, generator=gen, device=DEV)
    clean = linear_attention(t["q"], t["k"], t["v"], ld, initial_state=initial)
    initial[0, 1, 5, 7] = float("inf")
    o = linear_attention(t["q"], t["k"], t["v"], ld, initial_state=initial)
    others = [j for j in range(64) if j != 7]
    assert torch.isfinite(clean).all() and not torch.isfinite(o[0, :, 1, 7]).any()
    assert torch.equal(o[..., others], clean[..., others])
