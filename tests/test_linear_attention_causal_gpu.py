"""Infinities and NaN in rows that the causal mask hides: no row before them sees them, in the output or in a gradient, bit for bit."""
import pytest
import torch

from savanna_amd.operators.linear_attention import linear_attention
from test_linear_attention_gpu import DEV, TYPES, data, step

pytestmark = pytest.mark.gpu
ROWS = (0, 1, 15, 16, 17, 30, 31, 32, 47, 48, 63, 64, 100, 129)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128, 256, 40])
def test_rows_before_are_untouched(gcg_lib, d, dtype):
    """One element of v, then two of one column and one of another: rows before the first are those of the clean input, and so are the
    other columns everywhere."""
    q, k, v, _, _, _ = data(1, 130, 2, d, d, dtype, seed=d)
    ld = torch.tensor([-0.05, -0.002], device=DEV)
    clean = linear_attention(q, k, v, ld)
    for bad in (float("nan"), float("inf"), -float("inf")):
        for s in ROWS:
            u = v.clone()
            u[0, s, 1, 9] = bad
            o = linear_attention(q, k, u, ld)
            assert torch.equal(o[:, :s], clean[:, :s]) and torch.equal(o[:, :, 0], clean[:, :, 0]), (s, bad)
            assert not torch.isfinite(o[0, s:, 1, 9]).any(), (s, bad)
            others = [j for j in range(d) if j != 9]
            assert torch.equal(o[..., others], clean[..., others]), (s, bad)
    u = v.clone()
    u[0, 70, 0, 3], u[0, 75, 0, 3], u[0, 73, 0, 20] = float("nan"), float("inf"), float("inf")
    o = linear_attention(q, k, u, ld)
    assert torch.equal(o[:, :70], clean[:, :70]) and torch.equal(o[0, 70:73, 0, 20], clean[0, 70:73, 0, 20])
    assert not torch.isfinite(o[0, 70:, 0, 3]).any() and not torch.isfinite(o[0, 73:, 0, 20]).any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_gradients(gcg_lib, bad, dtype):
    """A row of do reaches the gradients of k and v at its own row and before, and of q at its own; a row of k the gradient of q from it
    on, of v at it and before it; a row of q likewise."""
    q, k, v, do, _, _ = data(1, 130, 2, 64, 64, dtype, seed=5)
    ld = torch.tensor([-0.05, -0.002], device=DEV)
    clean = step(q, k, v, do, ld)
    for s in ROWS:
        g = do.clone()
        g[0, s, 1, 9] = bad
        _, _, dq, dk, dv, _ = step(q, k, v, g, ld)
        assert torch.equal(dk[:, s + 1:], clean[3][:, s + 1:]) and torch.equal(dv[:, s + 1:], clean[4][:, s + 1:]), s
        assert torch.equal(dq[:, :s], clean[2][:, :s]) and not torch.isfinite(dv[0, :s + 1, 1, 9]).any(), s
        b = k.clone()
        b[0, s, 1, 9] = bad
        _, _, dq, dk, dv, _ = step(q, b, v, do, ld)
        assert torch.equal(dq[:, :s], clean[2][:, :s]) and not torch.isfinite(dq[0, s:, 1, 9]).any(), s
        assert torch.equal(dk, clean[3]) and torch.equal(dv[:, :s], clean[4][:, :s]) and torch.equal(dv[:, s + 1:], clean[4][:, s + 1:]), s
        a = q.clone()
        a[0, s, 1, 9] = bad
        _, _, dq, dk, dv, _ = step(a, k, v, do, ld)
        assert torch.equal(dk[:, s + 1:], clean[3][:, s + 1:]) and not torch.isfinite(dk[0, :s + 1, 1, 9]).any(), s
        assert torch.equal(dq, clean[2]) and torch.equal(dv[:, s + 1:], clean[4][:, s + 1:]), s
