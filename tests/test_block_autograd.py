"""What autograd sees of the operators around the convolution, without a GPU: the state that a step moves on in place."""
import pytest
import torch


def meta(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="meta")


def token(state, ld=None):
    q = meta(2, 3, 16)
    return torch.ops.gcg.linear_attn_step(q, q, meta(2, 3, 8), meta(3, dtype=torch.float32) if ld is None else ld, state, 0.25)


def test_a_step_counts_as_a_change_of_the_state(gcg_lib):
    """A state that a recorded call keeps for its backward must not be moved on before that, and torch says so; a view's base counts too."""
    state = meta(2, 3, 16, 8, dtype=torch.float32)
    for n in range(1, 3):
        assert token(state).shape == (2, 3, 8)
        assert state._version == n
    base = meta(4, 3, 16, 8, dtype=torch.float32)
    token(base[1:3])
    assert base._version == 1
    x = meta(2, 3, 16, 8, dtype=torch.float32).requires_grad_(True)
    kept = state * x                    # (keeps both for its backward)
    with torch.no_grad():
        token(state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        kept.sum().backward()


def test_a_step_on_inference_tensors(gcg_lib):
    """Inside inference mode and, as nothing can have kept such a state, after it."""
    with torch.inference_mode():
        state = meta(2, 3, 16, 8, dtype=torch.float32)
        assert token(state).is_inference()
    with torch.no_grad():
        assert token(state).shape == (2, 3, 8)
