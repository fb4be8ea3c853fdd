"""Single tokens of linear attention where they are many, against the recurrence in 64 bits."""
import pytest
import torch

from savanna_amd import _lib
from savanna_amd.operators.linear_attention import linear_attention, linear_attention_step
from test_linear_attention_gpu import DEV

pytestmark = pytest.mark.gpu


def test_thousands_of_tokens(gcg_lib):
    """The decay of every token is kept to more than fp32's 24 bits, as over the rows of a prompt: its rounding, the same way each time,
    would add up.  A state is off by 2^-17 of its terms' magnitudes, an output by one rounding more."""
    H, d, n = 3, 8, 8192
    gen = torch.Generator(device=DEV).manual_seed(6)
    q, k, v = (0.5 + 0.5 * torch.rand(n, 1, H, d, generator=gen, device=DEV) for _ in range(3))        # (of one sign: nothing cancels)
    ld = torch.tensor([-1.0 / 4096, -1.0 / 3000, -1e-5], device=DEV)
    state = 4 * torch.randn(1, H, d, d, generator=gen, device=DEV)
    f = torch.exp(ld.double())[:, None, None]
    S, A = state.double(), state.double().abs()
    with torch.no_grad():
        for t in range(n):
            o = linear_attention_step(q[t], k[t], v[t], ld, state, 0.5)
            S = f * S + k[t].double()[..., None] * v[t].double()[..., None, :]
            A = f * A + k[t].double().abs()[..., None] * v[t].double().abs()[..., None, :]
    assert ((state.double() - S).abs() <= 2.0 ** -17 * A).all()
    want, terms = ((x[..., None] * y).sum(-2) * 0.5 for x, y in ((q[-1].double(), S), (q[-1].double().abs(), A)))
    assert ((o.double() - want).abs() <= 2.0 ** -16 * terms).all()


def test_a_state_kept_for_a_backward_is_not_moved_on_unseen(gcg_lib):
    """A recorded sequence that began from a state, the state then moved on: its backward would form dq from another state, and raises."""
    gen = torch.Generator(device=DEV).manual_seed(7)
    q, k, v = (torch.randn(2, 5, 3, 16, generator=gen, device=DEV) for _ in range(3))
    ld = torch.tensor([-0.1, -0.01, 0.0], device=DEV)
    state = torch.randn(2, 3, 16, 16, generator=gen, device=DEV)
    o = linear_attention(q.requires_grad_(True), k, v, ld, initial_state=state)
    with torch.no_grad():
        linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, state.clone())
    torch.autograd.grad(o.sum(), q, retain_graph=True)
    with torch.no_grad():
        linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(o.sum(), q)
    with torch.inference_mode():
        prompt, state = linear_attention(q, k, v, ld, output_final_state=True)
        linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, state)
    with torch.no_grad():
        assert linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, state).shape == (2, 3, 16)


@pytest.mark.skipif(not _lib.TORCH_OPS, reason="the ctypes binding is not traced")
def test_a_step_traced(gcg_lib):
    """Through torch.compile the step gives the same bits and moves the same state on, and counts as a change of it."""
    gen = torch.Generator(device=DEV).manual_seed(8)
    q, k, v = (torch.randn(2, 3, 16, generator=gen, device=DEV) for _ in range(3))
    ld = torch.tensor([-0.1, -0.01, 0.0], device=DEV)
    state = torch.randn(2, 3, 16, 16, generator=gen, device=DEV)
    traced = torch.compile(lambda q, k, v, s: linear_attention_step(q, k, v, ld, s) * 2, fullgraph=True, backend="aot_eager")
    ours = state.clone()
    with torch.no_grad():
        for _ in range(3):
            version = state._version
            assert torch.equal(traced(q, k, v, state), linear_attention_step(q, k, v, ld, ours) * 2) and torch.equal(state, ours)
            assert state._version > version
