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


# ---- a module run again in the backward on its input's checkpoint -------------------------------------------

class Scaled(torch.nn.Module):
    """y = x w s, with a parameter that nothing uses."""

    def __init__(self):
        super().__init__()
        self.w = torch.nn.Parameter(torch.tensor([1.0, 2.0]))
        self.idle = torch.nn.Parameter(torch.zeros(2))
        self.register_buffer("s", torch.tensor([3.0, 3.0]))

    def forward(self, x):
        return x * self.w * self.s


class Holder(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.inner = Scaled()

    def forward(self, x):
        from savanna_amd.operators import hyena
        return hyena._recomputed8(self.inner, x)


@pytest.fixture
def exact_checkpoint(monkeypatch):
    """The checkpoint as a copy, so that gradients have values to compare with."""
    from savanna_amd import _lib
    monkeypatch.setattr(_lib, "pack8", lambda x: (x.clone(), torch.ones(1)))
    monkeypatch.setattr(_lib, "unpack8", lambda codes, scales, dtype: codes.clone())


def test_recomputation_sees_the_parameters_of_its_forward(exact_checkpoint):
    """Substituted by functional_call, parameters and buffers alike: gradients are theirs, at their values."""
    m = Holder()
    x = torch.tensor([10.0, 20.0], requires_grad=True)
    w = torch.tensor([5.0, 7.0], requires_grad=True)
    y = torch.func.functional_call(m, {"inner.w": w, "inner.s": torch.tensor([1.0, 2.0])}, (x,))
    dx, dw = torch.autograd.grad(y.sum(), [x, w])
    assert torch.equal(dx, torch.tensor([5.0, 14.0])) and torch.equal(dw, torch.tensor([10.0, 40.0]))
    y = m(x)
    dx, dw, idle = torch.autograd.grad(y.sum(), [x, m.inner.w, m.inner.idle], allow_unused=True)
    assert torch.equal(dx, torch.tensor([3.0, 6.0])) and torch.equal(dw, torch.tensor([30.0, 60.0])) and idle is None
    m.inner.w.requires_grad_(False)
    m(x).sum().backward()
    assert torch.equal(x.grad, torch.tensor([3.0, 6.0])) and m.inner.w.grad is None


def test_recomputation_under_saved_tensor_hooks(exact_checkpoint):
    """Hooks hand back other tensors than were saved (offloading, checkpointing): the gradients are the same."""
    m, x = Holder(), torch.tensor([10.0, 20.0], requires_grad=True)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(), lambda t: t):
        y = m(x)
    dx, dw = torch.autograd.grad(y.sum(), [x, m.inner.w])
    assert torch.equal(dx, torch.tensor([3.0, 6.0])) and torch.equal(dw, torch.tensor([30.0, 60.0]))
    y = torch.utils.checkpoint.checkpoint(m, x, use_reentrant=False)
    dx, dw = torch.autograd.grad(y.sum(), [x, m.inner.w])
    assert torch.equal(dx, torch.tensor([3.0, 6.0])) and torch.equal(dw, torch.tensor([30.0, 60.0]))


def test_recomputation_notices_changed_parameters(exact_checkpoint):
    m, x = Holder(), torch.tensor([10.0, 20.0], requires_grad=True)
    y = m(x)
    with torch.no_grad():
        m.inner.w.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


# ---- forward mode ---------------------------------------------------------------------------------------------

@pytest.mark.parametrize("grad", [False, True])
def test_tangents_are_refused_not_dropped(gcg_lib, grad):
    """None of the operators has a forward-mode derivative: inputs with tangents raise, with gradients recorded or not, and inputs without
    pass inside a level too."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.autograd import forward_ad

    from savanna_amd import _lib
    from savanna_amd.operators.linear_attention import linear_attention, linear_attention_features, linear_attention_step
    from savanna_amd.operators.norm import layer_norm

    with FakeTensorMode(), torch.set_grad_enabled(grad), forward_ad.dual_level():
        x, q, f = (torch.empty(*s, device="cuda") for s in ((4, 64), (1, 5, 2, 8), (1, 5, 48)))
        ld, state = torch.empty(2, device="cuda"), torch.empty(1, 2, 8, 8, device="cuda")
        t = q[:, 0]
        calls = [(lambda x: layer_norm(x), x), (lambda x: layer_norm(x, save_8bit=True), x), (lambda w: layer_norm(x, w), x[0]),
                 (lambda q: linear_attention(q, q, q, ld), q), (lambda s: linear_attention(q, q, q, ld, initial_state=s), state),
                 (lambda f: linear_attention_features(f, 2, ld), f), (lambda t: linear_attention_step(t, t, t, ld, state), t),
                 (lambda s: linear_attention_step(t, t, t, ld, s), state), (lambda x: _lib.layer_norm_fwd(x, None, None, 1e-5), x),
                 (lambda q: _lib.linear_attn_fwd(q, q, q, ld, None, None, 1.0, False), q)]
        for call, at in calls:
            call(at)
            with pytest.raises(NotImplementedError):
                call(forward_ad.make_dual(at, torch.empty_like(at)))


# ---- the decays -------------------------------------------------------------------------------------------------

def test_operators_refuse_a_gradient_of_the_decays(gcg_lib):
    """The registered operators as the Python layer does, and only where gradients are recorded."""
    ops = torch.ops.gcg
    ld = meta(3, dtype=torch.float32).requires_grad_(True)
    q, v, features = meta(2, 50, 3, 16), meta(2, 50, 3, 8), meta(2, 50, 144)
    calls = [lambda ld: ops.linear_attn(q, q, v, ld, None, None, 0.5, True)[0], lambda ld: ops.linear_attn_fwd(q, q, v, ld, None, None, 0.5, False)[0],
             lambda ld: ops.linear_attn_packed(features, 3, ld, 0.5, False), lambda ld: ops.linear_attn_packed_fwd(features, 3, ld, 0.5)]
    for q_grad in (False, True):
        q.requires_grad_(q_grad)
        features.requires_grad_(q_grad)
        for call in calls:
            with pytest.raises(RuntimeError, match="constant of the heads"):
                call(ld)
            assert call(ld.detach()).requires_grad == q_grad
            with torch.no_grad():
                assert not call(ld).requires_grad


# ---- the norm's gradients ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("need_dw,need_db", [(True, True), (True, False), (False, True), (False, False)])
def test_the_norms_backward_forms_what_is_needed(gcg_lib, need_dw, need_db):
    x, w, stats = meta(5, 96), meta(96), meta(5, 2, dtype=torch.float32)
    dx, dw, db = torch.ops.gcg.layer_norm_bwd(x, x, None, None, stats, w, w, need_dw, need_db)
    assert dx.shape == x.shape and dw.numel() == 96 * need_dw and db.numel() == 96 * need_db


@pytest.mark.parametrize("D", [16385, 2 ** 32 + 64])
def test_rows_wider_than_the_norm_takes(gcg_lib, D):
    """Refused by every form, traced ones too; a width is not taken modulo 2^32."""
    x, w, stats = meta(2, D), meta(D), meta(2, 2, dtype=torch.float32)
    for call in (lambda: torch.ops.gcg.layer_norm_fwd(x, w, None, 1e-5, False), lambda: torch.ops.gcg.layer_norm_infer(x, None, None, 1e-5),
                 lambda: torch.ops.gcg.layer_norm_bwd(x, x, None, None, stats, None, None)):
        with pytest.raises(RuntimeError, match="at most 16384"):
            call()


def test_more_heads_than_an_int_holds(gcg_lib):
    """Refused with its number, not taken modulo 2^32."""
    H = 2 ** 32 + 1
    q, ld = torch.empty(1, 1, H, 8, device="meta"), torch.empty(H, device="meta")
    with pytest.raises(RuntimeError, match="heads; at most"):
        torch.ops.gcg.linear_attn_fwd(q, q, q, ld, None, None, 1.0, False)


# ---- tensors that are not on the GPU ----------------------------------------------------------------------------

@pytest.mark.parametrize("call", ["pack8", "unpack8", "layer_norm", "LayerNorm", "linear_attention", "linear_attention_features",
                                  "linear_attention_step"])
@pytest.mark.parametrize("grad", [False, True])
def test_cpu_tensors_are_refused_by_name(gcg_lib, call, grad):
    from savanna_amd.operators.act8 import Packed8, pack8, unpack8
    from savanna_amd.operators.linear_attention import linear_attention, linear_attention_features, linear_attention_step
    from savanna_amd.operators.norm import LayerNorm, layer_norm

    x, q, ld = torch.randn(4, 64), torch.randn(1, 5, 2, 8), torch.zeros(2)
    calls = {"pack8": lambda: pack8(x), "unpack8": lambda: unpack8(Packed8(torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4, 1), x.dtype)),
             "layer_norm": lambda: layer_norm(x, torch.ones(64)), "LayerNorm": lambda: LayerNorm(64)(x),
             "linear_attention": lambda: linear_attention(q, q, q, ld),
             "linear_attention_features": lambda: linear_attention_features(torch.randn(1, 5, 48), 2, ld),
             "linear_attention_step": lambda: linear_attention_step(q[:, 0], q[:, 0], q[:, 0], ld, torch.zeros(1, 2, 8, 8))}
    with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="no CPU path"):
        calls[call]()
