"""Mixers and the layer around them with their activations kept in 8 bits: results do not change, nothing larger than the
checkpoint is kept, and gradients are bit for bit those of the same mixer on the checkpoint's values."""
import pytest
import torch

from savanna_amd.operators.act8 import pack8, unpack8
from savanna_amd.operators.block import MixerBlock
from savanna_amd.operators.hyena import CgcgConfig, HyenaMixer, HyenaMROperator, HyenaSEOperator
from savanna_amd.operators.linear_attention import LinearAttention

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def hyena(kind, types, planar, fused=True, g=6, dg=16):
    act, arith = types
    op = (HyenaMROperator(g * dg, g, 128, CgcgConfig(cgcg_dtype=arith), small_init=False, device=DEV) if kind == "mr"
          else HyenaSEOperator(g * dg, g, 7, CgcgConfig(cgcg_dtype=arith), device=DEV))
    return HyenaMixer(op, 3, dtype=act, device=DEV, fuse_short=fused, fuse_medium=fused, interleave_projections=not planar)


@pytest.mark.parametrize("kind", ["mr", "se"])
@pytest.mark.parametrize("types", [(torch.bfloat16, "bfloat16"), (torch.bfloat16, "float32"), (torch.float32, "float32")],
                         ids=["bf16", "bf16-f32", "f32"])
@pytest.mark.parametrize("planar,fused", [(False, True), (True, True), (False, False)])
def test_hyena_mixer(gcg_lib, kind, types, planar, fused):
    torch.manual_seed(1)
    mixer = hyena(kind, types, planar, fused)
    x = torch.randn(2, 333, 288, device=DEV).to(types[0])
    dy = torch.randn(2, 333, 96, device=DEV).to(types[0])
    params = list(mixer.parameters())

    def step(features, save_8bit):
        mixer.save_8bit = save_8bit
        features = features.detach().requires_grad_(True)
        y = mixer(features)
        return y, torch.autograd.grad(y, [features, *params], dy)

    y, got = step(x, True)
    assert torch.equal(y, step(x, False)[0])
    want = step(unpack8(pack8(x)), False)[1]
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.no_grad():
        assert torch.equal(mixer(x), y)


@pytest.mark.parametrize("kind", ["mr", "se"])
@pytest.mark.parametrize("fused", [False, True])
def test_frozen_parameters_and_lengths_of_zero_and_one(gcg_lib, kind, fused):
    torch.manual_seed(4)
    mixer = hyena(kind, (torch.bfloat16, "bfloat16"), False, fused)
    frozen = mixer.hyena_proj_conv.short_conv_weight.requires_grad_(False)
    params = [p for p in mixer.parameters() if p is not frozen]
    for L in (1, 5):
        x = torch.randn(2, L, 288, device=DEV).to(torch.bfloat16)
        dy = torch.randn(2, L, 96, device=DEV).to(torch.bfloat16)
        grads = []
        for mixer.save_8bit, at in ((True, x), (False, unpack8(pack8(x)))):
            at = at.detach().requires_grad_(True)
            grads.append(torch.autograd.grad(mixer(at), [at, *params], dy))
        assert all(torch.equal(a, b) for a, b in zip(*grads))
    mixer.save_8bit = True
    empty = torch.empty(0, 5, 288, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    plain = empty.detach().requires_grad_(True)
    got = mixer(empty)
    mixer.save_8bit = False
    assert got.shape == mixer(plain).shape


def test_kept_bytes(gcg_lib):
    """From forward to backward a mixer keeps 1.03 bytes an element of its features, and its parameters."""
    torch.manual_seed(2)
    for mixer in (hyena("mr", (torch.bfloat16, "bfloat16"), False, g=32), LinearAttention(512, 8, device=DEV)):
        x = torch.randn(2, 1024, 1536, device=DEV).to(torch.bfloat16).requires_grad_(True)
        kept = {}
        for mixer.save_8bit in (False, True):
            def pack(t):
                kept.setdefault(mixer.save_8bit, []).append(t)
                return t
            with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
                mixer(x)
        size = lambda ts: sum(t.numel() * t.element_size() for t in ts if t.numel() >= x.numel() // 128)       # noqa: E731
        assert size(kept[False]) >= 2 * x.numel()
        assert size(kept[True]) <= 1.04 * x.numel()


def test_block_trains_and_decodes(gcg_lib):
    """The layer's gradients in 8 bits stay near the exact ones, and decoding continues a prompt as the whole sequence does."""
    torch.manual_seed(3)
    x = torch.randn(2, 200, 128, device=DEV)
    dy = torch.randn(2, 200, 128, device=DEV)
    for make in (lambda: hyena("mr", (torch.float32, "float32"), False, g=8), lambda: LinearAttention(128, 2, device=DEV)):
        block = MixerBlock(128, make(), device=DEV)
        params = list(block.parameters())
        grads = {}
        for bits8 in (False, True):
            block.mixer.save_8bit = block.norm.save_8bit = bits8
            X = x.clone().requires_grad_(True)
            grads[bits8] = torch.autograd.grad(block(X), [X, *params], dy)
        for a, b in zip(grads[True], grads[False]):
            # a value is at most 1/254 of its block's largest off, 2 % of a normal value's own size; its errors are independent
            assert (a - b).norm() <= 0.04 * b.norm()
    with torch.no_grad():
        whole = block(x)
        y, state = block.prefill(x[:, :150])
        rest = torch.stack([block.step(x[:, t], state) for t in range(150, 200)], 1)
        assert (torch.cat([y, rest], 1) - whole).abs().max() <= 1e-4 * whole.abs().max()
        n = torch.tensor([200, 70], dtype=torch.int32, device=DEV)
        y, state = block.prefill(x, lengths=n)
        _, short = block.prefill(x[1:, :70])
        assert torch.equal(state[1], short[0]) and (y[1, :70] - whole[1, :70]).abs().max() <= 1e-4 * whole.abs().max()
    with pytest.raises(RuntimeError, match="carries no state"):
        MixerBlock(96, hyena("se", (torch.float32, "float32"), False), device=DEV).prefill(x)


def test_schemas_and_meta_results(gcg_lib):
    from savanna_amd import _ops

    r = lambda *s: torch.randn(*s, device=DEV).to(torch.bfloat16)                   # noqa: E731
    ld, state = torch.tensor([-0.1, -0.01], device=DEV), torch.randn(1, 2, 16, 24, device=DEV)
    x, w, q, v, features = r(5, 96), r(96), r(1, 70, 2, 16), r(1, 70, 2, 24), r(1, 70, 96)
    codes, scales = torch.ops.gcg.pack8(x)
    _, stats, _, _ = torch.ops.gcg.layer_norm_fwd(x, w, w, 1e-5, False)
    nodes = {"layer_norm": (x, w, w, 1e-5, True), "linear_attn": (q, q, v, ld, state, None, 0.25, True),
             "linear_attn_packed": (features, 2, ld, 0.25, True)}
    entries = {"pack8": (x,), "unpack8": (codes, scales, x.dtype), "layer_norm_fwd": (x, w, w, 1e-5, True), "layer_norm_infer": (x, w, None, 1e-5),
               "layer_norm_bwd": (x, None, codes, scales, stats, w, w), "linear_attn_fwd": (q, q, v, ld, state, None, 0.25, True),
               "linear_attn_bwd": (v, q, q, v, ld, state, None, None, 0.25, True), "linear_attn_packed_fwd": (features, 2, ld, 0.25),
               "linear_attn_packed_bwd": (r(1, 70, 2, 16), features, 2, ld, 0.25),
               "linear_attn_step": (q[:, 0], q[:, 0], v[:, 0], ld, state, 0.25)}
    assert set(nodes) == set(_ops.BLOCK_NODE_NAMES) and set(entries) == set(_ops.BLOCK_OP_NAMES)
    for name, a in {**nodes, **entries}.items():
        torch.library.opcheck(getattr(torch.ops.gcg, name), a, test_utils=("test_schema", "test_faketensor"))
