"""Layer norm, 8-bit checkpoints and linear attention without a GPU: shapes of the meta implementations on fake tensors, refusals of
the Python layer, and argument errors of the C entry points, which come before the device is looked at."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from savanna_amd.operators.act8 import pack8, unpack8
from savanna_amd.operators.linear_attention import LinearAttention, linear_attention, linear_attention_features, linear_attention_step
from savanna_amd.operators.norm import LayerNorm, layer_norm

BAD_ARG, UNSUPPORTED, WORKSPACE = -1, -2, -3


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_meta_shapes_of_norm_and_checkpoint(gcg_lib, dtype):
    with FakeTensorMode():
        x = torch.empty(3, 7, 300, dtype=dtype, device="cuda")
        codes, scales = torch.ops.gcg.pack8(x)
        assert codes.shape == x.shape and codes.dtype == torch.int8
        assert scales.shape == (3, 7, 3) and scales.dtype == torch.float32          # blocks of 128: the last has 44
        back = torch.ops.gcg.unpack8(codes, scales, dtype)
        assert back.shape == x.shape and back.dtype == dtype
        w = torch.empty(300, dtype=dtype, device="cuda")
        for save in (False, True):
            y, stats, codes, scales = torch.ops.gcg.layer_norm_fwd(x, w, w, 1e-5, save)
            assert y.shape == x.shape and y.dtype == dtype and stats.numel() == 2 * 21 and stats.dtype == torch.float32
            assert (codes.numel() > 0) == save
        assert torch.ops.gcg.layer_norm_infer(x, w, None, 1e-5).shape == x.shape
        dx, dw, db = torch.ops.gcg.layer_norm_bwd(x, x, None, None, stats, w, w)
        assert dx.shape == x.shape and dx.dtype == dtype and dw.shape == db.shape == w.shape and dw.dtype == dtype


@pytest.mark.parametrize("dk,dv", [(64, 64), (33, 7), (256, 1)])
def test_meta_shapes_of_linear_attention(gcg_lib, dk, dv):
    with FakeTensorMode():
        q = torch.empty(2, 50, 3, dk, dtype=torch.bfloat16, device="cuda")
        v = torch.empty(2, 50, 3, dv, dtype=torch.bfloat16, device="cuda")
        ld = torch.empty(3, device="cuda")
        state = torch.empty(2, 3, dk, dv, device="cuda")
        o, final = torch.ops.gcg.linear_attn_fwd(q, q, v, ld, state, None, 0.5, True)
        assert o.shape == v.shape and o.dtype == v.dtype and final.shape == state.shape and final.dtype == torch.float32
        assert torch.ops.gcg.linear_attn_fwd(q, q, v, ld, None, None, 0.5, False)[1].numel() == 0
        dq, d_k, d_v, di = torch.ops.gcg.linear_attn_bwd(v, q, q, v, ld, state, None, None, 0.5, True)
        assert dq.shape == d_k.shape == q.shape and d_v.shape == v.shape and di.shape == state.shape
        assert torch.ops.gcg.linear_attn_step(q[:, 0], q[:, 0], v[:, 0], ld, state, 0.5).shape == (2, 3, dv)
        features = torch.empty(2, 50, 3 * 3 * dk, dtype=torch.float16, device="cuda")
        o = torch.ops.gcg.linear_attn_packed_fwd(features, 3, ld, 0.5)
        assert o.shape == (2, 50, 3, dk)
        assert torch.ops.gcg.linear_attn_packed_bwd(o, features, 3, ld, 0.5).shape == features.shape


def test_cpu_tensors_are_refused(gcg_lib):
    x, w = torch.randn(4, 64), torch.ones(64)
    q, ld = torch.randn(1, 5, 2, 8), torch.zeros(2)
    for call in (lambda: pack8(x), lambda: layer_norm(x, w, w), lambda: LayerNorm(64)(x), lambda: linear_attention(q, q, q, ld),
                 lambda: linear_attention_features(torch.randn(1, 5, 48), 2, ld),
                 lambda: linear_attention_step(q[:, 0], q[:, 0], q[:, 0], ld, torch.zeros(1, 2, 8, 8)),
                 lambda: unpack8(type("P", (), dict(codes=torch.zeros(4, 64, dtype=torch.int8), scales=torch.zeros(4, 1), dtype=torch.float32))())):
        with pytest.raises(Exception):
            call()


def test_decays_of_the_module(gcg_lib):
    """Memories from 8 to 4096 tokens, spread over the heads; no parameter."""
    mixer = LinearAttention(256, 8)
    memory = -1 / mixer.log_decay
    assert torch.allclose(memory[[0, -1]], torch.tensor([8.0, 4096.0])) and (memory[1:] > memory[:-1]).all()
    assert not list(mixer.parameters()) and "log_decay" in mixer.state_dict()
    with pytest.raises(RuntimeError, match="constant of the heads"):
        linear_attention(*[torch.zeros(1, 1, 8, 32)] * 3, mixer.log_decay.requires_grad_(True))


def ptr(n=1 << 20):
    return ctypes.c_void_p(n)           # (never followed: the calls below fail before anything is launched)


def test_c_entries_of_norm_and_checkpoint_refuse(gcg_lib):
    p, none = ptr(), None
    for rows, D, dtype in ((0, 64, 1), (4, 0, 1), (4, 64, 7), (-1, 64, 0)):
        assert gcg_lib.gcg_pack8(p, p, p, rows, D, dtype, none) == BAD_ARG
        assert gcg_lib.gcg_unpack8(p, p, p, rows, D, dtype, none) == BAD_ARG
    assert gcg_lib.gcg_pack8(none, p, p, 4, 64, 1, none) == BAD_ARG
    assert gcg_lib.gcg_unpack8(p, none, p, 4, 64, 1, none) == BAD_ARG


def attn(lib, dtype=1, bs=1, L=64, H=2, dk=64, dv=64, scale=1.0, strides=None, q=ptr(), ws=None, ws_bytes=0):
    s = strides or [L * H * 64, H * 64, 64] * 4
    return lib.gcg_linear_attn_fwd(q, ptr(), ptr(), (ctypes.c_int64 * 12)(*s), ptr(), None, None, ptr(), None, ws, ws_bytes, bs, L, H, dk, dv,
                                   scale, dtype, None)


@pytest.mark.parametrize("args,code", [
    (dict(q=None), BAD_ARG), (dict(L=0), BAD_ARG), (dict(bs=0), BAD_ARG), (dict(H=0), BAD_ARG), (dict(dk=0), BAD_ARG), (dict(dv=-8), BAD_ARG),
    (dict(dtype=9), BAD_ARG), (dict(scale=0.0), BAD_ARG), (dict(scale=float("inf")), BAD_ARG), (dict(scale=float("nan")), BAD_ARG),
    (dict(scale=1e-39), BAD_ARG), (dict(strides=[-1, 128, 64] * 4), BAD_ARG),
    (dict(dk=264), UNSUPPORTED), (dict(dv=60), UNSUPPORTED), (dict(dk=62, dtype=0), UNSUPPORTED), (dict(bs=65536), UNSUPPORTED),
    (dict(bs=300, H=300), UNSUPPORTED), (dict(L=(1 << 30) + 1), UNSUPPORTED), (dict(strides=[0, (1 << 22) + 1, 64] * 4), UNSUPPORTED),
    (dict(L=4096), WORKSPACE), (dict(L=4096, ws=ptr(), ws_bytes=256), WORKSPACE), (dict(L=4096, ws=ptr((1 << 20) + 8), ws_bytes=1 << 30), WORKSPACE),
])
def test_c_entry_of_linear_attention_refuses(gcg_lib, args, code):
    assert attn(gcg_lib, **args) == code


def test_workspaces(gcg_lib):
    """Segments only where few heads leave the card idle; sizes do not pass what 768 workgroups can take."""
    need = gcg_lib.gcg_linear_attn_workspace_bytes
    assert need(2, 8192, 32, 128, 128, 0) == 0 and need(1, 512, 1, 64, 64, 1) == 0
    assert need(0, 64, 2, 64, 64, 0) == 0 and need(1, 64, 2, 512, 64, 0) == 0
    for L in (2048, 4097, 131072, 1 << 24):
        for dk, dv in ((64, 64), (256, 8)):
            for backward in (0, 1):
                n = need(1, L, 1, dk, dv, backward)
                assert n % 256 == 0 and 0 < n <= 768 * 4 * dk * dv * 3


def test_operators_are_registered(gcg_lib):
    from savanna_amd import _ops

    assert set(_ops.BLOCK_NODE_NAMES) == {"layer_norm", "linear_attn", "linear_attn_packed"}
    for name in _ops.BLOCK_NODE_NAMES + _ops.BLOCK_OP_NAMES:
        assert hasattr(torch.ops.gcg, name), name
