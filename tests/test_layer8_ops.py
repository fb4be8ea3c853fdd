"""Root-mean-square norm, 8-bit floating point and gated recurrence without a GPU: shapes of the meta implementations on fake tensors, refusals of the
Python layer, and argument errors of the C entry points, which come before the device is looked at."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from savanna_amd import _lib, _ops
from savanna_amd.operators.block import MixerBlock, MixerBlockFloat8
from savanna_amd.operators.float8 import E4M3, E5M2, Float8, LinearFloat8, from_float8, linear_float8, matmul_float8, norm_linear_float8, to_float8
from savanna_amd.operators.gated_recurrence import GatedRecurrence, gated_recurrence, gated_recurrence_features, gated_recurrence_step
from savanna_amd.operators.norm import RMSNorm, rms_norm, rms_norm_float8

BAD_ARG, UNSUPPORTED, WORKSPACE = -1, -2, -3


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_meta_shapes(gcg_lib, dtype):
    ops = torch.ops.gcg
    with FakeTensorMode():
        x, w = torch.empty(3, 7, 300, dtype=dtype, device="cuda"), torch.empty(300, dtype=dtype, device="cuda")
        for res in (None, x):
            y, r, rstd = ops.rms_norm_fwd(x, res, w, 1e-6)
            assert y.shape == x.shape and y.dtype == dtype and rstd.shape == (3, 7) and rstd.dtype == torch.float32
            assert r.shape == (x.shape if res is not None else (0,)) and ops.rms_norm_infer(x, res, w, 1e-6)[1].shape == r.shape
            codes, scales, r, rstd = ops.rms_norm_float8(x, res, w, 1e-6)
            assert codes.shape == (3, 7, 384) and codes.dtype == E4M3 and scales.shape == (3, 7, 4) and scales.dtype == torch.float8_e8m0fnu
        dx, dw = ops.rms_norm_bwd(x, x, x, rstd, w)
        assert dx.shape == x.shape and dw.shape == w.shape and ops.rms_norm_bwd(x, x, None, rstd, None)[1].numel() == 0
        m = torch.empty(70, 600, dtype=dtype, device="cuda")
        for fmt in (E4M3, E5M2):
            codes, scales = ops.to_float8(m, fmt)
            assert codes.shape == (70, 640) and codes.dtype == fmt and scales.shape == (70, 8)
            a, b, c, d = ops.to_float8_both(m, fmt)
            assert a.shape == codes.shape and c.shape == (600, 128) and d.shape == (600, 4) and ops.to_float8_columns(m, fmt)[0].shape == c.shape
            assert ops.float8_columns(codes, scales, 600, E4M3)[0].shape == (600, 128)
            assert ops.from_float8(codes, scales, 600, dtype).shape == (70, 600)
            if dtype != torch.float32:
                y = ops.matmul_float8(codes, scales, codes, scales, 600, dtype)
                assert [t.shape for t in ops.norm_linear_float8_infer(m, m, None, codes, scales, 600, 1e-6)] == [(70, 70), (70, 600)]
                assert y.shape == (70, 70) and y.dtype == dtype and ops.linear_float8_infer(m, codes, scales, 600).shape == (70, 70)
        f = torch.empty(2, 200, 30, dtype=dtype, device="cuda")
        bias, state = torch.empty(10, device="cuda"), torch.empty(2, 10, device="cuda")
        y, states = ops.scan_packed_fwd(f, bias, True)
        assert y.shape == (2, 200, 10) and states.shape == (2, 4, 10) and states.dtype == torch.float32
        df, db = ops.scan_packed_bwd(y, f, bias, states, True)
        assert df.shape == f.shape and db.shape == (10,)
        x = torch.empty(2, 200, 10, dtype=dtype, device="cuda")
        y, last, states = ops.scan_fwd(x, x, x, bias, state, None, True, False)
        assert last.shape == (2, 10) and states.numel() == 0
        out = ops.scan_bwd(x, x, x, None, None, torch.empty(2, 4, 10, device="cuda"), None, None, False, True)
        assert [t.shape for t in out] == [x.shape, x.shape, (0,), (0,), (2, 10)]
        assert ops.scan_step(x[:, 0], x[:, 0], None, bias, state).shape == (2, 10)


def test_operators_are_registered():
    for name in _ops.LAYER8_OP_NAMES + _ops.LAYER8_NODE_NAMES:
        assert hasattr(torch.ops.gcg, name), name


def test_cpu_tensors_are_refused(gcg_lib):
    x, w = torch.randn(4, 64).bfloat16(), torch.randn(8, 64).bfloat16()
    s = torch.randn(1, 5, 8)
    q = Float8(torch.zeros(4, 128).to(E4M3), torch.ones(4, 4).to(torch.float8_e8m0fnu), 64)
    for call in (lambda: rms_norm(x), lambda: RMSNorm(64, dtype=torch.bfloat16)(x, x), lambda: rms_norm_float8(x), lambda: to_float8(x),
                 lambda: from_float8(q, torch.float32), lambda: matmul_float8(q, q), lambda: linear_float8(x, w), lambda: linear_float8(x.detach(), q),
                 lambda: norm_linear_float8(x, None, w), lambda: LinearFloat8(64, 8)(x), lambda: gated_recurrence(s, s),
                 lambda: gated_recurrence_features(torch.randn(1, 5, 24)), lambda: gated_recurrence_step(s[:, 0], s[:, 0], torch.zeros(1, 8)),
                 lambda: GatedRecurrence(8)(torch.randn(1, 5, 24))):
        with pytest.raises(RuntimeError, match="MI355X"):
            call()


def test_python_refusals(gcg_lib):
    x, w = torch.randn(4, 64), torch.randn(8, 64)
    with pytest.raises(TypeError, match="bfloat16 or float16"):
        linear_float8(x, w)
    with pytest.raises(ValueError, match="dtype and device"):
        linear_float8(x.half(), w.bfloat16())
    with pytest.raises(TypeError, match="float8_e4m3fn or float8_e5m2"):
        linear_float8(x.half(), w.half(), torch.int8)
    q = Float8(torch.zeros(8, 128).to(E4M3), torch.ones(8, 4).to(torch.float8_e8m0fnu), 64)
    with pytest.raises(RuntimeError, match="not differentiable"):
        linear_float8(x.half().requires_grad_(True), q)
    with pytest.raises(ValueError, match="columns"):
        matmul_float8(q, Float8(q.codes, q.scales, 65))
    with pytest.raises(RuntimeError, match="not differentiable"):
        gated_recurrence_step(x.requires_grad_(True), x, torch.zeros(4, 64))
    with pytest.raises(ValueError, match="save_8bit"):
        MixerBlock(8, GatedRecurrence(8), save_8bit=True)
    assert MixerBlock(8, GatedRecurrence(8)).mixer.hidden_size == 8


def test_modules_on_the_host():
    m = GatedRecurrence(256)
    memory = torch.exp(m.decay_bias.detach())
    assert torch.allclose(memory[[0, -1]], torch.tensor([8.0, 4096.0])) and (memory[1:] > memory[:-1]).all()
    assert m.to(torch.bfloat16).decay_bias.dtype == torch.float32 and [n for n, _ in m.named_parameters()] == ["decay_bias"]
    block = MixerBlockFloat8(64, GatedRecurrence(64))
    assert block.projection.weight.shape == (192, 64) and block.projection.weight.dtype == torch.bfloat16
    assert sorted(n for n, _ in block.named_parameters()) == ["mixer.decay_bias", "norm.weight", "out.weight", "projection.weight"]
    from savanna_amd.operators.hyena import HyenaMixer
    with pytest.raises(RuntimeError, match="carries no state"):
        MixerBlockFloat8(64, HyenaMixer.__new__(HyenaMixer)).__class__.prefill(
            type("B", (), {"mixer": object(), "_features": lambda self, x, r: (x, r), "out": None})(), torch.zeros(1, 1, 1))


def ptr(n=1 << 20):
    return ctypes.c_void_p(n)           # (never followed: the calls below fail before anything is launched)


def test_c_entries_of_the_norm_refuse(gcg_lib):
    p, none = ptr(), None
    fwd = lambda *a, rows=4, D=64, eps=1e-6, dtype=0: gcg_lib.gcg_rms_norm_fwd(*a, rows, D, eps, dtype, none)                  # noqa: E731
    ok = [p, none, none, p, none, none, none, none]
    assert fwd(none, *ok[1:]) == BAD_ARG                                        # x
    assert fwd(p, p, none, p, none, none, none, none) == BAD_ARG                # a residual without r
    assert fwd(p, none, none, p, none, p, none, none) == BAD_ARG                # codes without scales
    assert fwd(p, none, none, p, none, p, p, none) == BAD_ARG                   # both outputs
    assert fwd(p, none, none, none, none, ptr((1 << 20) + 8), p, none) == BAD_ARG     # codes off 16 bytes
    assert fwd(*ok, rows=0) == fwd(*ok, D=0) == fwd(*ok, dtype=5) == fwd(*ok, eps=float("nan")) == fwd(*ok, eps=-1.0) == BAD_ARG
    assert fwd(*ok, D=16385) == UNSUPPORTED
    bwd = lambda *a, ws=none, n=0, D=64: gcg_lib.gcg_rms_norm_bwd(*a, ws, n, 4, D, 0, none)                                    # noqa: E731
    assert bwd(none, p, none, p, none, p, none) == bwd(p, none, none, p, none, p, none) == bwd(p, p, none, none, none, p, none) == BAD_ARG
    assert bwd(p, p, none, p, p, p, p) == WORKSPACE and bwd(p, p, none, p, p, p, p, ws=ptr((1 << 20) + 128), n=1 << 20) == WORKSPACE
    assert bwd(p, p, none, p, none, p, none, D=20000) == UNSUPPORTED
    assert gcg_lib.gcg_rms_norm_bwd_workspace_bytes(4, 64, 0) % 256 == 0 < gcg_lib.gcg_rms_norm_bwd_workspace_bytes(4, 64, 0)
    assert gcg_lib.gcg_rms_norm_bwd_workspace_bytes(0, 64, 0) == 0


def test_c_entries_of_float8_refuse(gcg_lib):
    p, none, odd = ptr(), None, ptr((1 << 20) + 2)
    for entry in (gcg_lib.gcg_to_float8, gcg_lib.gcg_from_float8):
        assert entry(none, p, p, 4, 64, 0, 16, none) == entry(p, none, p, 4, 64, 0, 16, none) == entry(p, p, none, 4, 64, 0, 16, none) == BAD_ARG
        assert entry(p, p, p, 0, 64, 0, 16, none) == entry(p, p, p, 4, 0, 0, 16, none) == entry(p, p, p, 4, 64, 3, 16, none) == BAD_ARG
        assert entry(p, p, p, 4, 64, 0, 15, none) == entry(p, p, p, 4, 64, 16, 16, none) == BAD_ARG
    assert gcg_lib.gcg_to_float8(p, odd, p, 4, 64, 0, 16, none) == gcg_lib.gcg_to_float8(p, p, odd, 4, 64, 0, 16, none) == BAD_ARG
    cols = lambda *a, rows=4, D=64, dtype=0, fmt=16: gcg_lib.gcg_to_float8_columns(*a, rows, D, dtype, fmt, none)              # noqa: E731
    assert cols(none, none, none, none, p, p) == cols(p, none, none, none, none, p) == cols(p, none, p, none, p, p) == BAD_ARG
    assert cols(p, p, p, p, p, p, dtype=16) == BAD_ARG                          # 8 bits along the rows again
    assert cols(p, p, none, none, p, p, dtype=0) == cols(p, none, none, none, p, p, dtype=16) == cols(p, none, none, none, p, p, fmt=0) == BAD_ARG
    mul = lambda *a, M=4, N=4, K=64, fa=16, fb=16, dtype=1, ws=none, n=0: gcg_lib.gcg_product8(*a, ws, n, M, N, K, fa, fb, dtype, none)   # noqa: E731
    for i in range(5):
        assert mul(*[none if i == j else p for j in range(5)]) == BAD_ARG
    ok = [p] * 5
    assert mul(*ok, M=0) == mul(*ok, N=-1) == mul(*ok, K=0) == mul(*ok, fa=0) == mul(*ok, fb=18) == mul(*ok, dtype=0) == mul(odd, *ok[1:]) == BAD_ARG
    assert mul(*ok, K=(1 << 22) + 1) == UNSUPPORTED
    need = gcg_lib.gcg_product8_workspace_bytes(65, 64, 16384)
    assert need > 0 and need % 256 == 0 and mul(*ok, M=65, N=64, K=16384) == WORKSPACE and gcg_lib.gcg_product8_workspace_bytes(4096, 4096, 4096) == 0
    assert gcg_lib.gcg_product8_workspace_bytes(1, 1, (1 << 22) + 1) == 0
    few = lambda *a, M=1, N=64, K=4096, fb=16, dtype=1: gcg_lib.gcg_linear8(*a, M, N, K, fb, dtype, none)                      # noqa: E731
    for i in range(4):
        assert few(*[none if i == j else p for j in range(4)]) == BAD_ARG
    assert few(p, p, p, p, M=0) == few(p, p, p, p, fb=1) == few(p, p, p, p, dtype=0) == BAD_ARG
    assert few(p, p, p, p, M=17, K=64) == few(p, p, p, p, M=5) == few(p, p, p, p, K=16385) == UNSUPPORTED
    assert gcg_lib.gcg_linear8_supported(4, 1, 4096) == 1 and gcg_lib.gcg_linear8_supported(5, 1, 4096) == gcg_lib.gcg_linear8_supported(0, 1, 1) == 0


def test_c_entries_of_the_recurrence_refuse(gcg_lib):
    p, none = ptr(), None
    strides = lambda n, time=64, batch=640: (ctypes.c_int64 * (2 * n))(*[batch, time] * n)                                     # noqa: E731
    fwd = lambda x=p, f=p, s=None, y=p, ws=none, n=0, bs=2, L=10, D=64, dtype=0: gcg_lib.gcg_scan_fwd(                         # noqa: E731
        x, f, none, s if s is not None else strides(4), none, none, none, y, none, none, ws, n, bs, L, D, dtype, none)
    assert fwd(x=none) == fwd(f=none) == fwd(y=none) == BAD_ARG
    assert fwd(bs=0) == fwd(L=0) == fwd(D=0) == fwd(dtype=3) == fwd(s=strides(4, time=-1)) == fwd(s=strides(4, batch=-1)) == BAD_ARG
    assert fwd(D=(1 << 19) + 1) == fwd(s=strides(4, time=(1 << 21) + 1)) == fwd(L=(1 << 30) + 1) == fwd(bs=1 << 31) == UNSUPPORTED
    assert gcg_lib.gcg_scan_workspace_bytes(2, 256, 64, 0) == 0 and fwd(L=257) == WORKSPACE
    need = gcg_lib.gcg_scan_workspace_bytes(2, 257, 64, 0)
    assert need % 256 == 0 and fwd(L=257, ws=ptr((1 << 20) + 64), n=need) == WORKSPACE and fwd(L=257, ws=p, n=need - 1) == WORKSPACE
    bwd = lambda *a, s=None, gate=none, dgate=none, L=10, D=64: gcg_lib.gcg_scan_bwd(                                          # noqa: E731
        a[0], a[1], a[2], gate, s if s is not None else strides(7), none, a[3], none, none, a[4], a[5], dgate, none, none, none, 0, 2, L, D, 0, none)
    for i in range(6):
        assert bwd(*[none if i == j else p for j in range(6)]) == BAD_ARG
    ok = [p] * 6
    assert bwd(*ok, gate=p) == bwd(*ok, dgate=p) == BAD_ARG and bwd(*ok) == WORKSPACE and bwd(*ok, D=(1 << 19) + 1) == UNSUPPORTED
    assert [gcg_lib.gcg_scan_states(n) for n in (0, 1, 64, 65)] == [0, 1, 1, 2]
    step = lambda x=p, f=p, s=(ctypes.c_int64 * 3)(64, 64, 64), state=p, y=p, bs=2, D=64: gcg_lib.gcg_scan_step(              # noqa: E731
        x, f, none, s, none, state, y, bs, D, 0, none)
    assert step(x=none) == step(f=none) == step(state=none) == step(y=none) == step(bs=0) == step(D=-1) == BAD_ARG
    assert step(s=(ctypes.c_int64 * 3)(64, -1, 64)) == BAD_ARG and step(D=(1 << 19) + 1) == UNSUPPORTED


def test_limits_agree_with_the_header():
    import os
    import re
    text = open(os.path.join(os.path.dirname(_lib.__file__), "..", "include", "gcg.h")).read()
    value = lambda name: int(eval(re.search(name + r" = ([^,}]+)", text).group(1)))                                           # noqa: E731
    assert (value("GCG_PRODUCT8_MAX_K"), value("GCG_SCAN_MAX_TIME_STRIDE"), value("GCG_SCAN_MAX_WIDTH"), value("GCG_SCAN_MAX_ROWS")) == \
        (_lib.PRODUCT8_MAX_K, _lib.SCAN_MAX_TIME_STRIDE, _lib.SCAN_MAX_WIDTH, _lib.SCAN_MAX_ROWS)
    assert (value("GCG_E4M3"), value("GCG_E5M2")) == (_lib.GCG_E4M3, _lib.GCG_E5M2)


def test_a_step_whose_gradients_sum_over_too_many_is_refused_before_it(gcg_lib):
    """The weight's gradient sums over the rows and x's over the outputs, at most 2^22 of either: said by the forward, not after it."""
    many = (1 << 22) + 1
    x, w, wide = torch.zeros(many, 1).half(), torch.zeros(2, 1).half(), torch.zeros(many, 1).half()
    needs = lambda t: t.clone().requires_grad_(True)                                                                           # noqa: E731
    ops = torch.ops.gcg
    for call in (lambda: linear_float8(x, needs(w)), lambda: linear_float8(x[:5].clone().requires_grad_(True), wide),
                 lambda: linear_float8(x.reshape(1, many, 1), needs(w)), lambda: norm_linear_float8(x, None, needs(w)),
                 lambda: norm_linear_float8(x[:5], needs(torch.ones(1).half()), wide), lambda: norm_linear_float8(x[:5], None, wide, residual=needs(x[:5])),
                 lambda: ops.linear_float8(x, needs(w), E4M3), lambda: ops.linear_float8(needs(x[:5]), wide, E4M3),
                 lambda: ops.norm_linear_float8(x, None, None, needs(w), 1e-6, E4M3)):
        with pytest.raises((ValueError, RuntimeError), match="4194304"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="MI355X|CPU"):
            call()                                                              # (nothing but the device is missing)
    for call in (lambda: linear_float8(needs(x), w), lambda: linear_float8(x, wide), lambda: linear_float8(x[:-1], needs(w))):
        with pytest.raises(RuntimeError, match="MI355X"):
            call()
