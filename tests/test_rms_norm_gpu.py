"""Root-mean-square norm's kernels against its formulas in 64 bits.

Tolerances.  r is one addition in fp32 and one rounding: compared bit for bit.  y, dx and dw are rounded once to their type (unit roundoff U).
What comes before is fp32: a row's sum adds at most 32 products in a lane and 6 + 4 partial sums after that, so its terms
carry fewer than 44 roundings of 2^-24, rstd half of that and three more, y two more: 2^-18 of |y|.  dx adds the product of such numbers:
2^-18 of the largest magnitude that enters.  A column's sum over R rows carries at most R + 64 roundings of its terms' magnitudes."""
import pytest
import torch

from layer8 import TINY, U, check, float8, values
from savanna_amd import _lib
from savanna_amd.operators.norm import RMSNorm, rms_norm, rms_norm_float8

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32 = 2.0 ** -18
TYPES = [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), (torch.bfloat16, torch.float32),
         (torch.float16, torch.float32)]


def data(shape, dtype, wtype, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen, device=DEV)                 # noqa: E731
    D = shape[-1]
    spread = torch.exp(0.5 * rand(D))
    x, res = (rand(*shape) * spread).to(dtype), (rand(*shape) * spread).to(dtype)
    return x, res, (1 + 0.3 * rand(D)).to(wtype), rand(*shape).to(dtype), rand(*shape).to(dtype)


def reference(r, w, dy, dr, eps):
    """((y, tol), (dx, tol), (dw, tol))"""
    dtype, R = r.dtype, r.numel() // r.shape[-1]
    X, W = r.double(), (w.double() if w is not None else torch.ones(r.shape[-1], dtype=torch.float64, device=r.device))
    rstd = (X.square().mean(-1, keepdim=True) + eps).rsqrt()
    xh, dY = X * rstd, dy.double()
    y, g = xh * W, dY * W
    dx = rstd * (g - xh * (g * xh).mean(-1, keepdim=True))
    size = rstd * (g.abs() + xh.abs() * (g * xh).abs().mean(-1, keepdim=True))
    if dr is not None:
        dx, size = dx + dr.double(), size + dr.double().abs()
    dw, dw_size = (dY * xh).flatten(0, -2).sum(0), (dY * xh).abs().flatten(0, -2).sum(0)
    wt = w.dtype if w is not None else dtype
    return ((y, (U[dtype] + F32) * y.abs() + TINY[dtype]), (dx, U[dtype] * dx.abs() + F32 * size + TINY[dtype]),
            (dw, U[wt] * dw.abs() + ((R + 64) * 2.0 ** -24 + F32) * dw_size + TINY[wt]))


@pytest.mark.parametrize("dtype,wtype", TYPES)
@pytest.mark.parametrize("rows,D", [(1, 1), (3, 7), (5, 128), (2, 511), (70, 513), (1100, 96), (33, 1001), (9, 2048), (7, 4096), (6, 4100),
                                    (5, 8192), (3, 8200), (2, 16384)])
@pytest.mark.parametrize("added", [False, True])
def test_forward_and_backward(rows, D, dtype, wtype, added):
    x, res, w, dy, dr = data((rows, D), dtype, wtype, seed=rows + D)
    leaves = [t.requires_grad_(True) for t in ((x, res, w) if added else (x, w))]
    r = (x.float() + res.float()).to(dtype).detach() if added else x.detach()
    out = rms_norm(x, w, 1e-6, residual=res if added else None)
    if added:
        y, got_r = out
        assert torch.equal(got_r, r)
        gx, gres, gw = torch.autograd.grad([y, got_r], leaves, [dy, dr])
        assert torch.equal(gx, gres)
    else:
        y = out
        gx, gw = torch.autograd.grad(y, leaves, dy)
    for name, got, (ref, tol) in zip(("y", "dx", "dw"), (y.detach(), gx, gw), reference(r, w.detach(), dy, dr if added else None, 1e-6)):
        assert got.dtype == (wtype if name == "dw" else dtype)
        check(got, ref, tol, f"{name} {rows} x {D}")
    with torch.no_grad():
        again = rms_norm(x, w, 1e-6, residual=res if added else None)
        for a, b in zip(again if added else (again,), out if added else (out,)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype,wtype", TYPES)
@pytest.mark.parametrize("D", [9, 10, 130, 131, 132, 133, 134, 135, 1031, 2053, 2054, 4099, 8201, 8207, 9003])
def test_rows_that_end_inside_a_vector(D, dtype, wtype):
    """Every length of the last vector, at several widths of the kernels, with more rows than go at once in none of them and in some."""
    test_forward_and_backward(23, D, dtype, wtype, True)
    test_output_in_8_bits(5, D, dtype)


def test_without_weight_more_dimensions_and_module():
    x, res, w, dy, _ = data((2, 5, 130), torch.bfloat16, torch.bfloat16)
    check(rms_norm(x), *reference(x, None, dy, None, 1e-6)[0], "no weight")
    strided = torch.randn(4, 130, 3, device=DEV).to(torch.bfloat16).transpose(1, 2)
    check(rms_norm(strided, w), *reference(strided.contiguous(), w, strided.contiguous(), None, 1e-6)[0], "strided")
    module = RMSNorm(130, dtype=torch.bfloat16, device=DEV)
    y, r = module(x, res)
    assert torch.equal(y, rms_norm(x, module.weight, residual=res)[0]) and torch.equal(r, (x.float() + res.float()).bfloat16())
    y.sum().backward()
    assert module.weight.grad.shape == (130,)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_only_one_of_the_outputs_is_used(dtype):
    x, res, w, dy, dr = data((37, 300), dtype, dtype)
    leaves = [t.requires_grad_(True) for t in (x, res, w)]
    r = (x.float() + res.float()).to(dtype).detach()
    gx, gres, gw = torch.autograd.grad(rms_norm(x, w, residual=res)[0], leaves, dy)
    _, (dx, tol), (dw, dw_tol) = reference(r, w.detach(), dy, None, 1e-6)
    check(gx, dx, tol, "dx"), check(gw, dw, dw_tol, "dw")
    gx, gres, gw = torch.autograd.grad(rms_norm(x, w, residual=res)[1], leaves, dr)
    assert torch.equal(gx, dr) and torch.equal(gres, dr) and not gw.any()
    frozen = w.detach()
    gx, = torch.autograd.grad(rms_norm(x, frozen, residual=res.detach())[0], [x], dy)
    check(gx, dx, tol, "dx of a frozen norm")


def test_gradient_against_differences():
    x, _, w, dy, _ = data((4, 20), torch.float32, torch.float32)
    x.requires_grad_(True)
    gx, = torch.autograd.grad(rms_norm(x, w), x, dy)
    X, W, dY = x.detach().double(), w.double(), dy.double()
    f = lambda X: ((X * (X.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * W) * dY).sum()        # noqa: E731
    for i, j in [(0, 0), (1, 7), (3, 19)]:
        h = torch.zeros_like(X)
        h[i, j] = 1e-5
        # the difference is off by h^2 / 6 of the third derivative and by 64-bit roundings over h: 1e-9 of the terms
        assert abs((f(X + h) - f(X - h)) / 2e-5 - gx[i, j].double()) <= 1e-5 * gx[i].double().abs().max()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,D", [(1, 1), (3, 7), (5, 128), (2, 511), (70, 513), (33, 1001), (5, 4096), (3, 8200), (2, 16384)])
def test_output_in_8_bits(rows, D, dtype):
    x, res, w, dy, _ = data((rows, D), dtype, dtype, seed=D)
    r = (x.float() + res.float()).to(dtype)
    q, got_r = rms_norm_float8(x, w, residual=res)
    assert torch.equal(got_r, r) and q.columns == D
    S = (D + 511) // 512 * 4
    assert q.codes.shape == (rows, (D + 127) // 128 * 128) and q.scales.shape == (rows, S)
    assert not q.codes.view(torch.uint8)[:, D:].any() and (q.scales.view(torch.uint8)[:, (D + 127) // 128:] == 127).all()
    y = reference(r, w, dy, None, 1e-6)[0][0]
    ref, e = float8(y)
    # y may fall on the other side of a tie, or its block's largest on the other side of a power's border, by its own error; then it is one
    # step of 8 bits off: half of one (2^-4 of its magnitude, 2^-10 of the scale below the normal numbers) from y, and that error
    scale = torch.ldexp(torch.ones_like(e, dtype=torch.float64), e + 1).repeat_interleave(128, -1)[:, :D]
    check(values(q), y, 2.0 ** -4 * y.abs() + 2.0 ** -10 * scale + F32 * y.abs(), "8 bits")
    # (the share of such elements: an error of 2^-18 at most against steps of 2^-4)
    assert (values(q) != ref).double().mean() <= 2.0 ** -10 + 2 / ref.numel()
    plain = rms_norm_float8(x, w)
    assert torch.equal(plain.codes.view(torch.uint8), rms_norm_float8(x.contiguous(), w).codes.view(torch.uint8))


def test_refusals():
    x = torch.randn(3, 64, device=DEV)
    for bad in (lambda: rms_norm(x, torch.ones(63, device=DEV)), lambda: rms_norm(x, torch.ones(64, device=DEV).half()),
                lambda: rms_norm(x, residual=x[:2]), lambda: rms_norm(x, residual=x.half()), lambda: rms_norm(torch.randn(2, 16385, device=DEV)),
                lambda: rms_norm(x.double()), lambda: rms_norm(torch.randn(3, 0, device=DEV)), lambda: rms_norm(x, torch.ones(64)),
                lambda: rms_norm(x.cpu()), lambda: rms_norm_float8(x, torch.ones(63, device=DEV))):
        with pytest.raises((RuntimeError, ValueError, TypeError)):
            bad()
    assert rms_norm(x[:0]).shape == (0, 64)
    e = torch.randn(0, 64, device=DEV, requires_grad=True)
    w = torch.ones(64, device=DEV, requires_grad=True)
    rms_norm(e, w).sum().backward()
    assert not w.grad.any()


@pytest.mark.parametrize("nodes", [True, False])
@pytest.mark.parametrize("grads", [(True, True), (True, False), (False, True)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_stream_beside_8_bits_keeps_its_gradient(dtype, grads, nodes, monkeypatch):
    """The 8 bits have none, the sum beside them is a sum: its gradient reaches both that were added."""
    if not nodes:
        monkeypatch.setattr(_lib, "native_nodes", lambda t: False)
    x, res, w, dy, dr = data((37, 300), dtype, dtype)
    want = rms_norm_float8(x, w, residual=res)
    leaves = [t.requires_grad_(need) for t, need in zip((x, res), grads)]
    q, r = rms_norm_float8(x * 1, w.requires_grad_(True), residual=res * 1)
    assert torch.equal(r, want[1]) and torch.equal(q.codes.view(torch.uint8), want[0].codes.view(torch.uint8))
    assert r.requires_grad and not q.codes.requires_grad and not q.scales.requires_grad
    for g in torch.autograd.grad(r, [t for t in leaves if t.requires_grad], dr):
        assert torch.equal(g, dr)
    r.mul_(2)                                               # r belongs to the caller
    with torch.no_grad():
        assert not rms_norm_float8(x, w, residual=res)[1].requires_grad
    assert not rms_norm_float8(x.detach(), w, residual=res.detach())[1].requires_grad
    assert not rms_norm_float8(x, w).codes.requires_grad


@pytest.mark.skipif(not _lib.TORCH_OPS, reason="the ctypes binding is not traced")
def test_the_stream_beside_8_bits_is_traced():
    x, res, w, dy, dr = data((37, 300), torch.bfloat16, torch.bfloat16)
    x.requires_grad_(True), res.requires_grad_(True)

    def f(x, res, w):
        q, r = rms_norm_float8(x, w, residual=res)
        return q.codes.view(torch.uint8), r * 2
    (a, r), (b, s) = f(x, res, w), torch.compile(f, fullgraph=True, backend="aot_eager")(x, res, w)
    assert torch.equal(a, b) and torch.equal(r, s)
    for g, h in zip(torch.autograd.grad(r, (x, res), dr), torch.autograd.grad(s, (x, res), dr)):
        assert torch.equal(g, h) and torch.equal(g, 2 * dr)


@pytest.mark.skipif(not _lib.TORCH_OPS, reason="the nodes are the torch binding's")
def test_the_stream_beside_8_bits_is_captured():
    """Replayed like the other operators, and refused where a leaf belongs to a living graph of the default stream."""
    x, res, w, _, dr = data((37, 300), torch.bfloat16, torch.bfloat16)
    x.requires_grad_(True), res.requires_grad_(True)

    def f():
        q, r = rms_norm_float8(x, w, residual=res)
        return [q.codes.view(torch.uint8), r.detach(), *torch.autograd.grad(r * 3, (x, res), dr)]
    want = f()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = f()
    for _ in range(3):
        g.replay()
        f()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    lives = (x * 1).sum()
    refused = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="still lives"), torch.cuda.graph(refused):
        res.detach() + 1
        rms_norm_float8(x, w, residual=res)
    del lives


@pytest.mark.parametrize("dtype,wtype", TYPES)
@pytest.mark.parametrize("rows,D", [(1, 1), (3, 7), (5, 128), (2, 511), (70, 513), (33, 1001), (23, 2054), (9, 2048), (5, 4096), (3, 8200), (2, 16384)])
def test_output_in_8_bits_without_a_residual(rows, D, dtype, wtype):
    """Tolerance and the share of other codes as with one."""
    x, _, w, dy, _ = data((rows, D), dtype, wtype, seed=D + 1)
    q = rms_norm_float8(x, w)
    assert q.columns == D and q.codes.shape == (rows, (D + 127) // 128 * 128) and q.scales.shape == (rows, (D + 511) // 512 * 4)
    assert not q.codes.view(torch.uint8)[:, D:].any() and (q.scales.view(torch.uint8)[:, (D + 127) // 128:] == 127).all()
    y = reference(x, w, dy, None, 1e-6)[0][0]
    ref, e = float8(y)
    scale = torch.ldexp(torch.ones_like(e, dtype=torch.float64), e + 1).repeat_interleave(128, -1)[:, :D]
    check(values(q), y, 2.0 ** -4 * y.abs() + 2.0 ** -10 * scale + F32 * y.abs(), "8 bits")
    assert (values(q) != ref).double().mean() <= 2.0 ** -10 + 2 / ref.numel()
