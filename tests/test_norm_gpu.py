"""Layer norm's kernels against its formulas in 64 bits.

Tolerances.  An output is rounded once to its type (unit roundoff U).  What comes before is fp32: a row's sums add at most 32
numbers in a lane and 6 + 4 partial sums after that, so with the products every term carries fewer than 64 roundings of 2^-24:
2^-18 of the largest magnitude that enters the sum.  Where the mean is far from zero, x - mean carries the mean's own
error, so the magnitude to go by is (|x - mean| + |mean|) rstd.  A column's sums over R rows carry at most R + 64 roundings:
(R + 64) 2^-24 of the sum of the terms' magnitudes."""
import pytest
import torch

from savanna_amd import _lib
from savanna_amd.operators.act8 import pack8, unpack8
from savanna_amd.operators.norm import LayerNorm, layer_norm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}      # half an f16 denormal
F32 = 2.0 ** -18


def data(rows, D, dtype, pdtype=None, seed=0, shift=0.5):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen, device=DEV)                 # noqa: E731
    x = (rand(rows, D) * torch.exp(0.5 * rand(D)) + shift * rand(D)).to(dtype)
    w, b = (1 + 0.3 * rand(D)).to(pdtype or dtype), (0.2 * rand(D)).to(pdtype or dtype)
    return x, w, b, rand(rows, D).to(dtype)


def reference(x, w, b, dy, eps, kept=None):
    """(y, dx, dw, db) in 64 bits and the tolerances of each, as above; kept: what the backward reads in x's place."""
    X, dtype = x.double(), x.dtype
    W = w.double() if w is not None else torch.ones(x.shape[-1], dtype=torch.float64, device=x.device)
    B = b.double() if b is not None else torch.zeros_like(W)
    mean = X.mean(-1, keepdim=True)
    rstd = ((X - mean).square().mean(-1, keepdim=True) + eps).rsqrt()
    y = (X - mean) * rstd * W + B
    K = X if kept is None else kept.double()
    xh, dY = (K - mean) * rstd, dy.double()
    g = dY * W
    c1, c2 = g.mean(-1, keepdim=True), (g * xh).mean(-1, keepdim=True)
    dx = rstd * (g - c1 - xh * c2)
    size = ((K - mean).abs() + mean.abs()) * rstd
    size_y = ((X - mean).abs() + mean.abs()) * rstd
    top = lambda t: t.abs().amax(-1, keepdim=True)                               # noqa: E731
    pt = w.dtype if w is not None else dtype
    R = x.shape[0]
    return [(y, U[dtype] * y.abs() + F32 * (top(size_y) * W.abs() + B.abs()) + TINY[dtype]),
            (dx, U[dtype] * dx.abs() + F32 * rstd * (top(g) + top(g * size) * top(size) + top(g) * top(size) ** 2) + TINY[dtype]),
            ((dY * xh).sum(0), U[pt] * (dY * xh).sum(0).abs() + ((R + 64) * 2.0 ** -24 + F32) * (dY.abs() * size).sum(0) + TINY[pt]),
            (dY.sum(0), U[pt] * dY.sum(0).abs() + (R + 64) * 2.0 ** -24 * dY.abs().sum(0) + TINY[pt])]


def check(got, want, what):
    for name, g, (ref, tol) in zip(("y", "dx", "dw", "db"), got, want):
        if g is None:
            continue
        off = (g.double() - ref).abs() - tol
        assert (off <= 0).all(), f"{what} {name}: {off.max().item():.3e} over a tolerance of {tol.flatten()[off.argmax()].item():.3e}"


def step(x, w, b, dy, eps=1e-5, save_8bit=False):
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b) if t is not None]
    it = iter(leaves)
    X, W, B = next(it), next(it) if w is not None else None, next(it) if b is not None else None
    y = layer_norm(X, W, B, eps, save_8bit)
    grads = iter(torch.autograd.grad(y, leaves, dy))
    return y.detach(), next(grads), next(grads) if w is not None else None, next(grads) if b is not None else None


WIDTHS = [1, 2, 7, 8, 63, 128, 255, 256, 257, 512, 520, 1000, 1023, 1024, 1025, 2048, 2051, 4096, 4100, 5001, 8192, 8200, 12288, 12345, 16383,
          16384]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", WIDTHS)
def test_widths(gcg_lib, D, dtype):
    for rows in (1, 37):
        x, w, b, dy = data(rows, D, dtype, seed=D)
        check(step(x, w, b, dy), reference(x, w, b, dy, 1e-5), f"{rows}x{D} {dtype}")
        check([layer_norm(x, w, b)], reference(x, w, b, dy, 1e-5), f"{rows}x{D} {dtype} forward")


@pytest.mark.parametrize("rows", [1, 2, 3, 5, 255, 2049, 5003, 20011])
@pytest.mark.parametrize("D,dtype", [(256, torch.float32), (640, torch.bfloat16), (96, torch.float16)])
def test_rows(gcg_lib, rows, D, dtype):
    x, w, b, dy = data(rows, D, dtype, seed=rows)
    check(step(x, w, b, dy), reference(x, w, b, dy, 1e-5), f"{rows}x{D} {dtype}")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,D", [(1, 1), (3, 100), (37, 128), (50, 1001), (300, 2560), (40, 8192), (9, 16384), (2051, 200)])
def test_backward_from_8_bits(gcg_lib, rows, D, dtype):
    """The checkpoint is pack8's, the forward's result does not change, and the gradients are the formula's at its values."""
    x, w, b, dy = data(rows, D, dtype, seed=rows + D)
    _, stats, codes, scales = _lib.layer_norm_fwd(x, w, b, 1e-5, True)
    p = pack8(x)
    assert torch.equal(codes, p.codes) and torch.equal(scales, p.scales)
    got = step(x, w, b, dy, save_8bit=True)
    assert torch.equal(got[0], layer_norm(x, w, b))
    kept = unpack8(p._replace(dtype=torch.float32))
    check(got, reference(x, w, b, dy, 1e-5, kept), f"8 bits {rows}x{D} {dtype}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_float32_parameters(gcg_lib, dtype):
    x, w, b, dy = data(77, 1030, dtype, torch.float32, seed=3)
    got = step(x, w, b, dy)
    assert got[2].dtype == got[3].dtype == torch.float32
    check(got, reference(x, w, b, dy, 1e-5), f"fp32 parameters, {dtype}")


@pytest.mark.parametrize("parts", ["", "w", "b"])
def test_optional_parameters(gcg_lib, parts):
    x, w, b, dy = data(33, 300, torch.bfloat16, seed=4)
    w, b = w if "w" in parts else None, b if "b" in parts else None
    check(step(x, w, b, dy), reference(x, w, b, dy, 1e-5), f"parameters {parts!r}")


def test_far_mean_and_tiny_variance(gcg_lib):
    """The variance is summed about the mean: rows whose mean is 1000 times their spread keep it; constant rows give b."""
    x, w, b, dy = data(20, 512, torch.float32, seed=5)
    x = x + 1000
    check(step(x, w, b, dy), reference(x, w, b, dy, 1e-5), "far mean")
    y = layer_norm(torch.full((3, 512), 0.25, device=DEV), w, b)
    assert torch.equal(y, b.expand(3, 512))


def test_rows_without_finite_values_stay_among_themselves(gcg_lib):
    x, w, b, dy = data(9, 700, torch.bfloat16, seed=6)
    x[2, 3], x[5, 699] = float("inf"), float("nan")
    for save_8bit in (False, True):
        y, dx, dw, db = step(x, w, b, dy, save_8bit=save_8bit)
        bad = torch.zeros(9, dtype=torch.bool, device=DEV)
        bad[[2, 5]] = True
        assert torch.isnan(y[bad]).all() and torch.isfinite(y[~bad]).all()
        assert torch.isnan(dx[bad]).all() and torch.isfinite(dx[~bad]).all()
        assert torch.isnan(dw).all() and torch.isfinite(db).all()


def test_gradients_against_differences(gcg_lib):
    """<gradient, direction> against (L(p + h d) - L(p - h d)) / 2h, L = <y, dy> added in 64 bits.  The forward's fp32
    error, 2^-20 of the terms, is divided by h; the remainder is h^2 / 6 times a third derivative of the order of L's terms."""
    x, w, b, dy = data(5, 37, torch.float32, seed=7)
    _, dx, dw, db = step(x, w, b, dy)
    gen = torch.Generator(device=DEV).manual_seed(8)
    h = 2.0 ** -6
    loss = lambda *p: (layer_norm(*p).double() * dy.double()).sum()              # noqa: E731
    for i, grad in enumerate((dx, dw, db)):
        p = [x, w, b]
        d = torch.randn(p[i].shape, generator=gen, device=DEV)
        d = d / d.norm()
        ends = [loss(*[t + s * h * d if j == i else t for j, t in enumerate(p)]) for s in (1, -1)]
        terms = dy.abs().double().sum()
        got = (grad.double() * d.double()).sum()
        assert abs((ends[0] - ends[1]) / (2 * h) - got) <= terms * (2.0 ** -20 / h + h * h)


def test_dimensions_strides_alignment_streams(gcg_lib):
    """Leading dimensions of any number, strided tensors, storage off the vectors, an odd width, another stream; two runs agree
    bit for bit."""
    x, w, b, dy = data(60, 333, torch.bfloat16, seed=9)
    want = reference(x, w, b, dy, 1e-5)
    got = step(x.view(3, 4, 5, 333), w, b, dy.view(3, 4, 5, 333))
    check([t.reshape(60, 333) if t.dim() == 4 else t for t in got], want, "leading dimensions")
    base = torch.empty(60 * 333 + 1, dtype=x.dtype, device=DEV)
    odd = base[1:].view(60, 333).copy_(x)
    wide = torch.empty(60, 666, dtype=x.dtype, device=DEV)
    wide[:, ::2] = x
    for t in (odd, wide[:, ::2]):
        assert all(torch.equal(a, c.reshape(a.shape)) for a, c in zip(step(t, w, b, dy), got))
    assert torch.equal(layer_norm(x[0], w, b), got[0].reshape(60, 333)[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step(x, w, b, dy)
    side.synchronize()
    assert all(torch.equal(a, c.reshape(a.shape)) for a, c in zip(again, got))
    dyt = dy.t().contiguous().t()
    assert all(torch.equal(a, c.reshape(a.shape)) for a, c in zip(step(x, w, b, dyt), got))


def test_empty(gcg_lib):
    w, b = torch.ones(64, device=DEV), torch.zeros(64, device=DEV)
    y, dx, dw, db = step(torch.empty(0, 64, device=DEV), w, b, torch.empty(0, 64, device=DEV))
    assert y.shape == dx.shape == (0, 64) and not dw.any() and not db.any()


def test_captured_in_a_graph(gcg_lib):
    x, w, b, dy = data(300, 1000, torch.bfloat16, seed=10)
    codes = [_lib.layer_norm_fwd(x, w, b, 1e-5, True)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        y, stats, codes, scales = _lib.layer_norm_fwd(x, w, b, 1e-5, True)
        grads = _lib.layer_norm_bwd(dy, None, codes, scales, stats, w, b)
    torch.cuda.current_stream().wait_stream(side)
    for seed in range(3):
        x.copy_(data(300, 1000, torch.bfloat16, seed=20 + seed)[0])
        eager = step(x, w, b, dy, save_8bit=True)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip((y, *grads), eager))


def test_module_compiled_and_dispatched(gcg_lib):
    """The module, the registered operator's own autograd formula, and a traced call give the same bits."""
    torch.manual_seed(0)
    m = LayerNorm(200, dtype=torch.bfloat16, device=DEV, save_8bit=True)
    x, _, _, dy = data(50, 200, torch.bfloat16, seed=11)
    want = step(x, m.weight.detach(), m.bias.detach(), dy, save_8bit=True)
    X = x.clone().requires_grad_(True)
    got = m(X)
    got.backward(dy)
    assert all(torch.equal(a, c) for a, c in zip((got, X.grad, m.weight.grad, m.bias.grad), want))
    X2 = x.clone().requires_grad_(True)
    if _lib.TORCH_OPS:
        y = torch.ops.gcg.layer_norm_fwd(X2, m.weight, m.bias, 1e-5, True)[0]
        assert all(torch.equal(a, c) for a, c in zip((y, *torch.autograd.grad(y, [X2, m.weight, m.bias], dy)), want))
    f = torch.compile(lambda t: layer_norm(t, m.weight, m.bias, save_8bit=True), fullgraph=True, backend="aot_eager")
    y = f(X2)
    assert all(torch.equal(a, c) for a, c in zip((y, *torch.autograd.grad(y, [X2, m.weight, m.bias], dy)), want))


def test_refusals(gcg_lib):
    x, w, b, _ = data(4, 64, torch.bfloat16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        layer_norm(x.cpu())
    with pytest.raises((RuntimeError, ValueError), match="size of x's last dimension"):
        layer_norm(x, w[:32].contiguous(), b)
    with pytest.raises((RuntimeError, TypeError), match="dtype or be float32"):
        layer_norm(x, w.to(torch.float16), b.to(torch.float16))
    with pytest.raises((RuntimeError, TypeError), match="share one dtype"):
        layer_norm(x, w, b.float())
    with pytest.raises((RuntimeError, TypeError), match="unsupported dtype"):
        layer_norm(x.double())
    with pytest.raises((RuntimeError, ValueError), match="16384"):
        layer_norm(torch.zeros(1, 16385, device=DEV))
    with pytest.raises((RuntimeError, ValueError), match="either x, or"):
        _lib.layer_norm_bwd(x, x, pack8(x).codes, pack8(x).scales, torch.zeros(4, 2, device=DEV), w, b)
    p = x.data_ptr()
    assert gcg_lib.gcg_layer_norm_fwd(None, p, p, p, None, None, None, 4, 64, 1e-5, 1, None) == -1
    assert gcg_lib.gcg_layer_norm_fwd(p, p, p, p, None, None, None, 4, 64, -1.0, 1, None) == -1
    assert gcg_lib.gcg_layer_norm_fwd(p, p, p, p, None, p, None, 4, 64, 1e-5, 1, None) == -1
    assert gcg_lib.gcg_layer_norm_fwd(p, p, p, p, None, None, None, 4, 16385, 1e-5, 1, None) == -2
    assert gcg_lib.gcg_layer_norm_bwd(p, p, None, None, p, p, p, p, p, None, 0, 4, 64, 1, None) == -3
    assert gcg_lib.gcg_layer_norm_bwd_workspace_bytes(4, 16385, 1) == 0
