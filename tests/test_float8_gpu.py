"""The 8-bit floating-point format: codes and scales bit for bit as its definition in 64 bits has them."""
import pytest
import torch

from layer8 import TOP, float8, values
from savanna_amd import _lib
from savanna_amd.operators.float8 import E4M3, E5M2, Float8, from_float8, to_float8

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def data(rows, D, dtype, seed=0):
    """Numbers over many powers of two, ties and borders among them, rows and blocks of zeros."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(rows, D, generator=gen, device=DEV) * torch.exp2(torch.randint(-12, 5, (rows, D), generator=gen, device=DEV).float())
    x = torch.where(torch.rand(rows, D, generator=gen, device=DEV) < 0.1, torch.randint(-64, 65, (rows, D), generator=gen, device=DEV) / 8.0, x)
    if rows > 2:
        x[1] = 0
        x[2, :128] = 0
        x[2, :1] = 1.75                                     # exactly the largest number
    return x.to(dtype)


def same(q, x, fmt):
    ref, e = float8(x, fmt)
    rows, D = x.shape[:-1], x.shape[-1]
    blocks = (D + 127) // 128
    assert q.codes.dtype == fmt and q.codes.shape == (*rows, blocks * 128) and q.scales.shape == (*rows, (D + 511) // 512 * 4) and q.columns == D
    scales = q.scales.view(torch.uint8).int()
    assert torch.equal(scales[..., :blocks], e.int() + 127) and (scales[..., blocks:] == 127).all()
    assert torch.equal(values(q), ref) and not q.codes.view(torch.uint8)[..., D:].any()


@pytest.mark.parametrize("fmt", [E4M3, E5M2])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,D", [(1, 1), (3, 127), (5, 128), (4, 130), (3, 512), (7, 513), (130, 1000), (2, 4096), (1, 20001)])
def test_rows(rows, D, dtype, fmt):
    x = data(rows, D, dtype, seed=rows * D)
    q = to_float8(x, fmt)
    same(q, x, fmt)
    for out in TYPES:
        want = values(q)
        got = from_float8(q, out)
        assert got.dtype == out and torch.equal(got, want.to(out))       # (one rounding: 64 bits hold the value)
    deep = to_float8(x.reshape(rows, 1, D).expand(rows, 2, D), fmt)      # more dimensions, strided
    assert torch.equal(deep.codes[:, 1].view(torch.uint8), q.codes.view(torch.uint8))


@pytest.mark.parametrize("fmt", [E4M3, E5M2])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,D", [(1, 1), (127, 3), (128, 128), (129, 130), (300, 513), (1, 1000), (1000, 1), (515, 70)])
def test_columns_and_both(rows, D, dtype, fmt):
    x = data(rows, D, dtype, seed=rows + D)
    codes, scales = _lib.to_float8_columns(x, fmt)
    same(Float8(codes, scales, rows), x.t(), fmt)
    a, b, c, d = _lib.to_float8_both(x, fmt)
    assert torch.equal(c.view(torch.uint8), codes.view(torch.uint8)) and torch.equal(d.view(torch.uint8), scales.view(torch.uint8))
    same(Float8(a, b, D), x, fmt)


@pytest.mark.parametrize("start,fmt", [(E4M3, E4M3), (E4M3, E5M2), (E5M2, E4M3), (E5M2, E5M2)])
@pytest.mark.parametrize("rows,D", [(1, 1), (129, 130), (300, 513), (128, 256)])
def test_columns_of_8_bits(rows, D, start, fmt):
    q = to_float8(data(rows, D, torch.bfloat16, seed=D), start)
    codes, scales = _lib.float8_columns(q.codes, q.scales, D, fmt)
    same(Float8(codes, scales, rows), values(q).t(), fmt)


@pytest.mark.parametrize("fmt", [E4M3, E5M2])
def test_extremes(fmt):
    x = torch.zeros(8, 256, device=DEV)
    x[0, 5] = float("inf")
    x[0, 6:9] = torch.tensor([1.0, 2.0 ** 112, -(2.0 ** 127)])
    x[1, 3] = float("nan")
    x[2, :3] = torch.tensor([2.0 ** -127, 2.0 ** -149, -(2.0 ** -140)])              # fp32's subnormal numbers
    x[3, :3] = torch.tensor([3.4028235e38, -3.4028235e38, 2.0 ** 110])
    x[4, :2] = torch.tensor([1.75, 2.0 ** -30])
    x[5, :2] = torch.tensor([1.7500001, 1.75])
    x[6, 130] = -0.0
    q = to_float8(x, fmt)
    v, s = values(q), q.scales.view(torch.uint8).int()
    most = 247 if fmt is E4M3 else 240                               # brings the largest fp32 number into the format's range
    assert (s[0, 0], s[1, 0]) == (most, most) and s[0, 1] == 127
    assert torch.isnan(v[0, 5]) if fmt is E4M3 else v[0, 5] == float("inf")
    assert torch.isnan(v[1, 3]) and torch.isnan(v[1]).sum() == 1
    assert v[0, 6] == 0 and v[0, 8] == -(2.0 ** 127)
    finite = x[2:].clone()
    ref, e = float8(finite, fmt)
    assert torch.equal(v[2:], ref) and torch.equal(s[2:, :2], e.int() + 127)
    assert s[4, 0] == s[5, 0] - 1 and v[3, 0] <= TOP[fmt] * 2.0 ** (most - 127)
    # columns find the same
    t = Float8(*_lib.to_float8_columns(x.t().contiguous(), fmt), 256)
    assert torch.equal(t.codes.view(torch.uint8), q.codes.view(torch.uint8)) and torch.equal(t.scales.view(torch.uint8), q.scales.view(torch.uint8))


def test_refusals():
    x = torch.randn(4, 300, device=DEV)
    q = to_float8(x)
    for bad in (lambda: to_float8(x.double()), lambda: to_float8(x, torch.int8), lambda: to_float8(x.cpu()), lambda: from_float8(q, torch.float64),
                lambda: from_float8(Float8(q.codes[:, :128], q.scales, 300), torch.float32), lambda: from_float8(Float8(q.codes, q.scales[:, :3], 300), torch.float32),
                lambda: from_float8(Float8(q.codes, q.scales, 200), torch.float32), lambda: from_float8(Float8(q.codes, q.scales.view(torch.uint8), 300), torch.float32),
                lambda: _lib.to_float8_columns(x[None], E4M3), lambda: _lib.to_float8_both(x.t(), E4M3),
                lambda: from_float8(Float8(q.codes.cpu(), q.scales.cpu(), 300), torch.float32)):
        with pytest.raises((RuntimeError, ValueError, TypeError)):
            bad()
    for shape in ((0, 300), (3, 0)):
        e = to_float8(torch.randn(*shape, device=DEV))
        assert from_float8(e, torch.float32).shape == shape
    grad = to_float8(x.requires_grad_(True))
    assert not grad.codes.requires_grad


def test_a_scale_that_is_no_number():
    """The byte 255 of float8_e8m0fnu, which tensors made elsewhere may hold, makes its whole block NaN, whatever the codes."""
    x = torch.randn(130, 300, device=DEV)
    for fmt in (E4M3, E5M2):
        q = to_float8(x, fmt)
        q.codes.view(torch.uint8)[3, 130] = 0
        clean = from_float8(q, torch.float32)
        q.scales.view(torch.uint8)[3, 1] = 255
        bad = torch.zeros(130, 300, dtype=torch.bool, device=DEV)
        bad[3, 128:256] = True
        for out in TYPES:
            v = from_float8(q, out)
            assert torch.equal(torch.isnan(v), bad) and torch.equal(v[~bad], clean[~bad].to(out))
        t = Float8(*_lib.float8_columns(q.codes, q.scales, 300, E4M3), 130)
        assert torch.equal(torch.isnan(from_float8(t, torch.float32)).t(), bad)
