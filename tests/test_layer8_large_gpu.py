"""The operators of a layer in 8-bit floating point on tensors beyond 2^31 elements (and 2^32 bytes): parts of the result against the operators on those
parts by themselves, bit for bit."""
import pytest
import torch

from savanna_amd import _lib
from savanna_amd.operators.float8 import E4M3, from_float8, matmul_float8, to_float8
from savanna_amd.operators.gated_recurrence import gated_recurrence_features
from savanna_amd.operators.norm import rms_norm_float8

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ROWS, WIDTH = (1 << 19) + 77, 4096                          # 2^31 elements and 77 rows
CUTS = [slice(0, 256), slice(1 << 18, (1 << 18) + 256), slice((1 << 19) - 128, ROWS)]


@pytest.fixture(autouse=True)
def room():
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("needs 80 GiB of device memory")
    yield
    torch.cuda.empty_cache()


def normal(*shape, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return torch.empty(*shape, dtype=torch.bfloat16, device=DEV).normal_(generator=gen)


def bits(t):
    return t.view(torch.uint8)


def test_norm():
    x, res, dy, dr = (normal(ROWS, WIDTH, seed=s) for s in range(4))
    w = 1 + normal(WIDTH, seed=4) / 4
    y, r, rstd = _lib.rms_norm_fwd(x, res, w, 1e-6)
    dx, dw = _lib.rms_norm_bwd(dy, r, dr, rstd, w)
    q, r8 = rms_norm_float8(x, w, residual=res)
    assert torch.equal(r8, r)
    for c in CUTS:
        a, b, s = _lib.rms_norm_fwd(x[c], res[c], w, 1e-6)
        assert torch.equal(y[c], a) and torch.equal(r[c], b) and torch.equal(rstd[c], s)
        assert torch.equal(dx[c], _lib.rms_norm_bwd(dy[c], b, dr[c], s, w)[0])
        p, _ = rms_norm_float8(x[c], w, residual=res[c])
        assert torch.equal(bits(q.codes[c]), bits(p.codes)) and torch.equal(bits(q.scales[c]), bits(p.scales))
    # the weight's gradient: fp32 sums of 2^19 terms, at most a rounding each, and one to bf16
    sums = [torch.zeros(WIDTH, dtype=torch.float64, device=DEV) for _ in range(2)]
    for i in range(0, ROWS, 1 << 15):
        t = dy[i:i + (1 << 15)].double() * r[i:i + (1 << 15)].double() * rstd[i:i + (1 << 15), None].double()
        sums[0] += t.sum(0)
        sums[1] += t.abs().sum(0)
    assert ((dw.double() - sums[0]).abs() <= 2.0 ** -8 * sums[0].abs() + (ROWS + 64) * 2.0 ** -24 * sums[1]).all()


def test_into_8_bits_and_back():
    x = normal(ROWS, WIDTH)
    q = to_float8(x)
    codes_t, scales_t = _lib.to_float8_columns(x, E4M3)
    both = _lib.to_float8_both(x, E4M3)
    for a, b in zip(both, (q.codes, q.scales, codes_t, scales_t)):
        assert torch.equal(bits(a), bits(b))
    del both
    again_t, again_s = _lib.float8_columns(q.codes, q.scales, WIDTH, E4M3)
    back = from_float8(q, torch.bfloat16)
    for c in CUTS:
        p = to_float8(x[c])
        assert torch.equal(bits(q.codes[c]), bits(p.codes)) and torch.equal(bits(q.scales[c]), bits(p.scales)) and torch.equal(back[c], from_float8(p, torch.bfloat16))
        n, first, blocks = c.stop - c.start, c.start // 128, (c.stop - c.start + 127) // 128
        for got, scales, (want, want_s) in ((codes_t, scales_t, _lib.to_float8_columns(x[c], E4M3)),
                                            (again_t, again_s, _lib.float8_columns(p.codes, p.scales, WIDTH, E4M3))):
            assert torch.equal(bits(got[:, c.start:c.stop]), bits(want[:, :n]))
            assert torch.equal(bits(scales)[:, first:first + blocks], bits(want_s)[:, :blocks])
    assert not bits(codes_t[:, ROWS:]).any() and (bits(scales_t)[:, (ROWS + 127) // 128:] == 127).all()


@pytest.mark.parametrize("M,N,K", [(70001, 32800, 200), (ROWS, 260, 4096), (129, ROWS, 4100), (300, 300, 1 << 22), (70, 130, (1 << 22) - 100)])
def test_products(M, N, K):
    """Whole numbers, whose sums are exact (random ones of 2^22 products stay far below 2^24): results, one operand or the other beyond 2^31, and the longest
    sums."""
    gen = torch.Generator(device=DEV).manual_seed(K)
    a, b = (torch.randint(-4, 5, (n, K), generator=gen, device=DEV, dtype=torch.int8).to(torch.bfloat16) for n in (M, N))
    y = matmul_float8(to_float8(a), to_float8(b))
    for rows in (slice(0, 200), slice(M // 2, M // 2 + 100), slice(max(M - 300, 0), M)):
        for cols in (slice(0, 300), slice(max(N - 700, 0), N)):
            assert torch.equal(y[rows, cols], (a[rows].float() @ b[cols].float().t()).bfloat16())


def test_recurrence():
    """Two sequences of 2^19 rows and 2048 channels, as if each were alone."""
    L, D = ROWS, 2048
    features, dy = normal(2, L, 3 * D), normal(2, L, D, seed=1)
    bias = torch.linspace(0, 8, D, device=DEV)
    features.requires_grad_(True)
    y = gated_recurrence_features(features, bias)
    g, = torch.autograd.grad(y, features, dy)
    for i in range(2):
        alone = features[i:i + 1].detach().requires_grad_(True)
        z = gated_recurrence_features(alone, bias)
        assert torch.equal(y[i:i + 1], z)
        assert torch.equal(g[i:i + 1], torch.autograd.grad(z, alone, dy[i:i + 1])[0])
        del z
