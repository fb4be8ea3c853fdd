"""The 8-bit checkpoint kernels against the format's definition in fp32 on the CPU, bit for bit: codes, scales and values.
(fp32 products, quotients and roundings to whole numbers are exact functions of their operands on both sides.)"""
import pytest
import torch

from savanna_amd import _lib
from savanna_amd.operators.act8 import Packed8, pack8, unpack8

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def plain(x):
    """(codes, scales, values) of a CPU tensor."""
    D = x.shape[-1]
    v = torch.nn.functional.pad(x.float(), (0, -D % 128)).unflatten(-1, (-1, 128))
    top = v.abs().amax(-1, keepdim=True)
    tiny, bad = top < 2.0 ** -100, ~torch.isfinite(top)
    scale = torch.where(tiny, 0.0, top * torch.tensor(1.0 / 127.0))
    scale = torch.where(bad, float("nan"), scale)
    inv = torch.where(tiny | bad, 0.0, torch.full_like(top, 127.0) / top)
    codes = torch.where(bad, 0.0, torch.round(v * inv))
    values = (codes * scale).flatten(-2)[..., :D].to(x.dtype)
    return codes.flatten(-2)[..., :D], scale.squeeze(-1), values


def same(a, b):
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.nan_to_num(a), torch.nan_to_num(b))


# one element to rows of many blocks; rows that end inside a vector, inside a block, at a block's end
SHAPES = [(1,), (7,), (128,), (129,), (3, 1), (5, 127), (4, 128), (33, 130), (2, 3, 257), (701, 1001), (17, 4096), (1, 1000003), (20000, 5),
          (0, 64), (4, 0)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_codes_scales_and_values(gcg_lib, shape, dtype):
    gen = torch.Generator().manual_seed(sum(shape))
    x = (torch.randn(shape, generator=gen) * torch.exp2(torch.randint(-20, 12, shape, generator=gen).float() / 2)).to(dtype)
    codes, scales, values = plain(x)
    p = pack8(x.to(DEV))
    assert p.codes.shape == x.shape and p.codes.dtype == torch.int8 and p.dtype == dtype
    assert torch.equal(p.codes.cpu().float(), codes)
    assert torch.equal(p.scales.cpu(), scales)
    back = unpack8(p)
    assert back.dtype == dtype and torch.equal(back.cpu(), values)
    if x.numel():
        half = 0.5 * scales.repeat_interleave(128, -1)[..., :x.shape[-1]].double()
        eps = {torch.float32: 2.0 ** -23, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
        # half a step, the roundings of inv, the product and the scale (each 2^-24 of a code up to 127), the value's own, and
        # half an f16 denormal
        off = (back.cpu().double() - x.double()).abs()
        assert (off <= half * (1 + 127 * 2.0 ** -21) + eps * x.double().abs() + 2.0 ** -25).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_blocks_without_finite_values_and_tiny_ones(gcg_lib, dtype):
    """Every block by itself: infinities and NaN make it NaN, zeros and values below 2^-100 make it zeros."""
    x = torch.randn(6, 300, generator=torch.Generator().manual_seed(1)).to(dtype)
    x[0, 5], x[1, 130], x[2, 299], x[3, :128] = float("inf"), float("-inf"), float("nan"), 0
    if dtype != torch.float16:
        x[4, 128:256] = 2.0 ** -110
        x[5, 256:] = torch.finfo(dtype).max
    codes, scales, values = plain(x)
    p = pack8(x.to(DEV))
    assert same(p.scales.cpu(), scales)
    assert same(unpack8(p).cpu(), values)
    assert torch.isnan(unpack8(p)[0, :128]).all() and not torch.isnan(unpack8(p)[0, 128:]).any()


def test_unaligned_tensors_streams_and_strides(gcg_lib):
    """Storage that starts at an odd element, a strided tensor (copied first), work on another stream."""
    base = torch.randn(40 * 201 + 1, device=DEV).to(torch.bfloat16)
    x = base[1:].view(40, 201)
    assert torch.equal(unpack8(pack8(x)).cpu(), plain(x.cpu())[2])
    strided = torch.randn(30, 64, device=DEV)[:, ::2]
    assert torch.equal(unpack8(pack8(strided)).cpu(), plain(strided.cpu())[2])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        back = unpack8(pack8(x))
    side.synchronize()
    assert torch.equal(back.cpu(), plain(x.cpu())[2])


def test_captured_in_a_graph(gcg_lib):
    x = torch.randn(50, 777, device=DEV)
    pack8(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        back = unpack8(pack8(x))
    torch.cuda.current_stream().wait_stream(side)
    for seed in range(3):
        x.copy_(torch.randn(50, 777, generator=torch.Generator().manual_seed(seed)))
        eager = unpack8(pack8(x))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(back, eager)


def test_refusals(gcg_lib):
    x = torch.randn(4, 256, device=DEV)
    p = pack8(x)
    with pytest.raises(RuntimeError, match="no CPU path"):
        pack8(x.cpu())
    with pytest.raises((RuntimeError, TypeError), match="unsupported dtype"):
        pack8(x.double())
    with pytest.raises((RuntimeError, TypeError), match="unsupported dtype"):
        unpack8(Packed8(p.codes, p.scales, torch.float64))
    with pytest.raises((RuntimeError, ValueError), match="scales"):
        unpack8(Packed8(p.codes, p.scales[:, :1].contiguous(), x.dtype))
    with pytest.raises((RuntimeError, ValueError), match="int8"):
        unpack8(Packed8(p.codes.to(torch.uint8), p.scales, x.dtype))
    assert gcg_lib.gcg_pack8(None, p.codes.data_ptr(), p.scales.data_ptr(), 4, 256, _lib.GCG_F32, None) == -1
    assert gcg_lib.gcg_unpack8(p.codes.data_ptr(), p.scales.data_ptr(), x.data_ptr(), 4, 0, _lib.GCG_F32, None) == -1
    assert gcg_lib.gcg_pack8(x.data_ptr(), p.codes.data_ptr(), p.scales.data_ptr(), 4, 256, _lib.GCG_BF16_F32, None) == -1


def test_not_differentiable(gcg_lib):
    x = torch.randn(4, 256, device=DEV, requires_grad=True)
    assert not unpack8(pack8(x)).requires_grad
