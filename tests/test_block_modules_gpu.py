"""The modules around the convolution after casts."""
import pytest
import torch

from savanna_amd.operators.block import MixerBlock
from savanna_amd.operators.linear_attention import LinearAttention

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("save_8bit", [False, True])
def test_a_cast_block_trains_and_decodes(gcg_lib, dtype, save_8bit):
    """The same bits as a block made in that type with these weights."""
    torch.manual_seed(0)
    block = MixerBlock(128, LinearAttention(128, 2), save_8bit=save_8bit)
    made = MixerBlock(128, LinearAttention(128, 2, device=DEV), save_8bit=save_8bit, dtype=dtype, device=DEV)
    made.load_state_dict(block.state_dict())
    block = block.to(DEV, dtype)
    x = torch.randn(2, 70, 128, device=DEV).to(dtype)
    grads = [torch.autograd.grad(b(x).float().square().sum(), list(b.parameters())) for b in (block, made)]
    assert all(torch.equal(a, b) for a, b in zip(*grads))
    (y, s), (z, t) = (b.prefill(x[:, :60]) for b in (block, made))
    assert torch.equal(y, z) and torch.equal(s, t) and s.dtype == torch.float32
    assert torch.equal(block.step(x[:, 60], s), made.step(x[:, 60], t)) and torch.equal(s, t)
