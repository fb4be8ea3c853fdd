"""Layer norm with frozen parameters: no gradient is formed of what is frozen, and the others keep their bits."""
import pytest
import torch

from savanna_amd import _lib
from savanna_amd.operators.norm import layer_norm
from test_norm_gpu import data, step

pytestmark = pytest.mark.gpu
FROZEN = [(w, b) for w in (False, True) for b in (False, True)]


@pytest.mark.parametrize("frozen_w,frozen_b", FROZEN)
@pytest.mark.parametrize("save_8bit", [False, True])
@pytest.mark.parametrize("rows,D", [(50, 1000), (3, 9000), (0, 64)])
def test_gradients(gcg_lib, rows, D, save_8bit, frozen_w, frozen_b):
    x, w, b, dy = data(rows, D, torch.bfloat16, seed=rows + D)
    want = step(x, w, b, dy, save_8bit=save_8bit)
    X, W, B = x.detach().requires_grad_(True), w.detach().requires_grad_(not frozen_w), b.detach().requires_grad_(not frozen_b)
    y = layer_norm(X, W, B, 1e-5, save_8bit)
    y.backward(dy)
    assert torch.equal(y, want[0]) and torch.equal(X.grad, want[1])
    assert W.grad is None if frozen_w else torch.equal(W.grad, want[2])
    assert B.grad is None if frozen_b else torch.equal(B.grad, want[3])
    if _lib.TORCH_OPS:
        X2 = x.detach().requires_grad_(True)
        z = torch.ops.gcg.layer_norm_fwd(X2, W, B, 1e-5, save_8bit)[0]
        got = torch.autograd.grad(z, [t for t in (X2, W, B) if t.requires_grad], dy)
        assert all(torch.equal(g, v) for g, v in zip(got, [want[1]] + [want[2]] * (not frozen_w) + [want[3]] * (not frozen_b)))


def test_nothing_is_summed_for_frozen_parameters(gcg_lib):
    """With both frozen the backward is one kernel, without a workspace."""
    x, w, b, dy = data(2000, 512, torch.bfloat16)
    for frozen, kernels in ((False, 2), (True, 1)):
        X, W, B = x.detach().requires_grad_(True), w.detach().requires_grad_(not frozen), b.detach().requires_grad_(not frozen)
        leaves = [t for t in (X, W, B) if t.requires_grad]
        torch.autograd.grad(layer_norm(X, W, B), leaves, dy)
        y = layer_norm(X, W, B)
        with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA, torch.profiler.ProfilerActivity.CPU]) as prof:
            torch.autograd.grad(y, leaves, dy)
            torch.cuda.synchronize()
        names = [e.name for e in prof.events() if e.device_type == torch.autograd.DeviceType.CUDA and "layer_norm" in e.name]
        assert len(names) == kernels, names
