"""Hyena mixers that keep their features in 8 bits, under what wraps a training step: substituted parameters, checkpointing, offloading,
autocast.  Gradients are bit for bit those of a mixer that has these parameters, on the checkpoint's values."""
import copy

import pytest
import torch

from savanna_amd.operators import hyena as module
from savanna_amd.operators.act8 import pack8, unpack8
from test_mixer_block_gpu import DEV, hyena

pytestmark = pytest.mark.gpu
ROUTES = [("mr", True), ("mr", False), ("se", True), ("se", False)]


def setup(kind, fused, seed):
    torch.manual_seed(seed)
    mixer = hyena(kind, (torch.bfloat16, "bfloat16"), False, fused)
    x = torch.randn(2, 200, 288, device=DEV).to(torch.bfloat16)
    return mixer, x, torch.randn(2, 200, 96, device=DEV).to(torch.bfloat16)


def wanted(mixer, x, dy):
    """(y, gradients of the features and of every parameter) without a checkpoint, on its values."""
    mixer = copy.deepcopy(mixer)
    mixer.save_8bit = False
    at = unpack8(pack8(x)).requires_grad_(True)
    return mixer(x).detach(), torch.autograd.grad(mixer(at), [at, *mixer.parameters()], dy)


@pytest.mark.parametrize("kind,fused", ROUTES)
def test_substituted_parameters(gcg_lib, kind, fused):
    mixer, x, dy = setup(kind, fused, 1)
    mixer.save_8bit = True
    other = copy.deepcopy(mixer)
    with torch.no_grad():
        for t in (*other.parameters(), *other.buffers()):
            t.mul_(1.5).add_(0.01)
    named = {n: t.detach().clone().requires_grad_(True) for n, t in other.named_parameters()}
    X = x.clone().requires_grad_(True)
    y = torch.func.functional_call(mixer, {**named, **dict(other.named_buffers())}, (X,))
    want_y, want = wanted(other, x, dy)
    assert torch.equal(y, want_y)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, [X, *named.values()], dy), want))


@pytest.mark.parametrize("kind,fused", ROUTES)
@pytest.mark.parametrize("wrap", ["checkpoint", "offload"])
def test_saved_tensors_that_come_back_as_others(gcg_lib, kind, fused, wrap):
    mixer, x, dy = setup(kind, fused, 2)
    mixer.save_8bit = True
    X = x.clone().requires_grad_(True)
    if wrap == "checkpoint":
        y = torch.utils.checkpoint.checkpoint(mixer, X, use_reentrant=False)
    else:
        with torch.autograd.graph.save_on_cpu():
            y = mixer(X)
    want_y, want = wanted(mixer, x, dy)
    assert torch.equal(y, want_y)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, [X, *mixer.parameters()], dy), want))


def test_autocast_of_the_forward(gcg_lib):
    """The backward's run of a module that is run again sees the forward's autocast state, and none outside of it."""
    class Probe(torch.nn.Module):
        def forward(self, x):
            seen.append((torch.is_autocast_enabled("cuda"), torch.get_autocast_dtype("cuda")))
            return x * 2
    for dtype in (torch.bfloat16, torch.float16):
        seen = []
        x = torch.ones(2, 128, device=DEV, requires_grad=True)
        with torch.autocast("cuda", dtype=dtype):
            y = module._recomputed8(Probe(), x)
        y.sum().backward()
        assert seen == [(True, dtype)] * 2 and torch.equal(x.grad, torch.full_like(x, 2.0))
    seen = []
    y = module._recomputed8(Probe(), x)
    with torch.autocast("cuda", dtype=torch.float16):
        y.sum().backward()
    assert [on for on, _ in seen] == [False, False]
