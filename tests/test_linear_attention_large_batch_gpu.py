"""Linear attention over more heads than a launch of the walk takes (65535 heads times entries): the bits of the same batch in parts."""
import pytest
import torch

from savanna_amd.operators.linear_attention import linear_attention, linear_attention_features, linear_attention_step
from test_linear_attention_gpu import DEV, data, decays, step

pytestmark = pytest.mark.gpu
SPANS = ((0, 700), (700, 1400), (1400, 2000))


@pytest.mark.parametrize("dk,dv", [(8, 8), (5, 7)])
@pytest.mark.parametrize("H", [37, 48])
def test_sequences(gcg_lib, H, dk, dv):
    q, k, v, do, initial, dfinal = data(2000, 3, H, dk, dv, torch.bfloat16)
    n = torch.randint(0, 4, (2000,), dtype=torch.int32, device=DEV)
    ld = decays(H)
    whole = step(q, k, v, do, ld, None, initial, dfinal, n)
    for a, b in SPANS:
        part = step(*(t[a:b] for t in (q, k, v, do)), ld, None, initial[a:b], dfinal[a:b], n[a:b].contiguous())
        assert all(torch.equal(x[a:b], y) for x, y in zip(whole, part))


def test_projected_features(gcg_lib):
    features = torch.randn(2000, 3, 3 * 37 * 8, device=DEV).to(torch.bfloat16).requires_grad_(True)
    do = torch.randn(2000, 3, 37, 8, device=DEV).to(torch.bfloat16)
    o = linear_attention_features(features, 37, decays(37))
    (df,) = torch.autograd.grad(o, features, do)
    for a, b in SPANS:
        f = features[a:b].detach().requires_grad_(True)
        y = linear_attention_features(f, 37, decays(37))
        assert torch.equal(o[a:b], y) and torch.equal(df[a:b], torch.autograd.grad(y, f, do[a:b])[0])


@pytest.mark.parametrize("bs,H", [(1024, 64), (70000, 1), (3, 30000)])
def test_single_tokens(gcg_lib, bs, H):
    q, k, v, _, state, _ = data(bs, 1, H, 8, 12, torch.bfloat16)
    ld = decays(H)
    whole, parts = state.clone(), state.clone()
    o = linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, whole)
    n = 65535 // H
    y = [linear_attention_step(q[a:a + n, 0], k[a:a + n, 0], v[a:a + n, 0], ld, parts[a:a + n]) for a in range(0, bs, n)]
    assert torch.equal(o, torch.cat(y)) and torch.equal(whole, parts)


def test_refusals(gcg_lib):
    """One entry of more heads than the walk takes; more heads than a launch of single tokens takes."""
    q = torch.zeros(1, 2, 65536, 8, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError, match="not supported"):
        linear_attention(q, q, q, torch.zeros(65536, device=DEV))
    p = q.data_ptr()
    st = (__import__("ctypes").c_int64 * 8)(*([0] * 8))
    assert gcg_lib.gcg_linear_attn_step(p, p, p, p, st, p, p, 1 << 20, 16, 8, 8, 1.0, 1, None) == -2
    assert gcg_lib.gcg_linear_attn_step(p, p, p, p, st, p, p, 1 << 32, 1, 8, 8, 1.0, 1, None) == -2


def test_rows_of_features_further_apart_than_the_walk_takes(gcg_lib):
    """Features of 6000 heads of 256: the forward takes them by a copy, and so does the backward."""
    features = torch.randn(1, 3, 3 * 6000 * 256, device=DEV).to(torch.bfloat16).requires_grad_(True)
    do = torch.randn(1, 3, 6000, 256, device=DEV).to(torch.bfloat16)
    ld = decays(6000)
    o = linear_attention_features(features, 6000, ld)
    (df,) = torch.autograd.grad(o, features, do)
    q, k, v = features.detach().view(1, 3, 3, 6000, 256).unbind(2)
    want = step(q, k, v, do, ld)
    assert torch.equal(o, want[0]) and torch.equal(df.view(1, 3, 3, 6000, 256), torch.stack(want[2:5], 2))
