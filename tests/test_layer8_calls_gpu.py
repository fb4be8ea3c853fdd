"""Calls of the operators of a layer in 8-bit floating point that the documentation allows beside the usual ones: tensors of one dimension, parts of
8-bit tensors, outputs of which only one is used, arguments given twice, second passes over one graph, other memory orders."""
import pytest
import torch

from savanna_amd import _lib
from savanna_amd.operators.float8 import E4M3, E5M2, Float8, from_float8, linear_float8, matmul_float8, norm_linear_float8, to_float8
from savanna_amd.operators.gated_recurrence import GatedRecurrence, gated_recurrence, gated_recurrence_features, gated_recurrence_step
from savanna_amd.operators.norm import rms_norm, rms_norm_float8

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def rand(*shape, dtype=torch.bfloat16, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed + sum(shape))
    return torch.randn(*shape, generator=gen, device=DEV).to(dtype)


def bits(t):
    return t.view(torch.uint8)


@pytest.fixture(params=[True, False], ids=["nodes", "functions"])
def nodes(request, monkeypatch):
    if not request.param:
        monkeypatch.setattr(_lib, "native_nodes", lambda t: False)


def equal(a, b):
    return all(torch.equal(x.reshape(-1), y.reshape(-1)) for x, y in zip(a, b))


def test_one_row_without_its_dimension(nodes):
    x, res, g, w = (t.requires_grad_(True) for t in (rand(300), rand(300, seed=1), rand(300, seed=2), rand(70, 300)))
    row, res_row = x.detach()[None].requires_grad_(True), res.detach()[None].requires_grad_(True)
    for f, leaves in ((lambda x, r: [linear_float8(x, w)], (w,)), (lambda x, r: [rms_norm(x, g)], (g,)),
                      (lambda x, r: list(rms_norm(x, g, residual=r)), (g,)), (lambda x, r: list(norm_linear_float8(x, g, w, residual=r)), (g, w))):
        a, b = f(x, res), f(row, res_row)
        assert [t.shape for t in a] == [t.shape[1:] for t in b] and equal(a, b)
        dy = [torch.ones_like(t) for t in a]
        two = len(a) > 1
        assert equal(torch.autograd.grad(a, (x, *((res,) if two else ()), *leaves), dy),
                     torch.autograd.grad(b, (row, *((res_row,) if two else ()), *leaves), [t[None] for t in dy]))
    q, p = to_float8(x), to_float8(row)
    assert q.codes.shape == (384,) and q.scales.shape == (4,) and torch.equal(bits(q.codes), bits(p.codes[0]))
    assert torch.equal(from_float8(q, torch.float32), from_float8(p, torch.float32)[0])
    y = matmul_float8(q, to_float8(w))
    assert y.shape == (70,) and torch.equal(y, matmul_float8(p, to_float8(w))[0])
    n = rms_norm_float8(x.detach(), g, residual=res.detach())
    assert n[0].codes.shape == (384,) and n[1].shape == (300,)
    with torch.no_grad():
        assert torch.equal(linear_float8(x, to_float8(w)), y)


def test_parts_of_8_bit_tensors():
    a, b = rand(40, 700), rand(90, 700, seed=1)
    qa, qb = to_float8(a), to_float8(b, E5M2)
    whole = matmul_float8(qa, qb)
    for rows, cols in ((slice(3, 11), slice(1, 90)), (slice(39, 40), slice(17, 18)), (slice(0, 40), slice(89, 90))):
        p, r = Float8(qa.codes[rows], qa.scales[rows], 700), Float8(qb.codes[cols], qb.scales[cols], 700)
        assert torch.equal(from_float8(p, torch.float32), from_float8(qa, torch.float32)[rows])
        part = matmul_float8(p, r)
        assert (part.float() - whole[rows, cols].float()).abs().max() <= 2.0 ** -7 * whole.float().abs().max()
        ref = from_float8(p, torch.float32).double() @ from_float8(r, torch.float32).double().t()
        assert (part.double() - ref).abs().max() <= 2.0 ** -7 * ref.abs().max()
    deep = Float8(qa.codes.reshape(4, 10, -1), qa.scales.reshape(4, 10, -1), 700)
    assert torch.equal(matmul_float8(deep, qb), whole.reshape(4, 10, 90))


def test_only_one_output_of_the_recurrence_is_used(nodes):
    d = [rand(2, 130, 40, dtype=torch.float32, seed=s).requires_grad_(True) for s in range(3)]
    bias, h = rand(40, dtype=torch.float32).requires_grad_(True), rand(2, 40, dtype=torch.float32).requires_grad_(True)
    leaves = (*d, bias, h)
    f = lambda: gated_recurrence(*d, bias, initial_state=h, output_final_state=True)                    # noqa: E731
    dy, dl = rand(2, 130, 40, dtype=torch.float32, seed=9), rand(2, 40, dtype=torch.float32, seed=10)
    y, last = f()
    z, zl = torch.zeros_like(dy), torch.zeros_like(dl)
    for pair, given in (((y, last), (dy, zl)), ((y, last), (z, dl))):
        both = torch.autograd.grad(pair, leaves, given, retain_graph=True)
        i = 0 if given[1] is zl else 1
        assert equal(torch.autograd.grad(pair[i], leaves, given[i], retain_graph=True), both)
        assert equal(torch.autograd.grad(pair, leaves, given, retain_graph=True), both)                  # a second pass over the same graph
    y2, l2 = f()
    assert torch.equal(y, y2) and torch.equal(last, l2)
    for t in leaves:                                        # each gradient alone
        g, = torch.autograd.grad([y, last], t, [dy, dl], retain_graph=True)
        k = [u is t for u in leaves].index(True)
        assert torch.equal(g, torch.autograd.grad([y, last], leaves, [dy, dl], retain_graph=True)[k])


def test_arguments_given_twice(nodes):
    x = rand(2, 130, 40, dtype=torch.float32).requires_grad_(True)
    parts = [x.detach().clone().requires_grad_(True) for _ in range(3)]
    dy = rand(2, 130, 40, dtype=torch.float32, seed=1)
    a, b = gated_recurrence(x, x, x), gated_recurrence(*parts)
    assert torch.equal(a, b)
    g, = torch.autograd.grad(a, x, dy)
    dx, df, dg = torch.autograd.grad(b, parts, dy)
    assert torch.allclose(g, dx + df + dg, rtol=2.0 ** -21, atol=2.0 ** -21 * g.abs().max().item())      # (two additions, in either order)
    with torch.no_grad():
        state = rand(5, 40, dtype=torch.float32)
        before = state.clone()
        y = gated_recurrence_step(state, state, state, state)
        other = before.clone()
        assert torch.equal(y, gated_recurrence_step(before, before, other, before)) and torch.equal(state, other)
        q = to_float8(rand(64, 300))
        assert torch.equal(matmul_float8(q, q), matmul_float8(q, Float8(q.codes.clone(), q.scales.clone(), 300)))
    w = rand(300, 300).requires_grad_(True)
    v = w.detach().clone().requires_grad_(True)
    u = w.detach().clone().requires_grad_(True)
    a, b = linear_float8(w, w), linear_float8(u, v)
    assert torch.equal(a, b)
    dy = rand(300, 300, seed=4)
    (g,), (p, q) = torch.autograd.grad(a, w, dy), torch.autograd.grad(b, (u, v), dy)
    assert torch.equal(g, p + q)


def test_other_memory_orders(nodes):
    x, w, g = rand(6, 5, 300).requires_grad_(True), rand(70, 300).requires_grad_(True), rand(300, seed=3).requires_grad_(True)
    orders = [x.detach().transpose(0, 1).contiguous().transpose(0, 1), x.detach().permute(2, 0, 1).contiguous().permute(1, 2, 0),
              torch.stack([x.detach()] * 2, -1)[..., 1]]
    dy = rand(6, 5, 70, seed=5)
    for t in orders:
        assert not t.is_contiguous()
        t.requires_grad_(True)
        for f in (lambda x: linear_float8(x, w), lambda x: norm_linear_float8(x, g, w), lambda x: norm_linear_float8(x, g, w, residual=x)[0]):
            assert torch.equal(f(t), f(x))
            d = dy.permute(2, 0, 1).contiguous().permute(1, 2, 0)
            assert equal(torch.autograd.grad(f(t), (t, w), d), torch.autograd.grad(f(x), (x, w), dy))
        assert torch.equal(bits(to_float8(t).codes), bits(to_float8(x).codes))
    # y.sum() and y.sum(1) hand over gradients whose strides are zero
    for f in (lambda x: linear_float8(x, w), lambda x: norm_linear_float8(x, g, w), lambda x: rms_norm(x, g)):
        y = f(x)
        for s, d in ((y.sum(), torch.ones_like(y)), (y.sum(1), torch.ones_like(y))):
            assert equal(torch.autograd.grad(s, x, torch.ones_like(s), retain_graph=True), torch.autograd.grad(y, x, d, retain_graph=True))
    features = rand(2, 130, 96, dtype=torch.float32).requires_grad_(True)
    bias = rand(32, dtype=torch.float32)
    y = gated_recurrence_features(features, bias)
    for s in (y.sum(), y.sum(1), y.sum(0)):
        assert equal(torch.autograd.grad(s, features, torch.ones_like(s), retain_graph=True),
                     torch.autograd.grad(y, features, torch.ones_like(y), retain_graph=True))
    m = GatedRecurrence(32, device=DEV)
    assert torch.equal(m(features.detach().transpose(0, 1).contiguous().transpose(0, 1)), m(features))


def test_leaves_of_which_some_are_frozen(nodes):
    x, res, g, w = rand(20, 300), rand(20, 300, seed=1), rand(300, seed=2), rand(70, 300)
    dy, dr = rand(20, 70, seed=3), rand(20, 300, seed=4)
    every = [t.clone().requires_grad_(True) for t in (x, res, g, w)]
    want = torch.autograd.grad(norm_linear_float8(every[0], every[2], every[3], residual=every[1]), every, [dy, dr])
    for mask in range(1, 16):
        t = [v.clone().requires_grad_(bool(mask >> i & 1)) for i, v in enumerate((x, res, g, w))]
        needed = [v for v in t if v.requires_grad]
        out = norm_linear_float8(t[0], t[2], t[3], residual=t[1])
        if mask & 3 == 0:                                   # (nothing behind r: a gradient of y alone)
            got = torch.autograd.grad(out[0], needed, dy)
        else:
            got = torch.autograd.grad(out, needed, [dy, dr])
        assert equal(got, [v for i, v in enumerate(want) if mask >> i & 1]), mask
