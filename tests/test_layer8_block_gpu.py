"""The operators of a layer in 8-bit floating point together: the layer against its parts, training and decoding, captured graphs, other streams, the
ctypes binding, torch's own operator checks and tracing."""
import os
import subprocess
import sys

import pytest
import torch

from savanna_amd import _lib, _ops
from savanna_amd.operators.block import MixerBlock, MixerBlockFloat8
from savanna_amd.operators.float8 import E4M3, E5M2, linear_float8, norm_linear_float8, to_float8
from savanna_amd.operators.gated_recurrence import GatedRecurrence, gated_recurrence, gated_recurrence_features, gated_recurrence_step
from savanna_amd.operators.hyena import CgcgConfig, HyenaMixer, HyenaMROperator
from savanna_amd.operators.linear_attention import LinearAttention
from savanna_amd.operators.norm import rms_norm, rms_norm_float8

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def mixer(kind, width):
    if kind == "hyena":
        op = HyenaMROperator(width, width // 16, 128, CgcgConfig(cgcg_dtype="bfloat16"), small_init=False, device=DEV)
        return HyenaMixer(op, dtype=torch.bfloat16, device=DEV)
    return LinearAttention(width, width // 32, device=DEV) if kind == "attention" else GatedRecurrence(width, device=DEV)


@pytest.mark.parametrize("kind", ["hyena", "attention", "recurrence"])
def test_layers_are_their_parts(kind):
    torch.manual_seed(0)
    layers = [MixerBlockFloat8(96, mixer(kind, 96), grad_dtype=fmt, device=DEV) for fmt in (E4M3, E5M2)]
    x = torch.randn(2, 150, 96, device=DEV).bfloat16().requires_grad_(True)
    a, r = layers[0](x)
    assert r is x
    b, r2 = layers[1](a, r)
    (b.float().square().sum() + r2.float().sum()).backward()
    grads = [p.grad.clone() for layer in layers for p in layer.parameters()] + [x.grad.clone()]
    assert all(torch.isfinite(g).all() and g.any() for g in grads)
    for p in [x] + [p for layer in layers for p in layer.parameters()]:
        p.grad = None
    h, res = x, None
    for layer in layers:
        f = norm_linear_float8(h, layer.norm.weight, layer.projection.weight, layer.norm.eps, res, layer.grad_dtype)
        f, res = (f, h) if res is None else f
        h = linear_float8(layer.mixer(f), layer.out.weight, layer.grad_dtype)
    assert torch.equal(h, b) and torch.equal(res, r2)
    (h.float().square().sum() + res.float().sum()).backward()
    again = [p.grad for layer in layers for p in layer.parameters()] + [x.grad]
    assert all(torch.equal(g, w) for g, w in zip(again, grads))
    # the stream is the sum of what the layers added
    assert torch.equal(r2, (a.float() + x.float()).bfloat16())


@pytest.mark.parametrize("kind", ["attention", "recurrence"])
def test_decoding(kind):
    torch.manual_seed(1)
    block = MixerBlockFloat8(96, mixer(kind, 96), device=DEV).eval()
    x, res = torch.randn(3, 60, 96, device=DEV).bfloat16(), torch.randn(3, 60, 96, device=DEV).bfloat16()
    with torch.no_grad():
        whole, r = block(x, res)
        block.lay_out()
        same, _ = block(x, res)
        assert torch.equal(whole, same)
        y, r1, state = block.prefill(x[:, :40], res[:, :40])
        assert torch.equal(r1, r[:, :40])
        steps = [block.step(x[:, t], state, res[:, t]) for t in range(40, 60)]
        assert torch.equal(torch.stack([s[1] for s in steps], 1), r[:, 40:])
        got, want = torch.cat([y, torch.stack([s[0] for s in steps], 1)], 1).float(), whole.float()
        # the mixer's output, rounded to bf16 after sums in another order, differs in a unit here and there, and its 8 bits in a step (2^-4): of few
        # numbers, so of the whole 2^-4 of a hundredth
        assert (got - want).norm() <= 2.0 ** -4 * 0.5 * want.norm()
        n = torch.tensor([60, 17, 1], dtype=torch.int32, device=DEV)
        _, _, state = block.prefill(x, res, lengths=n)
        _, _, short = block.prefill(x[1:2, :17], res[1:2, :17])
        assert (state[1] - short[0]).norm() <= 2.0 ** -6 * short.norm()      # (a product of another size adds in another order: bf16 features)


def test_recurrence_in_the_other_layer():
    torch.manual_seed(2)
    block = MixerBlock(64, GatedRecurrence(64, device=DEV), device=DEV)
    x = torch.randn(2, 100, 64, device=DEV, requires_grad=True)
    whole = block(x)
    whole.sum().backward()
    assert torch.isfinite(x.grad).all() and block.mixer.decay_bias.grad.any()
    with torch.no_grad():
        y, state = block.prefill(x[:, :70])
        rest = torch.stack([block.step(x[:, t], state) for t in range(70, 100)], 1)
        assert (torch.cat([y, rest], 1) - whole).abs().max() <= 1e-4 * whole.abs().max()


def everything(x, res, gain, w, w8, features, bias, state, lengths, dy, df):
    """A run of all of them with their gradients, as tensors."""
    y, r = norm_linear_float8(x, gain, w, residual=res)
    grads = torch.autograd.grad([y, r], (x, res, gain, w), [dy, x.detach()])
    s = gated_recurrence_features(features, bias)
    more = torch.autograd.grad(s, (features, bias), df)
    n, _ = rms_norm(x, gain, residual=res)
    also = torch.autograd.grad(n, (x, gain), x.detach())
    with torch.no_grad():
        q = rms_norm_float8(x, gain)
        z = linear_float8(x, w8)
        one = linear_float8(x[:1], w8)
        a, b, c = features.unflatten(-1, (3, -1)).unbind(-2)
        h, last = gated_recurrence(a, b, c, bias, initial_state=state, lengths=lengths, output_final_state=True)
        t = state.clone()
        token = gated_recurrence_step(a[:, 0], b[:, 0], t, c[:, 0], bias)
    return [y.detach(), r.detach(), *grads, s.detach(), *more, n.detach(), *also, q.codes.view(torch.uint8), q.scales.view(torch.uint8), z, one, h, last, t, token]


def inputs(seed=0, rows=200, K=300, N=500, bs=2, L=1100, D=70):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device=DEV)                       # noqa: E731
    h = lambda *s: r(*s).bfloat16()                                                 # noqa: E731
    w = (r(N, K) / 16).bfloat16()
    leaf = lambda t: t.requires_grad_(True)                                         # noqa: E731
    return [leaf(h(rows, K)), leaf(h(rows, K)), leaf(h(K)), leaf(w), to_float8(w), leaf(h(bs, L, 3 * D)), leaf(2 + r(D)), r(bs, D),
            torch.tensor([L, L // 2], dtype=torch.int32, device=DEV), h(rows, N), h(bs, L, D)]


def test_two_captured_graphs_and_eager_work_between_their_replays():
    ins = [inputs(s) for s in (1, 2)]
    want = [everything(*i) for i in ins]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for i in ins:
            everything(*i)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for i in ins:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(everything(*i))
        graphs.append(g)
    for turn in range(4):
        for g in graphs:
            g.replay()
        eager = everything(*ins[turn % 2])
        torch.cuda.synchronize()
        for got, ref in zip(outs + [eager], want + [want[turn % 2]]):
            assert all(torch.equal(a, b) for a, b in zip(got, ref)), turn
    # other values in the same places
    new = inputs(3)
    with torch.no_grad():
        for a, b in zip(ins[0], new):
            for p, q in zip(a, b) if isinstance(a, tuple) else ((a, b),):
                if isinstance(p, torch.Tensor):
                    p.view(torch.uint8).copy_(q.view(torch.uint8)) if p.element_size() == 1 else p.copy_(q)
    graphs[0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs[0], everything(*new)))


@pytest.mark.skipif(not _lib.TORCH_OPS, reason="the check is the torch binding's")
def test_a_capture_with_leaves_of_a_living_graph_is_refused():
    i = inputs(11)
    x, res, gain, w, _, features, bias = i[:7]
    lives = [(x * 1).sum(), (gain * 1).sum(), (w * 1).sum(), (features * 1).sum(), (bias * 1).sum()]
    calls = [lambda: rms_norm(x, gain, residual=res), lambda: linear_float8(res.detach(), w), lambda: norm_linear_float8(res.detach(), gain, w.detach()),
             lambda: gated_recurrence_features(features.detach(), bias), lambda: gated_recurrence_features(features)]
    for call in calls:
        call()                                                                      # (not captured: allowed)
        g = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="still lives"), torch.cuda.graph(g):
            res.detach() + 1
            call()
        del g
    del lives
    torch.cuda.synchronize()
    want = everything(*i)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = everything(*i)
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("nodes", [True, False])
def test_no_second_derivative(nodes, monkeypatch):
    """A gradient that is recorded itself is the same, and its own gradient an error rather than zero."""
    x, res, gain, w, _, features, bias = inputs(12)[:7]
    if not nodes:
        monkeypatch.setattr(_lib, "native_nodes", lambda t: False)
    for f, leaf in ((lambda: rms_norm(x, gain), x), (lambda: linear_float8(x, w), w), (lambda: norm_linear_float8(x, gain, w), x),
                    (lambda: gated_recurrence_features(features, bias), features)):
        once = torch.autograd.grad(f().float().square().sum(), leaf)[0]
        kept = torch.autograd.grad(f().float().square().sum(), leaf, create_graph=True)[0]
        assert torch.equal(once, kept)
        with pytest.raises(RuntimeError, match="differentia"):
            torch.autograd.grad(kept.float().square().sum(), leaf)


def test_gradients_of_one_tensor_in_two_places():
    """x and the residual are one leaf, or two whose gradients are then written to."""
    x, _, gain = inputs(13)[:3]
    dy, dr = torch.randn_like(x), torch.randn_like(x)
    a, b = x.detach().clone().requires_grad_(True), x.detach().clone().requires_grad_(True)
    torch.autograd.backward(rms_norm(a, gain, residual=b), [dy, dr])
    torch.autograd.backward(rms_norm(x, gain, residual=x), [dy, dr])
    assert torch.equal(a.grad, b.grad) and torch.equal(x.grad, a.grad + b.grad)
    before = b.grad.clone()
    a.grad.zero_()
    assert torch.equal(b.grad, before)


@pytest.mark.parametrize("rows,K,N", [(0, 40, 30), (5, 40, 0), (5, 0, 30), (0, 0, 30)])
def test_products_of_nothing(rows, K, N):
    x = torch.randn(rows, K, device=DEV).bfloat16().requires_grad_(True)
    w = torch.randn(N, K, device=DEV).bfloat16().requires_grad_(True)
    for nograd in (False, True):
        with torch.set_grad_enabled(not nograd):
            y = linear_float8(x, w)
        assert y.shape == (rows, N) and not y.any()
    y = linear_float8(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), torch.ones_like(y))
    assert dx.shape == x.shape and dw.shape == w.shape and not dw.any() and (K == 0 or N == 0 or rows == 0) and not (N == 0 and dx.any())


def test_two_streams_at_once():
    ins = [inputs(s, L=3000, D=130) for s in (4, 5)]
    want = [everything(*i) for i in ins]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ins]
    got = []
    for _ in range(3):
        for st, i in zip(streams, ins):
            with torch.cuda.stream(st):
                got.append(everything(*i))
    torch.cuda.synchronize()
    for n, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[n % 2]))


def test_the_python_functions_and_the_nodes_are_the_same(monkeypatch):
    i = inputs(6)
    want = everything(*i)
    monkeypatch.setattr(_lib, "native_nodes", lambda t: False)
    assert all(torch.equal(a, b) for a, b in zip(everything(*i), want))


def test_ctypes_binding(tmp_path):
    """The same numbers through the other binding, in a process of its own."""
    if not _lib.TORCH_OPS:
        pytest.skip("this is the ctypes binding")
    here = os.path.dirname(os.path.abspath(__file__))
    out = tmp_path / "out.pt"
    code = ("import sys, torch; sys.path[:0] = [%r, %r]; import test_layer8_block_gpu as t; from savanna_amd import _lib; assert not _lib.TORCH_OPS;"
            "torch.save([v.cpu() for v in t.everything(*t.inputs(7))], %r)") % (os.path.dirname(here), here, str(out))
    subprocess.run([sys.executable, "-c", code], check=True, env={**os.environ, "GCG_BINDING": "ctypes"}, timeout=100)
    got = torch.load(out, weights_only=True)
    for a, b in zip(got, everything(*inputs(7))):
        assert torch.equal(a, b.cpu())


def test_schemas_and_meta_results(gcg_lib):
    r = lambda *s: torch.randn(*s, device=DEV).bfloat16()                           # noqa: E731
    x, g, w, s = r(70, 300), r(300), r(40, 300), r(1, 70, 32)
    codes, scales = torch.ops.gcg.to_float8(x, E4M3)
    wc, ws = torch.ops.gcg.to_float8(w, E4M3)
    _, _, rstd = torch.ops.gcg.rms_norm_fwd(x, x, g, 1e-6)
    bias, state = torch.randn(32, device=DEV), torch.randn(1, 32, device=DEV)
    features = r(1, 70, 96)
    _, _, states = torch.ops.gcg.scan_fwd(s, s, s, bias, state, None, True, True)
    nodes = {"rms_norm": (x, x, g, 1e-6), "linear_float8": (x, w, E4M3), "norm_linear_float8": (x, x, g, w, 1e-6, E5M2),
             "scan": (s, s, s, bias, state, None, True), "scan_packed": (features, bias)}
    entries = {"rms_norm_fwd": (x, x, g, 1e-6), "rms_norm_infer": (x, None, g, 1e-6), "rms_norm_float8": (x, x, g, 1e-6), "rms_norm_bwd": (x, x, x, rstd, g),
               "to_float8": (x, E5M2), "to_float8_both": (x, E4M3), "to_float8_columns": (x, E4M3), "float8_columns": (codes, scales, 300, E4M3),
               "from_float8": (codes, scales, 300, torch.float16), "matmul_float8": (codes, scales, wc, ws, 300, torch.bfloat16),
               "linear_float8_infer": (x, wc, ws, 300), "norm_linear_float8_infer": (x, x, g, wc, ws, 300, 1e-6), "scan_fwd": (s, s, s, bias, state, None, True, True),
               "scan_bwd": (s, s, s, s, bias, states, None, state, True, True), "scan_packed_fwd": (features, bias, True),
               "scan_packed_bwd": (s, features, bias, states, True), "scan_step": (s[:, 0], s[:, 0], None, bias, state)}
    assert set(nodes) == set(_ops.LAYER8_NODE_NAMES) and set(entries) == set(_ops.LAYER8_OP_NAMES)
    from torch._subclasses.fake_tensor import FakeTensorMode
    for name, a in {**nodes, **entries}.items():
        op = getattr(torch.ops.gcg, name)
        flat = lambda v: list(v) if isinstance(v, (list, tuple)) else [v]           # noqa: E731
        outs = flat(op(*[v.clone() if v is state else v for v in a]))
        with FakeTensorMode() as mode:
            metas = flat(op(*[mode.from_tensor(v) if isinstance(v, torch.Tensor) else v for v in a]))
        assert [(o.shape, o.dtype, o.device, o.stride()) for o in outs] == [(m.shape, m.dtype, m.device, m.stride()) for m in metas], name
        if "float8" not in name:                      # (torch's checks multiply what passes the dispatcher, which 8-bit types do not)
            torch.library.opcheck(op, a, test_utils=("test_schema", "test_faketensor"))


def test_operators_differentiate():
    """torch.ops.gcg's forward operators have their gradients themselves; those without one say so."""
    i = inputs(8)
    x, res, gain, w, _, features, bias, state = i[:8]
    y, r, _ = torch.ops.gcg.rms_norm_fwd(x, res, gain, 1e-6)
    a = torch.autograd.grad([y, r], (x, gain), [x.detach(), x.detach()])
    y, r = rms_norm(x, gain, residual=res)
    assert all(torch.equal(p, q) for p, q in zip(a, torch.autograd.grad([y, r], (x, gain), [x.detach(), x.detach()])))
    y, _ = torch.ops.gcg.scan_packed_fwd(features, bias, True)
    a = torch.autograd.grad(y, (features, bias), i[-1])
    assert all(torch.equal(p, q) for p, q in zip(a, torch.autograd.grad(gated_recurrence_features(features, bias), (features, bias), i[-1])))
    p = [t.contiguous() for t in features.unflatten(-1, (3, -1)).unbind(-2)]
    y, last, _ = torch.ops.gcg.scan_fwd(*p, bias, state, None, True, True)
    a = torch.autograd.grad([y, last], (features, bias), [i[-1], state])
    b = torch.autograd.grad(gated_recurrence(*p, bias, initial_state=state, output_final_state=True), (features, bias), [i[-1], state])
    assert all(torch.equal(u, v) for u, v in zip(a, b))
    with pytest.raises(RuntimeError, match="keep=True"):
        torch.ops.gcg.scan_fwd(*p, bias, state, None, True, False)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.ops.gcg.rms_norm_infer(x, None, gain, 1e-6)[0].sum().backward()


@pytest.mark.skipif(not _lib.TORCH_OPS, reason="the ctypes binding is not traced")
def test_traced():
    i = inputs(9)
    x, res, gain, w, _, features, bias = i[:7]

    def layer(x, res, gain, w, features, bias):
        y, r = norm_linear_float8(x, gain, w, residual=res)
        n, _ = rms_norm(x, gain, residual=res)
        return y, r, n, gated_recurrence_features(features, bias), linear_float8(x, w)

    args = (x, res, gain, w, features, bias)
    outs = [f(*args) for f in (layer, torch.compile(layer, fullgraph=True, backend="aot_eager"))]
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    grads = [torch.autograd.grad([t.float().sum() for t in o], args) for o in outs]
    assert all(torch.equal(a, b) for a, b in zip(*grads))


def test_no_forward_mode_and_no_lost_tangents():
    i = inputs(10)
    x, gain, w, features, bias, state = i[0].detach(), i[2].detach(), i[3].detach(), i[5].detach(), i[6].detach(), i[7]
    import torch.autograd.forward_ad as fwAD
    with fwAD.dual_level():
        d = fwAD.make_dual(x, torch.ones_like(x))
        s = fwAD.make_dual(features, torch.ones_like(features))
        t = fwAD.make_dual(features[:, 0, :70].contiguous(), torch.ones_like(features[:, 0, :70]))
        for f in (lambda: rms_norm(d, gain), lambda: linear_float8(d, w), lambda: norm_linear_float8(d, gain, w), lambda: gated_recurrence_features(s, bias)):
            with pytest.raises((NotImplementedError, RuntimeError)):
                f()
        with torch.no_grad(), pytest.raises(NotImplementedError):
            gated_recurrence_step(t, t, state, None, bias)


def test_example():
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
    import recurrent_float8
    assert recurrent_float8.main(["--width", "192", "--length", "150", "--steps", "2"])


def test_ctypes_binding_says_that_a_step_modifies_its_state(tmp_path):
    """Whatever saved the state for a backward pass finds it modified, as through the other binding; an inference tensor has no count of it."""
    here = os.path.dirname(os.path.abspath(__file__))
    code = ("import sys, torch; sys.path[:0] = [%r]; from savanna_amd import _lib; from savanna_amd.operators.gated_recurrence import gated_recurrence_step as step\n"
            "assert not _lib.TORCH_OPS\n"
            "x, state = torch.randn(3, 70, device='cuda:0'), torch.zeros(3, 70, device='cuda:0')\n"
            "w = torch.ones_like(state).requires_grad_(True)\n"
            "loss = (w * state).sum()\n"
            "for n in (1, 2, 3):\n"
            "    with torch.no_grad(): step(x, x, state)\n"
            "    assert state._version == n, state._version\n"
            "try: loss.backward()\n"
            "except RuntimeError as e: assert 'modified by an inplace operation' in str(e)\n"
            "else: raise AssertionError('a gradient of what is no longer there')\n"
            "with torch.inference_mode(): step(x, x, torch.zeros(3, 70, device='cuda:0'))\n") % os.path.dirname(here)
    subprocess.run([sys.executable, "-c", code], check=True, env={**os.environ, "GCG_BINDING": "ctypes"}, timeout=100)


def test_ctypes_binding_refuses_tangents():
    here = os.path.dirname(os.path.abspath(__file__))
    code = ("import sys, torch; sys.path[:0] = [%r]\n"
            "import torch.autograd.forward_ad as fwAD\n"
            "from savanna_amd import _lib\n"
            "from savanna_amd.operators.float8 import linear_float8, norm_linear_float8, to_float8\n"
            "from savanna_amd.operators.norm import rms_norm_float8\n"
            "from savanna_amd.operators.gated_recurrence import gated_recurrence_step\n"
            "assert not _lib.TORCH_OPS\n"
            "x, w = torch.randn(4, 300, device='cuda:0').bfloat16(), torch.randn(20, 300, device='cuda:0').bfloat16()\n"
            "q, lost = to_float8(w), []\n"
            "with fwAD.dual_level(), torch.no_grad():\n"
            "    d = fwAD.make_dual(x, torch.ones_like(x))\n"
            "    for name, f in dict(to_float8=lambda: to_float8(d), rms_norm_float8=lambda: rms_norm_float8(d), linear_float8=lambda: linear_float8(d, q),\n"
            "                        norm_linear_float8=lambda: norm_linear_float8(x, None, q, residual=d), weight=lambda: rms_norm_float8(x, d[0]),\n"
            "                        step=lambda: gated_recurrence_step(d, x, torch.zeros(4, 300, device='cuda:0'))).items():\n"
            "        try: f()\n"
            "        except NotImplementedError: continue\n"
            "        lost.append(name)\n"
            "    to_float8(x), rms_norm_float8(x), linear_float8(x, q), norm_linear_float8(x, None, q)\n"
            "assert not lost, lost\n") % os.path.dirname(here)
    subprocess.run([sys.executable, "-c", code], check=True, env={**os.environ, "GCG_BINDING": "ctypes"}, timeout=100)


def test_no_lost_tangents_of_tensors_that_need_gradients():
    """The graphs of these operators' arguments are left alone, their tangents are not."""
    import torch.autograd.forward_ad as fwAD
    x, w = (torch.randn(n, 300, device=DEV).bfloat16().requires_grad_(True) for n in (4, 1))
    with fwAD.dual_level():
        d, g = fwAD.make_dual(x, torch.ones_like(x)), fwAD.make_dual(w, torch.ones_like(w))[0]
        for grad in (True, False):
            with torch.set_grad_enabled(grad):
                for f in (lambda: to_float8(d), lambda: rms_norm_float8(d), lambda: rms_norm_float8(x, g), lambda: rms_norm_float8(x.detach(), residual=d)):
                    with pytest.raises((NotImplementedError, RuntimeError), match="forward-mode|jvp|forward AD"):
                        f()
                to_float8(x), rms_norm_float8(x, w[0])
