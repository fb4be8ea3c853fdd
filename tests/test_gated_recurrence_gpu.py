"""The gated recurrence's kernels against the recurrence in 64 bits, token by token, and its adjoint.

Tolerances.  The decay a and 1 - a carry k = 8 + |z| roundings of 2^-24 (exp's argument |z| of them), the products and sums of a row four more.  So an
error e_t of the state obeys e_t <= a_t e_{t-1} + 2^-24 ((k + 4) a_t H_{t-1} + (k + 4) u_t), H the recurrence of the magnitudes and u_t = (1 - a_t) |x_t|:
the same recurrence once more.  Chunks put pairs together in another order, with as many roundings for every row they pass: the row's own, a
product of decays and a sum, at each of three levels: 8 more.  G likewise, from the other end.  Outputs are then products of these with
numbers rounded to their type (U)."""
import pytest
import torch

from layer8 import TINY, U, check
from savanna_amd import _lib
from savanna_amd.operators.gated_recurrence import (GatedRecurrence, gated_recurrence, gated_recurrence_features, gated_recurrence_step)

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
E = 2.0 ** -24


def data(bs, L, D, dtype, seed=0, shift=2.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device=DEV)                                       # noqa: E731
    x, f, gate, dy = (r(bs, L, D).to(dtype) for _ in range(4))
    return dict(x=x, f=f, gate=gate, dy=dy, bias=shift + 2 * r(D), initial=r(bs, D), dstate=r(bs, D))


def scan(a, u, h):
    out = torch.empty_like(u)
    for t in range(u.shape[1]):
        h = a[:, t] * h + u[:, t]
        out[:, t] = h
    return out


def reference(d, gate=True, bias=True, initial=True, lengths=None, dfinal=True):
    """{name: (value, tolerance)} in 64 bits"""
    x, f, dy = (d[n].double() for n in ("x", "f", "dy"))
    bs, L, D = x.shape
    dtype = d["x"].dtype
    u_t, tiny = U[dtype], TINY[dtype]
    g = d["gate"].double() if gate else torch.ones_like(x)
    z = f + (d["bias"].double() if bias else 0)
    a, b = torch.sigmoid(z), torch.sigmoid(-z)
    n = torch.full((bs,), L, device=DEV) if lengths is None else lengths.clamp(0, L)
    inside = (torch.arange(L, device=DEV)[None] < n[:, None])[..., None]
    a, b = torch.where(inside, a, 1.0), torch.where(inside, b, 0.0)
    x, dy, g = (torch.where(inside, t, 0.0) for t in (x, dy, g))
    h0 = d["initial"].double() if initial else torch.zeros(bs, D, dtype=torch.float64, device=DEV)
    k = (20 + torch.where(inside, z, 0.0).abs()) * E
    before = lambda h, first: torch.cat([first[:, None], h[:, :-1]], 1)                            # noqa: E731
    h = scan(a, b * x, h0)
    H = scan(a, b * x.abs(), h0.abs())
    zero = torch.zeros_like(h0)
    e = scan(a, k * (a * before(H, h0.abs()) + b * x.abs()), zero)
    last = h[:, -1] if L else h0
    out = {"y": (g * h, u_t * (g * h).abs() + 1.01 * g.abs() * e + 2 * E * (g * h).abs() + tiny), "final": (last, e[:, -1] + E * last.abs())}
    K0 = d["dstate"].double() if dfinal else zero
    # K_t of rows t = L - 1 .. 0 by the same recurrence: K_{t-1} = a_t (K_t + g_t dy_t)
    ar, gd = a.flip(1), (g * dy).flip(1)
    K = scan(ar, ar * gd, K0)
    KK = scan(ar, ar * gd.abs(), K0.abs())
    kr = k.flip(1)
    eK = scan(ar, kr * ar * (before(KK, K0.abs()) + gd.abs()), zero)
    G = (before(K, K0) + gd).flip(1)
    GG = (before(KK, K0.abs()) + gd.abs()).flip(1)
    eG = before(eK, zero).flip(1) + 2 * E * GG
    hb, Hb, eb = before(h, h0), before(H, h0.abs()), before(e, zero)
    dx, df, dg = b * G, G * (hb - x) * a * b, dy * h
    tol_df = a * b * ((eG + 4 * k * GG) * (Hb + x.abs()) + GG * (eb + 2 * E * (Hb + x.abs())))
    out["dx"] = (dx, u_t * dx.abs() + 1.01 * b * (eG + k * GG) + tiny)
    out["df"] = (df, u_t * df.abs() + 1.01 * tol_df + tiny)
    if gate:
        out["dgate"] = (dg, u_t * dg.abs() + 1.01 * dy.abs() * (e + 2 * E * H) + tiny)
    if bias:
        out["dbias"] = (df.sum((0, 1)), tol_df.sum((0, 1)) + (bs * L + 64) * E * df.abs().sum((0, 1)))
    if initial:
        first = K[:, -1]
        out["dinitial"] = (first, eK[:, -1] + E * first.abs())
    return out


def run(d, gate=True, bias=True, initial=True, lengths=None, final=True):
    t = {n: v.clone().requires_grad_(True) for n, v in d.items() if n in ("x", "f")}
    t["gate"] = d["gate"].clone().requires_grad_(True) if gate else None
    t["bias"] = d["bias"].clone().requires_grad_(True) if bias else None
    t["initial"] = d["initial"].clone().requires_grad_(True) if initial else None
    out = gated_recurrence(t["x"], t["f"], t["gate"], t["bias"], initial_state=t["initial"], lengths=lengths, output_final_state=final)
    leaves = [v for v in t.values() if v is not None]
    grads = torch.autograd.grad(out, leaves, [d["dy"], d["dstate"]] if final else d["dy"])
    got = dict(zip(["d" + n for n, v in t.items() if v is not None], grads))
    got["y"] = (out[0] if final else out).detach()
    if final:
        got["final"] = out[1].detach()
    return got


def compare(got, want, what):
    for name, v in got.items():
        check(v, *want[name], f"{name} {what}")


SHAPES = [(1, 1, 1), (2, 2, 3), (1, 7, 64), (3, 64, 130), (2, 65, 129), (1, 127, 66), (2, 128, 33), (2, 129, 128), (1, 200, 257), (3, 513, 20),
          (1, 1100, 130), (2, 1025, 5), (1, 2500, 64)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bs,L,D", SHAPES)
def test_forward_and_backward(bs, L, D, dtype):
    d = data(bs, L, D, dtype, seed=L + D)
    got = run(d)
    compare(got, reference(d), f"{bs} x {L} x {D}")
    with torch.no_grad():
        y, last = gated_recurrence(d["x"], d["f"], d["gate"], d["bias"], initial_state=d["initial"], output_final_state=True)
    assert torch.equal(y, got["y"]) and torch.equal(last, got["final"])
    again = run(d)
    assert all(torch.equal(again[n], v) for n, v in got.items())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bs,L,D,lengths", [(2, 256, 129, None), (2, 255, 70, [255, 130]), (6, 700, 1601, [700, 0, 1, 256, 257, 513]), (1, 3000, 1300, None),
                                            (2, 2300, 896, [2300, 2049]), (1, 12500, 40, None), (1, 9000, 70, [8321]), (3, 17000, 20, [16999, 12345, 0]),
                                            (2, 17000, 20, [16999, 300])])
def test_sizes_whose_chunks_are_long(bs, L, D, lengths, dtype):
    """Those that the card holds at once in chunks of 256 rows: a sequence in one chunk, in several, in more than a group of them."""
    d = data(bs, L, D, dtype, seed=L + D)
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=DEV)
    got = run(d, lengths=n)
    compare(got, reference(d, lengths=n), f"{bs} x {L} x {D}")
    again = run(d, lengths=n)
    assert all(torch.equal(again[n], v) for n, v in got.items())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gate,bias,initial,final", [(False, False, False, False), (True, False, False, False), (False, True, True, False), (True, True, False, True),
                                                     (False, False, True, True)])
def test_what_may_be_absent(gate, bias, initial, final, dtype):
    d = data(2, 300, 70, dtype, seed=3)
    compare(run(d, gate, bias, initial, final=final), reference(d, gate, bias, initial, dfinal=final), f"{gate} {bias} {initial} {final}")


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("lengths", [[700, 0, 1, 128], [64, 63, 65, 700], [129, 1000, -5, 400], [0, 0, 0, 0], [640, 512, 511, 513]])
def test_lengths(lengths, dtype):
    d = data(4, 700, 66, dtype, seed=sum(lengths))
    n = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    inside = torch.arange(700, device=DEV)[None] < n[:, None]
    want = reference(d, lengths=n)
    for name in ("x", "f", "gate", "dy"):                   # nothing behind a length is read
        d[name] = torch.where(inside[..., None], d[name], float("nan"))
    got = run(d, lengths=n)
    compare(got, want, str(lengths))
    for name in ("y", "dx", "df", "dgate"):
        assert not got[name][~inside].any()
    assert torch.equal(got["final"][n <= 0], d["initial"][n <= 0]) and torch.equal(got["dinitial"][n <= 0], d["dstate"][n <= 0])


@pytest.mark.parametrize("dtype,shift", [(torch.float32, 9.0), (torch.float32, -9.0), (torch.bfloat16, 9.0), (torch.float16, -6.0)])
def test_long_and_short_memories(dtype, shift):
    d = data(1, 3000, 40, dtype, shift=shift)
    compare(run(d), reference(d), f"shift {shift}")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 33])
def test_features_and_views(dtype, D):
    bs, L = 2, 333
    d = data(bs, L, D, dtype, seed=D)
    want = reference(d, initial=False, dfinal=False)
    features = torch.cat([d["x"], d["f"], d["gate"]], -1).requires_grad_(True)
    bias = d["bias"].clone().requires_grad_(True)
    y = gated_recurrence_features(features, bias)
    g, db = torch.autograd.grad(y, (features, bias), d["dy"])
    dx, df, dg = g.unflatten(-1, (3, D)).unbind(-2)
    got = {"y": y.detach(), "dx": dx, "df": df, "dgate": dg, "dbias": db}
    compare(got, want, "features")
    with torch.no_grad():
        assert torch.equal(gated_recurrence_features(features, bias), y)
    # the same through views of the features, time-major storage, odd offsets and a transposed dy
    separate = run(d, initial=False, final=False)
    for name, v in separate.items():
        assert torch.equal(got[name], v), name
    views = dict(d, dy=d["dy"].transpose(0, 1).contiguous().transpose(0, 1))
    views["x"], views["f"], views["gate"] = features.detach().unflatten(-1, (3, D)).unbind(-2)
    shifted = torch.empty(bs * L * D + 1, dtype=dtype, device=DEV)[1:].view(bs, L, D)
    views["x"] = shifted.copy_(views["x"])
    t = [views[n].detach().requires_grad_(True) for n in ("x", "f", "gate")]
    y2 = gated_recurrence(*t, d["bias"])
    assert torch.equal(y2, got["y"])
    for name, v in zip(("dx", "df", "dgate"), torch.autograd.grad(y2, t, views["dy"])):
        assert torch.equal(v, got[name])
    strided = torch.stack([d["x"], d["x"]], -1)[..., 0]     # a last dimension that is not contiguous
    assert torch.equal(gated_recurrence(strided, d["f"], d["gate"], d["bias"]), got["y"])
    same = d["x"][:, :1].expand(bs, L, D)                   # one row for all
    assert torch.equal(gated_recurrence(same, d["f"]), gated_recurrence(same.contiguous(), d["f"]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bs,D", [(1, 1), (3, 70), (5, 257), (70, 1000)])
@pytest.mark.parametrize("gate,bias", [(True, True), (False, False)])
def test_step(bs, D, dtype, gate, bias):
    d = data(bs, 1, D, dtype)
    x, f, g = (d[n][:, 0] for n in ("x", "f", "gate"))
    state = d["initial"].clone()
    y = gated_recurrence_step(x, f, state, g if gate else None, d["bias"] if bias else None)
    want = reference(d, gate, bias)
    check(y, want["y"][0][:, 0], want["y"][1][:, 0], "y")
    check(state, *want["final"], "state")
    features = torch.cat([x, f, g], -1)
    a, b, c = features.unflatten(-1, (3, D)).unbind(-2)
    state2 = d["initial"].clone()
    assert torch.equal(gated_recurrence_step(a, b, state2, c if gate else None, d["bias"] if bias else None), y) and torch.equal(state, state2)


def test_prompt_and_tokens_agree():
    D, L = 96, 300
    m = GatedRecurrence(D, device=DEV).to(torch.bfloat16)
    assert m.decay_bias.dtype == torch.float32
    features = torch.randn(2, L, 3 * D, device=DEV).bfloat16()
    whole = m(features)
    with torch.no_grad():
        y, state = m.prefill(features[:, :200])
        version = state._version
        rest = torch.stack([m.step(features[:, t], state) for t in range(200, L)], 1)
        assert state._version == version + 100
        _, last = m.prefill(features)
        # decays and states of either way carry the roundings counted above, 100 rows' of them
        assert (state - last).abs().max() <= 100 * 28 * E * last.abs().max()
        assert (torch.cat([y, rest], 1).float() - whole.float()).abs().max() <= 2.0 ** -7 * whole.float().abs().max()
        n = torch.tensor([300, 77], dtype=torch.int32, device=DEV)
        y, state = m.prefill(features, lengths=n)
        _, short = m.prefill(features[1:, :77])
        assert torch.equal(state[1], short[0])
    whole.sum().backward()
    assert m.decay_bias.grad.shape == (D,)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_infinities_and_nan_stay_in_their_channel_and_behind_their_row(dtype):
    d = data(2, 700, 40, dtype)
    clean = gated_recurrence(d["x"], d["f"], d["gate"], d["bias"])
    d["x"][0, 300, 3], d["x"][1, 100, 7], d["f"][0, 200, 9] = float("inf"), float("nan"), float("nan")
    y, last = gated_recurrence(d["x"], d["f"], d["gate"], d["bias"], output_final_state=True)
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[0, 300:, 3], bad[1, 100:, 7], bad[0, 200:, 9] = True, True, True
    assert torch.equal(~torch.isfinite(y), bad) and torch.equal(y[~bad], clean[~bad])
    assert torch.isinf(y[0, 300:, 3]).all() and torch.isnan(y[1, 100:, 7]).all() and last[0, 3] == float("inf")
    # decays of zero and one: no memory, and nothing but memory
    f = torch.zeros(1, 300, 2, device=DEV).to(dtype)
    f[:, 150, 0], f[:, :, 1] = -float("inf"), float("inf")
    x = torch.ones(1, 300, 2, device=DEV).to(dtype)
    x[:, 150] = 5
    y = gated_recurrence(x, f, initial_state=torch.full((1, 2), 3.0, device=DEV))
    assert y[0, 150, 0] == 5 and (y[0, :, 1] == 3).all()


def test_gradient_against_differences():
    d = data(1, 150, 4, torch.float32)
    got = run(d)

    def f(**change):
        t = {n: v.double() for n, v in d.items()} | change
        z = t["f"] + t["bias"]
        h = scan(torch.sigmoid(z), torch.sigmoid(-z) * t["x"], t["initial"])
        return (t["gate"] * h * t["dy"]).sum() + (h[:, -1] * t["dstate"]).sum()

    for name, at in (("x", (0, 0, 1)), ("x", (0, 149, 0)), ("f", (0, 75, 2)), ("gate", (0, 64, 3)), ("bias", (1,)), ("initial", (0, 2))):
        e = torch.zeros_like(d[name], dtype=torch.float64)
        e[at] = 1e-5
        base = d[name].double()
        # a difference is off by (1e-5)^2 / 6 of the third derivative and by 64-bit roundings over 1e-5
        assert abs((f(**{name: base + e}) - f(**{name: base - e})) / 2e-5 - got["d" + name][at].double()) <= 2e-5 * max(1.0, got["d" + name].abs().max().item())


def test_refusals():
    x = torch.randn(2, 5, 8, device=DEV)
    state = torch.zeros(2, 8, device=DEV)
    g = x[:, 0].clone().requires_grad_(True)
    for bad in (lambda: gated_recurrence(x, x[:, :4]), lambda: gated_recurrence(x, x.half()), lambda: gated_recurrence(x, x, x[..., :4]),
                lambda: gated_recurrence(x, x, bias=torch.zeros(7, device=DEV)), lambda: gated_recurrence(x, x, bias=torch.zeros(8, device=DEV).half()),
                lambda: gated_recurrence(x, x, initial_state=state.half()), lambda: gated_recurrence(x, x, initial_state=state[:1]),
                lambda: gated_recurrence(x, x, lengths=torch.tensor([5, 5], device=DEV)), lambda: gated_recurrence(x.double(), x.double()),
                lambda: gated_recurrence_features(x), lambda: gated_recurrence_step(x[:, 0], x[:, 0], state.half()), lambda: gated_recurrence(x.cpu(), x.cpu()),
                lambda: gated_recurrence_step(g, x[:, 0], state), lambda: gated_recurrence_step(x, x, state)):
        with pytest.raises((RuntimeError, ValueError, TypeError)):
            bad()
    y, last = gated_recurrence(x[:, :0], x[:, :0], initial_state=state + 2, output_final_state=True)
    assert y.shape == (2, 0, 8) and (last == 2).all()
    e = x[:, :0].clone().requires_grad_(True)
    b, s = torch.zeros(8, device=DEV, requires_grad=True), (state + 1).requires_grad_(True)
    y, last = gated_recurrence(e, e, bias=b, initial_state=s, output_final_state=True)
    last.sum().backward()
    assert (s.grad == 1).all() and not b.grad.any()
    assert gated_recurrence(x[:0], x[:0]).shape == (0, 5, 8)


@pytest.mark.parametrize("nodes", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bs,L,D,lengths", [(1, 70, 3, None), (2, 70, 66, None), (3, 70, 33, [70, 0, 9]), (2, 300, 64, [300, 129]), (2, 70, 1, None),
                                            (1, 1100, 70, None)])
def test_rows_that_share_their_elements(bs, L, D, lengths, dtype, nodes, monkeypatch):
    """What the rows behind a sequence's end hold in memory is no part of it: gradients of one row for all, as that of a sum over the
    rows is, and rows that overlap, are those of the same numbers in rows of their own.  So also with such gates and inputs."""
    if not nodes:
        monkeypatch.setattr(_lib, "native_nodes", lambda t: False)
    d = data(bs, L, D, dtype, seed=L + D)
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=DEV)
    rows = lambda name: d[name][:, :1].expand(bs, L, D)                                             # noqa: E731
    overlapping = lambda name: torch.cat([d[name][..., 0], d[name][:, :D - 1, 0]], 1).unfold(1, D, 1) if D <= L else rows(name)   # noqa: E731

    def gradients(x, f, gate, dy):
        t = [v.detach().requires_grad_(True) for v in (x, f, d["bias"], d["initial"])]
        y, last = gated_recurrence(t[0], t[1], gate, t[2], initial_state=t[3], lengths=n, output_final_state=True)
        return y, t, torch.autograd.grad([y, last], t, [dy, d["dstate"]], retain_graph=True)

    for view in (rows, overlapping):
        for x, f, gate in ((d["x"], d["f"], None), (d["x"], d["f"], view("gate")), (view("x"), view("f"), d["gate"]), (view("x"), view("f"), None)):
            own = [v if v is None else v.contiguous() for v in (x, f, gate)]
            y, t, got = gradients(x, f, gate, view("dy"))
            _, _, want = gradients(*own, view("dy").contiguous())
            assert all(torch.equal(a, b) for a, b in zip(got, want)), (view, gate is None, [(a - b).abs().max().item() for a, b in zip(got, want)])
            if view is rows:
                summed = torch.autograd.grad(y.sum(1), t, d["dy"][:, 0], retain_graph=True)
                alone = torch.autograd.grad(y, t, view("dy").contiguous(), retain_graph=True)
                assert all(torch.equal(a, b) for a, b in zip(summed, alone))
                if D == 1:
                    whole = torch.autograd.grad(y.sum(), t, retain_graph=True)
                    assert all(torch.equal(a, b) for a, b in zip(whole, torch.autograd.grad(y, t, torch.ones_like(y))))
    c = dict(d, dy=rows("dy").contiguous())
    y, t, got = gradients(d["x"], d["f"], None, rows("dy"))
    want = reference(c, gate=False, lengths=n)
    compare(dict(zip(("dx", "df", "dbias", "dinitial"), got)), want, f"{bs} x {L} x {D}")
