"""Linear attention with a decay for each head, chunked and recurrent, against its recurrence in 64 bits.

Tolerances, by output element, from the sum of its terms' magnitudes A (that same recurrence on magnitudes, divided by 2^k
for nothing): a 16-bit walk rounds the scores, the state's copy and the result once each, by the type's unit roundoff U, and takes
products of what it read exactly; fp32 sums and the decays' powers add fewer than 64 roundings of 2^-24 a chunk and 2^-16 by the
weighted rows' remainder where the state is not itself a result.  So an element is off by at most U |ref| + (2 U + 2^-15) A in
16 bits and 2^-17 A in fp32, and a state by 2^-17 A of its own."""
import pytest
import torch

from savanna_amd import _lib
from savanna_amd.operators.act8 import pack8, unpack8
from savanna_amd.operators.linear_attention import LinearAttention, linear_attention, linear_attention_features, linear_attention_step

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -20}


def decays(H):
    """From f = 0 and f = exp(-3) to f = 1, in between memories of 4 to 4096 tokens."""
    some = [-float("inf"), -3.0, 0.0] + [-(0.25 * 2.0 ** (-10 * i / max(1, H - 4))) for i in range(H)]
    return torch.tensor(some[:H] if H >= 4 else some[3:3 + H], device=DEV)


def data(bs, L, H, dk, dv, dtype, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen, device=DEV)                 # noqa: E731
    q, k, v, do = (rand(bs, L, H, d).to(dtype) for d in (dk, dk, dv, dv))
    return q, k, v, do, rand(bs, H, dk, dv), rand(bs, H, dk, dv)


def recurrence(q, k, v, do, log_decay, scale, initial, dfinal, lengths=None):
    """o, final, dq, dk, dv, dinitial of the definition, as fp64 tensors; on magnitudes if the inputs are."""
    q, k, v, do = (t.double() for t in (q, k, v, do))
    bs, L, H, dk = q.shape
    f = torch.exp(log_decay.double())[:, None, None]
    n = lengths if lengths is not None else torch.full((bs,), L, device=q.device)
    n = n.clamp(0, L)[:, None, None, None]
    S = initial.double().clone() if initial is not None else torch.zeros(bs, H, dk, v.shape[-1], dtype=torch.float64, device=q.device)
    G = dfinal.double().clone() if dfinal is not None else torch.zeros_like(S)
    o, dq, dk_, dv_ = torch.zeros_like(v), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for t in range(L):
        inside = t < n
        S = torch.where(inside, f * S + k[:, t, :, :, None] * v[:, t, :, None, :], S)
        o[:, t] = torch.where(inside[..., 0], scale * (q[:, t, :, :, None] * S).sum(-2), 0.0)
        dq[:, t] = torch.where(inside[..., 0], scale * (S * do[:, t, :, None, :]).sum(-1), 0.0)
    for t in reversed(range(L)):
        inside = t < n
        G = torch.where(inside, G + scale * q[:, t, :, :, None] * do[:, t, :, None, :], G)
        dk_[:, t] = torch.where(inside[..., 0], (G * v[:, t, :, None, :]).sum(-1), 0.0)
        dv_[:, t] = torch.where(inside[..., 0], (G * k[:, t, :, :, None]).sum(-2), 0.0)
        G = torch.where(inside, f * G, G)
    return o, S, dq, dk_, dv_, G


def reference(q, k, v, do, log_decay, scale, initial, dfinal, lengths=None):
    size = lambda t: t.abs() if t is not None else None                          # noqa: E731
    if lengths is not None:                                                      # whatever lies past the end
        inside = torch.arange(q.shape[1], device=q.device)[None, :, None, None] < lengths[:, None, None, None]
        q, k, v, do = (torch.where(inside, t, torch.zeros_like(t)) for t in (q, k, v, do))
    ref = recurrence(q, k, v, do, log_decay, scale, initial, dfinal, lengths)
    mag = recurrence(size(q), size(k), size(v), size(do), log_decay, abs(scale), size(initial), size(dfinal), lengths)
    dtype, out = q.dtype, []
    for i, (r, a) in enumerate(zip(ref, mag)):
        if i in (1, 5) or dtype == torch.float32:
            out.append((r, 2.0 ** -17 * a + U[torch.float32]))
        else:
            out.append((r, U[dtype] * r.abs() + (2 * U[dtype] + 2.0 ** -15) * a + TINY[dtype]))
    return out


def check(got, want, what):
    for name, g, (ref, tol) in zip(("o", "final", "dq", "dk", "dv", "dinitial"), got, want):
        if g is None:
            continue
        off = (g.double() - ref).abs()
        assert g.shape == ref.shape
        within = bool((off <= tol).all())
        assert within, f"{what} {name}: off by {off.max().item():.3e}, {(off - tol).max().item():.3e} over the tolerance"


def step(q, k, v, do, log_decay, scale=None, initial=None, dfinal=None, lengths=None):
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)] + ([initial.detach().requires_grad_(True)] if initial is not None else [])
    out = linear_attention(*leaves[:3], log_decay, scale, leaves[3] if initial is not None else None, lengths,
                           output_final_state=dfinal is not None)
    o, final = out if dfinal is not None else (out, None)
    grads = torch.autograd.grad([o] + ([final] if dfinal is not None else []), leaves, [do] + ([dfinal] if dfinal is not None else []))
    return (o.detach(), final.detach() if final is not None else None, *grads[:3], grads[3] if initial is not None else None)


DIMS = [(128, 128), (64, 64), (256, 256), (64, 128), (128, 32), (1, 1), (3, 5), (8, 24), (33, 65), (100, 72), (130, 200), (256, 16), (17, 256)]
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dk,dv", DIMS)
def test_head_dimensions(gcg_lib, dk, dv, dtype):
    """With and without states, lengths that a chunk does not divide."""
    q, k, v, do, initial, dfinal = data(2, 150, 6, dk, dv, dtype, seed=dk * 300 + dv)
    ld, scale = decays(6), dk ** -0.5
    check(step(q, k, v, do, ld, None, initial, dfinal), reference(q, k, v, do, ld, scale, initial, dfinal), f"{dk}x{dv} {dtype}")
    check(step(q, k, v, do, ld, 0.3), reference(q, k, v, do, ld, 0.3, None, None), f"{dk}x{dv} {dtype} no states")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("L", [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 700])
def test_lengths_of_the_sequence(gcg_lib, L, dtype):
    q, k, v, do, initial, dfinal = data(1, L, 5, 64, 48, dtype, seed=L)
    ld = decays(5)
    check(step(q, k, v, do, ld, None, initial, dfinal), reference(q, k, v, do, ld, 0.125, initial, dfinal), f"L={L} {dtype}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("L", [1024, 1500, 2049])
def test_split_sequences(gcg_lib, L, dtype):
    """Few heads: the sequence is walked in segments that are joined (their workspace is not empty), states included."""
    for backward in (0, 1):        # (1024 rows are walked in one piece)
        assert (gcg_lib.gcg_linear_attn_workspace_bytes(1, L, 2, 64, 64, backward) > 0) == (L > 1024)
    q, k, v, do, initial, dfinal = data(1, L, 2, 64, 64, dtype, seed=L)
    ld = torch.tensor([-0.01, -0.0003], device=DEV)
    check(step(q, k, v, do, ld, None, initial, dfinal), reference(q, k, v, do, ld, 0.125, initial, dfinal), f"split {L} {dtype}")
    check(step(q, k, v, do, ld), reference(q, k, v, do, ld, 0.125, None, None), f"split {L} {dtype} no states")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("L,lengths", [(200, [200, 0, 1, 64, 65, 137]), (1600, [1600, 0, 3, 700])])
def test_ragged_batches(gcg_lib, L, lengths, dtype):
    """Entries of lengths 0 to L; what lies past an entry's end (NaN here) is not read, its outputs and gradients are zero."""
    bs = len(lengths)
    H = 5 if L < 1000 else 1
    q, k, v, do, initial, dfinal = data(bs, L, H, 64, 64, dtype, seed=bs)
    n = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    past = torch.arange(L, device=DEV)[None, :] >= n[:, None]
    for t in (q, k, v, do):
        t[past] = float("nan")
    ld = decays(5)[-H:].contiguous()
    got = step(q, k, v, do, ld, None, initial, dfinal, n)
    check(got, reference(q, k, v, do, ld, 0.125, initial, dfinal, n), f"ragged {dtype}")
    for i in (0, 2, 3, 4):
        assert not got[i][past].any()
    assert torch.equal(got[1][lengths.index(0)], initial[lengths.index(0)]) and torch.equal(got[5][lengths.index(0)], dfinal[lengths.index(0)])


def test_lengths_outside_the_sequence_are_clamped(gcg_lib):
    q, k, v, _, initial, _ = data(2, 70, 2, 32, 32, torch.bfloat16)
    ld = decays(2)
    n = torch.tensor([-5, 1000], dtype=torch.int32, device=DEV)
    o, final = linear_attention(q, k, v, ld, initial_state=initial, lengths=n, output_final_state=True)
    whole, last = linear_attention(q, k, v, ld, initial_state=initial, output_final_state=True)
    assert not o[0].any() and torch.equal(final[0], initial[0])
    assert torch.equal(o[1], whole[1]) and torch.equal(final[1], last[1])


@pytest.mark.parametrize("dtype", TYPES)
def test_long_memory(gcg_lib, dtype):
    """Thousands of chunks through factors next to 1: powers are kept to more than fp32's 24 bits."""
    q, k, v, do, initial, dfinal = data(1, 6000, 1, 16, 16, dtype, seed=3)
    ld = torch.tensor([-1e-5], device=DEV)
    check(step(q, k, v, do, ld, None, initial, dfinal), reference(q, k, v, do, ld, 0.25, initial, dfinal), f"long memory {dtype}")


@pytest.mark.parametrize("dtype", TYPES)
def test_continued_from_a_state(gcg_lib, dtype):
    """A prompt in two parts and single tokens after it are the whole prompt."""
    q, k, v, _, initial, _ = data(2, 140, 3, 40, 24, dtype, seed=4)
    ld, scale = decays(5)[2:].contiguous(), 40 ** -0.5
    want = reference(q, k, v, torch.zeros_like(v), ld, scale, initial, None)
    o1, s = linear_attention(q[:, :77], k[:, :77], v[:, :77], ld, initial_state=initial, output_final_state=True)
    o2, s = linear_attention(q[:, 77:130], k[:, 77:130], v[:, 77:130], ld, initial_state=s, output_final_state=True)
    rest = [linear_attention_step(q[:, t], k[:, t], v[:, t], ld, s) for t in range(130, 140)]
    check([torch.cat([o1, o2, torch.stack(rest, 1)], 1), s], want, f"continued {dtype}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bs,H,dk,dv", [(1, 1, 1, 1), (1, 4, 128, 128), (3, 5, 33, 65), (2, 7, 256, 256), (40, 30, 64, 40), (1, 3, 7, 4), (5, 1, 256, 2)])
def test_single_tokens(gcg_lib, bs, H, dk, dv, dtype):
    q, k, v, _, state, _ = data(bs, 3, H, dk, dv, dtype, seed=dk + dv)
    ld, scale = decays(H), dk ** -0.5
    want = reference(q, k, v, torch.zeros_like(v), ld, scale, state, None)
    s = state.clone()
    o = torch.stack([linear_attention_step(q[:, t], k[:, t], v[:, t], ld, s) for t in range(3)], 1)
    check([o, s], want, f"tokens {bs}x{H} {dk}x{dv} {dtype}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [32, 60, 128])
def test_projected_features(gcg_lib, d, dtype):
    """Read in place, the gradient in one tensor; with save_8bit the gradient is that at the checkpoint's values."""
    bs, L, H = 2, 130, 3
    q, k, v, do, _, _ = data(bs, L, H, d, d, dtype, seed=d)
    ld = decays(5)[2:].contiguous()
    features = torch.stack([q, k, v], 2).flatten(2).requires_grad_(True)
    for save_8bit in (False, True):
        o = linear_attention_features(features, H, ld, save_8bit=save_8bit)
        (df,) = torch.autograd.grad(o, features, do)
        kept = unpack8(pack8(features)) if save_8bit else features.detach()
        qb, kb, vb = kept.view(bs, L, 3, H, d).unbind(2)
        want = reference(qb, kb, vb, do, ld, d ** -0.5, None, None)
        check([None, None, *df.view(bs, L, 3, H, d).unbind(2)], want, f"features {d} {dtype} {save_8bit}")
        check([o.detach()], reference(q, k, v, do, ld, d ** -0.5, None, None), f"features {d} {dtype} {save_8bit}")


def test_gradients_against_differences(gcg_lib):
    """<gradient, direction> against (L(p + h d) - L(p - h d)) / 2h.  L is linear in each operand by itself, so the
    difference has no remainder; the fp32 forward's error, 2^-20 of L's terms, is divided by h."""
    q, k, v, do, initial, dfinal = data(1, 90, 2, 20, 12, torch.float32, seed=6)
    ld = torch.tensor([-0.1, -0.01], device=DEV)
    grads = step(q, k, v, do, ld, None, initial, dfinal)[2:]
    gen = torch.Generator(device=DEV).manual_seed(7)
    def loss(q, k, v, initial):
        o, final = linear_attention(q, k, v, ld, initial_state=initial, output_final_state=True)
        return (o.double() * do).sum() + (final.double() * dfinal).sum()
    mag = recurrence(q.abs(), k.abs(), v.abs(), do.abs(), ld, 20 ** -0.5, initial.abs(), None)
    terms = (mag[0] * do.abs()).sum() + (mag[1] * dfinal.abs()).sum()
    for i, grad in enumerate(grads):
        p = [q, k, v, initial]
        d = torch.randn(p[i].shape, generator=gen, device=DEV)
        h = 0.5
        ends = [loss(*[t + s * h * d if j == i else t for j, t in enumerate(p)]) for s in (1, -1)]
        assert abs((ends[0] - ends[1]) / (2 * h) - (grad.double() * d.double()).sum()) <= 4 * terms * 2.0 ** -20 / h


def test_strides_alignment_streams_and_repeatability(gcg_lib):
    """Views of one projection, (bs, H, L, d) storage, storage off the vectors, broadcast heads, an expanded gradient, another
    stream: the same bits as contiguous tensors give."""
    bs, L, H, d = 2, 100, 3, 64
    q, k, v, do, initial, dfinal = data(bs, L, H, d, d, torch.bfloat16, seed=8)
    ld = decays(5)[2:].contiguous()
    want = step(q, k, v, do, ld, None, initial, dfinal)
    same = lambda got: all(torch.equal(a, b) for a, b in zip(got, want))         # noqa: E731
    packed = torch.stack([q, k, v], 2)
    assert same(step(*packed.unbind(2), do, ld, None, initial, dfinal))
    swap = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)              # noqa: E731
    assert same(step(swap(q), swap(k), swap(v), swap(do), ld, None, initial, dfinal))
    odd = lambda t: torch.cat([t.flatten()[:1], t.flatten()])[1:].view(t.shape)  # noqa: E731
    assert same(step(odd(q), odd(k), odd(v), odd(do), ld, None, initial, dfinal))
    last = lambda t: t.transpose(-1, -2).contiguous().transpose(-1, -2)          # noqa: E731
    assert same(step(last(q), last(k), last(v), last(do), ld, None, initial, dfinal))
    shared = k[:, :, :1].expand(bs, L, H, d)
    kk = k[:, :, :1].detach().requires_grad_(True)
    o = linear_attention(q, kk.expand(bs, L, H, d), v, ld)
    (dk,) = torch.autograd.grad(o, kk, do)
    full = step(q, shared, v, do, ld)
    assert torch.equal(o, full[0]) and dk.shape == kk.shape
    ref = reference(q, shared, v, do, ld, d ** -0.5, None, None)[3]
    assert ((dk.double() - ref[0].sum(2, keepdim=True)).abs() <= ref[1].sum(2, keepdim=True) + H * U[torch.bfloat16] * ref[0].abs().sum(2, keepdim=True)).all()
    g = do[:, :1].expand(bs, L, H, d)
    assert all(torch.equal(a, b) for a, b in zip(step(q, k, v, g, ld)[2:5], step(q, k, v, g.contiguous(), ld)[2:5]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step(q, k, v, do, ld, None, initial, dfinal)
    side.synchronize()
    assert same(again)
    q2, k2, v2, do2, i2, f2 = data(1, 3000, 2, 64, 64, torch.float16, seed=9)
    ld2 = torch.tensor([-0.01, -0.001], device=DEV)
    assert all(torch.equal(a, b) for a, b in zip(step(q2, k2, v2, do2, ld2, None, i2, f2), step(q2, k2, v2, do2, ld2, None, i2, f2)))


def test_heads_and_entries_without_finite_values_stay_among_themselves(gcg_lib):
    """A NaN decay, an infinity in one head's k: other heads and entries are untouched, and rows of earlier chunks too."""
    q, k, v, do, _, _ = data(2, 200, 3, 64, 64, torch.bfloat16, seed=10)
    ld = torch.tensor([-0.1, -0.02, -0.003], device=DEV)
    clean = linear_attention(q, k, v, ld)
    k2 = k.clone()
    k2[0, 150, 1, 7] = float("inf")
    o = linear_attention(q, k2, v, ld)
    assert torch.equal(o[1], clean[1]) and torch.equal(o[0, :, [0, 2]], clean[0, :, [0, 2]])
    assert torch.equal(o[0, :150, 1], clean[0, :150, 1]) and not torch.isfinite(o[0, 192:, 1]).any()
    v2 = v.clone()
    v2[0, 150, 1, 7] = float("nan")
    o = linear_attention(q, k, v2, ld)
    assert torch.equal(o[0, :119, 1], clean[0, :119, 1]) and torch.isnan(o[0, 150:, 1, 7]).all()
    bad = ld.clone()
    bad[1] = float("nan")
    o = linear_attention(q, k, v, bad)
    assert torch.equal(o[:, :, [0, 2]], clean[:, :, [0, 2]]) and torch.isnan(o[:, 1:, 1]).all()


def test_empty(gcg_lib):
    ld = decays(2)
    for bs, L in ((0, 5), (2, 0)):
        q, k, v, do, initial, dfinal = data(bs, L, 2, 16, 8, torch.bfloat16)
        got = step(q, k, v, do, ld, None, initial, dfinal)
        assert got[0].shape == (bs, L, 2, 8) and torch.equal(got[1], initial) and torch.equal(got[5], dfinal)
    assert linear_attention_step(q[:, :0].reshape(0, 2, 16), q[:, :0].reshape(0, 2, 16), v[:, :0].reshape(0, 2, 8), ld,
                                 torch.zeros(0, 2, 16, 8, device=DEV)).shape == (0, 2, 8)


@pytest.mark.parametrize("L", [1100, 3000])
def test_captured_in_a_graph(gcg_lib, L):
    """A prompt, in one piece and split, and a token after it, replayed with new inputs."""
    q, k, v, do, initial, dfinal = data(1, L, 2, 64, 64, torch.bfloat16, seed=11)
    ld = torch.tensor([-0.01, -0.001], device=DEV)
    state = torch.zeros_like(initial)
    def call():
        o, final = _lib.linear_attn_fwd(q, k, v, ld, initial, None, 0.125, True)
        grads = _lib.linear_attn_bwd(do, q, k, v, ld, initial, None, dfinal, 0.125, True)
        state.copy_(final)
        return o, linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, state), *grads
    call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        out = call()
    torch.cuda.current_stream().wait_stream(side)
    for seed in range(3):
        for t, new in zip((q, k, v, do, initial, dfinal), data(1, L, 2, 64, 64, torch.bfloat16, seed=20 + seed)):
            t.copy_(new)
        eager = [t.clone() for t in call()] + [state.clone()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((*out, state), eager))


def test_offsets_beyond_32_bits(gcg_lib):
    """A row's offset past 2^31 elements: a strided view over a long storage (two heads of a wide row)."""
    L, width = 70000, 32768
    base = torch.zeros(L * width, dtype=torch.bfloat16, device=DEV).view(1, L, width)
    base[:, :, :192] = torch.randn(1, L, 192, device=DEV).to(torch.bfloat16)
    q, k, v = (base[:, :, 64 * i:64 * i + 64].unflatten(2, (2, 32)) for i in range(3))
    ld = torch.tensor([-0.1, -0.01], device=DEV)
    assert torch.equal(linear_attention(q, k, v, ld), linear_attention(*(t.contiguous() for t in (q, k, v)), ld))


def test_module_compiled_and_dispatched(gcg_lib):
    torch.manual_seed(0)
    for save_8bit in (False, True):
        m = LinearAttention(192, 3, save_8bit=save_8bit, device=DEV)
        x = torch.randn(2, 90, 576, device=DEV).to(torch.bfloat16).requires_grad_(True)
        dy = torch.randn(2, 90, 192, device=DEV).to(torch.bfloat16)
        y = m(x)
        (dx,) = torch.autograd.grad(y, x, dy)
        z = torch.compile(lambda t: m(t), fullgraph=True, backend="aot_eager")(x)
        assert torch.equal(z, y) and torch.equal(torch.autograd.grad(z, x, dy)[0], dx)
        with torch.no_grad():
            p, s = m.prefill(x)
            assert torch.equal(m(x), y)
            # (with a final state the weighted rows have a third part: the outputs may round differently)
            assert (p.double() - y.double()).abs().max() <= 2.0 ** -7 * y.abs().max()
            first, s2 = m.prefill(x[:, :89])
            last = m.step(x[:, 89], s2)
        assert torch.equal(first, y[:, :89]) or (first.double() - y[:, :89].double()).abs().max() <= 2.0 ** -6 * y.abs().max()
        assert (last.double() - y[:, 89].double()).abs().max() <= 2.0 ** -5 * y.abs().max()
        assert (s2 - s).abs().max() <= 2.0 ** -17 * 90 * x.abs().max() ** 2
    if _lib.TORCH_OPS:
        q, k, v, do, initial, dfinal = data(2, 80, 3, 32, 32, torch.bfloat16)
        ld = decays(5)[2:].contiguous()
        want = step(q, k, v, do, ld, 0.5, initial, dfinal)
        leaves = [t.requires_grad_(True) for t in (q, k, v, initial)]
        o, final = torch.ops.gcg.linear_attn_fwd(q, k, v, ld, initial, None, 0.5, True)
        got = (o, final, *torch.autograd.grad([o, final], leaves, [do, dfinal]))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        (dq,) = torch.autograd.grad(linear_attention(q, k, v, ld, 0.5, output_final_state=True)[1].sum(), q, allow_unused=True)
        assert not dq.any()


def test_refusals(gcg_lib):
    q, k, v, do, initial, _ = data(2, 20, 3, 16, 8, torch.bfloat16)
    ld = decays(3)
    with pytest.raises(RuntimeError, match="no CPU path"):
        linear_attention(q.cpu(), k.cpu(), v.cpu(), ld.cpu())
    for bad in ((q, k[:, :10], v), (q, k, v[:, :, :2]), (q[0], k[0], v[0])):
        with pytest.raises((RuntimeError, ValueError), match="must be"):
            linear_attention(*bad, ld)
    with pytest.raises((RuntimeError, ValueError), match="share dtype"):
        linear_attention(q, k, v.float(), ld)
    with pytest.raises((RuntimeError, ValueError), match="log_decay"):
        linear_attention(q, k, v, ld[:2].contiguous())
    with pytest.raises((RuntimeError, ValueError), match="log_decay"):
        linear_attention(q, k, v, ld.double())
    with pytest.raises((RuntimeError, ValueError), match="initial_state"):
        linear_attention(q, k, v, ld, initial_state=initial.to(torch.bfloat16))
    with pytest.raises((RuntimeError, ValueError), match="initial_state"):
        linear_attention(q, k, v, ld, initial_state=initial.transpose(2, 3))
    with pytest.raises((RuntimeError, ValueError), match="lengths"):
        linear_attention(q, k, v, ld, lengths=torch.tensor([3, 4], device=DEV))
    wide = torch.zeros(1, 2, 1, 257, device=DEV)
    with pytest.raises((RuntimeError, ValueError), match="256"):
        linear_attention(wide, wide, wide, ld[:1].contiguous())
    with pytest.raises((RuntimeError, TypeError), match="unsupported dtype"):
        linear_attention(q.double(), k.double(), v.double(), ld)
    with pytest.raises(RuntimeError, match="constant of the heads"):
        linear_attention(q, k, v, ld.clone().requires_grad_(True))
    with pytest.raises(RuntimeError, match="not differentiable"):
        linear_attention_step(q[:, 0].clone().requires_grad_(True), k[:, 0], v[:, 0], ld, initial)
    with pytest.raises((RuntimeError, ValueError), match="state"):
        linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, initial.half())
    with pytest.raises((RuntimeError, ValueError), match="features"):
        linear_attention_features(torch.zeros(2, 4, 25, device=DEV), 3, ld)
    with pytest.raises(RuntimeError, match="bad argument"):
        linear_attention(q, k, v, ld, scale=float("nan"))
    assert gcg_lib.gcg_linear_attn_workspace_bytes(0, 5, 1, 16, 16, 0) == 0
    p = q.data_ptr()
    st = (__import__("ctypes").c_int64 * 21)(*([0] * 21))
    assert gcg_lib.gcg_linear_attn_fwd(p, p, p, None, p, None, None, p, None, None, 0, 1, 4, 1, 16, 16, 1.0, 1, None) == -1
    assert gcg_lib.gcg_linear_attn_fwd(p, p, p, st, p, None, None, p, None, None, 0, 1, 4, 1, 300, 16, 1.0, 1, None) == -2
    assert gcg_lib.gcg_linear_attn_fwd(p, p, p, st, p, None, None, p, None, None, 0, 1, 5000, 1, 16, 16, 1.0, 1, None) == -3
    assert gcg_lib.gcg_linear_attn_step(p, p, p, p, st, p, None, 1, 1, 16, 16, 1.0, 1, None) == -1
