"""The operators around a hyena layer's convolution, as cases that can be timed and compared: layer norm, activation
checkpoints in 8 bits, and linear attention with a decay for each head.

``run`` makes one pass: in plain torch operations, in 32 bits and rounded once at the end, or, where ``own`` is set,
through the package's entry points.  ``listed()`` holds the named cases, ``draw()`` makes more over the same ranges,
``exact()`` evaluates a case in 64 bits.

Fields: op ("norm", "pack", "attn", "token"), dtype, and by op

* norm: rows, width, step (forward and backward), bits8 (the backward reads the input from its 8-bit checkpoint)
* pack: rows, width; the tensor goes into 8 bits and comes back
* attn: bs, L, heads, dk, dv, step, state (an initial state is given, the final one returned), ragged (every batch entry has a
  length of its own), packed (one (bs, L, 3 * heads * dk) features tensor instead of q, k, v), bits8 (the backward
  reads the features from their 8-bit checkpoint)
* token: bs, heads, dk, dv; one token for every batch entry, the state updated in place
"""
import math

import torch

own = False

DEVICE = "cuda:0"
BYTES = {"float32": 4, "bfloat16": 2, "float16": 2}
EPS = 1e-5
BLOCK = 128                 # elements that share a scale of the 8-bit checkpoints
CHUNK = 256                 # rows of a chunk of the plain linear attention


def _norm(rows, width, dtype, step=True, bits8=False, **name):
    return dict(name, op="norm", rows=rows, width=width, dtype=dtype, step=step, bits8=bits8)


def _pack(rows, width, dtype, **name):
    return dict(name, op="pack", rows=rows, width=width, dtype=dtype)


def _attn(bs, L, heads, dk, dv, dtype, step=True, state=False, ragged=False, packed=False, bits8=False, **name):
    return dict(name, op="attn", bs=bs, L=L, heads=heads, dk=dk, dv=dv, dtype=dtype, step=step, state=state,
                ragged=ragged, packed=packed, bits8=bits8)


def _token(bs, heads, dk, dv, dtype, **name):
    return dict(name, op="token", bs=bs, heads=heads, dk=dk, dv=dv, dtype=dtype)


def listed():
    return [
        # norm in front of the smallest benchmark layer (2048 tokens, 256 channels): hardly more than a launch
        _norm(2048, 256, "float32", step=False, name="norm_forward_small"),
        # norm of a 7B layer, training step on 2 sequences of 8192 tokens
        _norm(16384, 4096, "bfloat16", name="norm_step_7b"),
        # norm of a layer of another width on a ragged batch, training step in half precision
        _norm(15009, 2560, "float16", name="norm_step_ragged"),
        # norm of a 40B layer, 32768 tokens: the backward reads the residual stream from 8 bits
        _norm(32768, 8192, "bfloat16", bits8=True, name="norm_step_40b_8bit"),
        # checkpoint of a short prompt's activations in an odd width: rows that end inside a block and off the sectors
        _pack(701, 1001, "float32", name="pack_odd_small"),
        # checkpoint of a 7B layer's projected features (2 x 8192 tokens, three times 4096 channels)
        _pack(16384, 12288, "bfloat16", name="pack_features_7b"),
        # four prompts of different lengths, none of which a tile divides, go into the state that the decoding starts from
        _attn(4, 701, 32, 128, 128, "bfloat16", step=False, state=True, ragged=True, name="attn_prefill_ragged"),
        # training step of the mixer at the 7B layer shape
        _attn(2, 8192, 32, 128, 128, "bfloat16", name="attn_step_7b"),
        # training step from the projected features of an odd batch, kept in 8 bits for the backward
        _attn(3, 5003, 20, 64, 64, "float16", packed=True, bits8=True, name="attn_step_8bit_ragged"),
        # long context on few heads (one tensor-parallel rank's share): the sequence has to be split to fill the card
        _attn(1, 131072, 8, 128, 128, "bfloat16", step=False, state=True, name="attn_forward_long"),
        # one token of one sequence: latency
        _token(1, 32, 128, 128, "bfloat16", name="token_one"),
        # one token of a full serving batch at the 40B width: the states' bandwidth
        _token(128, 64, 128, 128, "bfloat16", name="token_batch"),
    ]


def _loguniform(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return n + 1 if n == 3072 else n


def draw(rng):
    """One more case: rows, widths, lengths, heads and batches over their logarithm; at most 2^27 elements in a norm, a
    checkpoint or a long context (norm and checkpoint 2^26 in fp32), 2^25 in the other sequences, 2^27 in a token's states."""
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    op = rng.choice(["norm", "norm", "norm8", "pack", "attn_step", "attn_step", "attn_packed", "attn_forward", "attn_long", "token", "token"])
    if op in ("norm", "norm8", "pack"):
        width = _loguniform(rng, 64, 12288)
        width = rng.choice([width, max(64, width // 64 * 64), max(128, width // 128 * 128)])
        width = width + 128 if width == 3072 else width
        rows = min(_loguniform(rng, 16, 65536), (1 << (26 if dtype == "float32" else 27)) // width)
        if op == "pack":
            return _pack(rows, width, dtype)
        return _norm(rows, width, dtype, step=op == "norm8" or rng.random() < 0.7, bits8=op == "norm8")
    d = rng.choice([32, 64, 64, 128, 128, 128, 256, rng.randint(16, 160)])
    e = rng.choice([d, d, 64, 128, rng.randint(16, 160)])
    heads = _loguniform(rng, 1, 48)
    heads = heads + 1 if {heads * d, heads * e} & {1024, 3072} else heads
    if op == "token":
        bs = min(_loguniform(rng, 1, 256), max(1, (1 << 27) // (heads * d * e)))
        return _token(bs, heads, d, e, dtype)
    if op == "attn_long":
        heads = rng.randint(1, 8)
        L = min(_loguniform(rng, 16384, 131072), (1 << 27) // (heads * max(d, e)))
        return _attn(1, L, heads, d, e, dtype, step=False, state=rng.random() < 0.5)
    bs = _loguniform(rng, 1, 8)
    if op == "attn_forward":
        L = min(_loguniform(rng, 1, 8192), max(1, (1 << 25) // (bs * heads * max(d, e))))
        return _attn(bs, L, heads, d, e, dtype, step=False, state=rng.random() < 0.7, ragged=rng.random() < 0.5)
    L = min(_loguniform(rng, 16, 16384), max(1, (1 << 25) // (bs * heads * max(d, e))))
    if op == "attn_packed":
        return _attn(bs, L, heads, d, d, dtype, packed=True, bits8=rng.random() < 0.7)
    return _attn(bs, L, heads, d, e, dtype, state=rng.random() < 0.5, ragged=rng.random() < 0.3)


def _lengths(c):
    """Lengths of the batch entries: of a ragged batch evenly spaced down from L."""
    return [max(1, c["L"] * (c["bs"] - i) // c["bs"]) if c["ragged"] else c["L"] for i in range(c["bs"])]


def _normal(shape, dtype, gen):
    return torch.empty(shape, dtype=dtype, device=DEVICE).normal_(generator=gen)


def prepare(c, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = getattr(torch, c["dtype"])
    s = {"case": c}
    if c["op"] in ("norm", "pack"):
        # a residual stream: channels of different scale and offset
        R, D = c["rows"], c["width"]
        spread = torch.exp(0.5 * torch.randn(D, generator=gen, device=DEVICE)).to(dtype)
        shift = (0.3 * torch.randn(D, generator=gen, device=DEVICE)).to(dtype)
        s["x"] = _normal((R, D), dtype, gen).mul_(spread).add_(shift)
        if c["op"] == "pack":
            return s
        s["w"] = (1 + 0.2 * torch.randn(D, generator=gen, device=DEVICE)).to(dtype)
        s["b"] = (0.1 * torch.randn(D, generator=gen, device=DEVICE)).to(dtype)
        if c["step"]:
            s["dy"] = _normal((R, D), dtype, gen)
            for n in "xwb":
                s[n].requires_grad_(True)
        return s
    bs, H, dk, dv = c["bs"], c["heads"], c["dk"], c["dv"]
    # decay rates spaced over the heads' logarithm, from a memory of 8 tokens to one of 4096
    rate = torch.logspace(-3, -12, H, base=2.0, device=DEVICE)
    s["log_decay"] = -rate * (0.8 + 0.4 * torch.rand(H, generator=gen, device=DEVICE))
    if c["op"] == "token":
        s["q"], s["k"] = (_normal((bs, H, dk), dtype, gen) for _ in range(2))
        s["v"] = _normal((bs, H, dv), dtype, gen)
        s["state"] = _normal((bs, H, dk, dv), torch.float32, gen).mul_(4)
        return s
    L = c["L"]
    if c["packed"]:
        s["features"] = _normal((bs, L, 3 * H * dk), dtype, gen)
        leaves = [s["features"]]
    else:
        s["q"], s["k"] = (_normal((bs, L, H, dk), dtype, gen) for _ in range(2))
        s["v"] = _normal((bs, L, H, dv), dtype, gen)
        leaves = [s["q"], s["k"], s["v"]]
    s["initial_state"] = _normal((bs, H, dk, dv), torch.float32, gen).mul_(4) if c["state"] else None
    s["lengths"] = torch.tensor(_lengths(c), dtype=torch.int32, device=DEVICE) if c["ragged"] else None
    if c["step"]:
        s["do"] = _normal((bs, L, H, dv), dtype, gen)
        if c["state"]:
            s["dstate"] = _normal((bs, H, dk, dv), torch.float32, gen)
            leaves.append(s["initial_state"])
        for t in leaves:
            t.requires_grad_(True)
    s["leaves"] = leaves
    return s


def run(s):
    if own:
        return _run_own(s)
    with torch.no_grad():
        return {"norm": _plain_norm, "pack": _plain_pack, "attn": _plain_attn, "token": _plain_token}[s["case"]["op"]](s)


# ---- the package's entry points ---------------------------------------------------------------------------

def _run_own(s):
    from savanna_amd.operators.act8 import pack8, unpack8
    from savanna_amd.operators.linear_attention import linear_attention, linear_attention_features, linear_attention_step
    from savanna_amd.operators.norm import layer_norm

    c = s["case"]
    if c["op"] == "pack":
        return unpack8(pack8(s["x"]))
    if c["op"] == "token":
        o = linear_attention_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"])
        return o, s["state"]
    if c["op"] == "norm":
        if not c["step"]:
            with torch.no_grad():
                return layer_norm(s["x"], s["w"], s["b"], EPS)
        y = layer_norm(s["x"], s["w"], s["b"], EPS, save_8bit=c["bits8"])
        return [y.detach(), *torch.autograd.grad(y, [s["x"], s["w"], s["b"]], s["dy"])]
    if c["packed"]:
        o = linear_attention_features(s["features"], c["heads"], s["log_decay"], save_8bit=c["bits8"])
        return [o.detach(), *torch.autograd.grad(o, s["leaves"], s["do"])]
    if not c["step"]:
        with torch.no_grad():
            return linear_attention(s["q"], s["k"], s["v"], s["log_decay"], initial_state=s["initial_state"],
                                    lengths=s["lengths"], output_final_state=c["state"])
    o = linear_attention(s["q"], s["k"], s["v"], s["log_decay"], initial_state=s["initial_state"], lengths=s["lengths"],
                         output_final_state=c["state"])
    if c["state"]:
        o, final = o
        return [o.detach(), final.detach(), *torch.autograd.grad([o, final], s["leaves"], [s["do"], s["dstate"]])]
    return [o.detach(), *torch.autograd.grad(o, s["leaves"], s["do"])]


# ---- plain forms ------------------------------------------------------------------------------------------

def _codes(x):
    """(codes, scales) of the 8-bit checkpoint of (..., D) in fp32: blocks of 128 along the last dimension share a
    scale; a block whose largest magnitude is below 2^-100 is kept as zeros, one that holds no finite numbers as NaN."""
    D = x.shape[-1]
    v = torch.nn.functional.pad(x.float(), (0, -D % BLOCK)).unflatten(-1, (-1, BLOCK))
    top = v.abs().amax(-1, keepdim=True)
    tiny = top < 2.0 ** -100
    scale = torch.where(tiny, 0.0, top * (1.0 / 127.0))
    inv = torch.where(tiny, 0.0, torch.full_like(top, 127.0) / top)
    codes = torch.round(v * inv)
    bad = ~torch.isfinite(top)
    return torch.where(bad, 0.0, codes).flatten(-2)[..., :D], torch.where(bad, float("nan"), scale).squeeze(-1)


def _values(codes, scales):
    D = codes.shape[-1]
    return codes * scales.repeat_interleave(BLOCK, -1)[..., :D]


def _plain_pack(s):
    return _values(*_codes(s["x"])).to(s["x"].dtype)


def _plain_norm(s):
    c, dtype = s["case"], s["x"].dtype
    x, w, b = s["x"].float(), s["w"].float(), s["b"].float()
    mean = x.mean(-1, keepdim=True)
    rstd = torch.rsqrt((x - mean).square().mean(-1, keepdim=True) + EPS)
    y = ((x - mean) * rstd * w + b).to(dtype)
    if not c["step"]:
        return y
    if c["bits8"]:
        x = _values(*_codes(x))
    dy, xh = s["dy"].float(), (x - mean) * rstd
    g = dy * w
    dx = rstd * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    return [y, dx.to(dtype), (dy * xh).sum(0).to(dtype), dy.sum(0).to(dtype)]


def _plain_token(s):
    q, k, v, state = s["q"].float(), s["k"].float(), s["v"].float(), s["state"]
    state.mul_(torch.exp(s["log_decay"])[:, None, None]).add_(k[..., :, None] * v[..., None, :])
    o = (q[..., :, None] * state).sum(-2) * q.shape[-1] ** -0.5
    return o.to(s["q"].dtype), state


def _decayed(a, b, c, log_decay, initial=None):
    """out_t = sum_{s <= t} f^(t-s) (a_t . b_s) c_s + f^(t+1) a_t initial, on (bs, H, L, .) in fp32: products inside
    chunks, and the chunks' states joined by a product over the chunks."""
    L, log_f = a.shape[2], log_decay[:, None, None]
    C = min(CHUNK, L)
    a, b, c = (torch.nn.functional.pad(t, (0, 0, 0, -L % C)).unflatten(2, (-1, C)) for t in (a, b, c))
    n = a.shape[2]
    at = torch.arange(C, device=a.device)
    gap = at[:, None] - at[None, :]
    inside = torch.where(gap >= 0, torch.exp(log_f * gap.clamp(min=0)), 0.0)                       # (H, C, C)
    out = torch.matmul(torch.matmul(a, b.transpose(-1, -2)) * inside[None, :, None], c)
    to_end = torch.exp(log_f * (C - 1 - at)[None, :, None])                                       # (H, C, 1)
    states = torch.matmul((b * to_end[None, :, None]).transpose(-1, -2), c)                       # (bs, H, n, da, dc)
    chunk = torch.arange(n, device=a.device)
    hops = chunk[:, None] - chunk[None, :] - 1
    join = torch.where(hops >= 0, torch.exp(log_f * C * hops.clamp(min=0)), 0.0)                  # (H, n, n)
    before = torch.matmul(join[None], states.flatten(3)).unflatten(3, states.shape[3:])
    from_start = torch.exp(log_f * (1 + at)[None, :, None])                                       # (H, C, 1)
    out = out + torch.matmul(a, before) * from_start[None, :, None]
    out = out.flatten(2, 3)[:, :, :L]
    if initial is not None:
        t = torch.arange(L, device=a.device)
        out = out + torch.matmul(a.flatten(2, 3)[:, :, :L], initial) * torch.exp(log_f * (t + 1)[None, :, None])[None]
    return out


def _plain_attn(s):
    c = s["case"]
    bs, L, H = c["bs"], c["L"], c["heads"]
    scale = c["dk"] ** -0.5
    dtype = getattr(torch, c["dtype"])
    heads_first = lambda t: t.float().transpose(1, 2).contiguous()                                 # noqa: E731
    if c["packed"]:
        kept = s["features"]
        q, k, v = (heads_first(t) for t in kept.unflatten(-1, (3, H, -1)).unbind(2))
    else:
        q, k, v = heads_first(s["q"]), heads_first(s["k"]), heads_first(s["v"])
    init, log_decay = s["initial_state"], s["log_decay"]
    t = torch.arange(L, device=q.device)
    length = s["lengths"] if s["lengths"] is not None else torch.full((bs,), L, device=q.device)
    valid = (t[None] < length[:, None])[:, None, :, None]                                          # (bs, 1, L, 1)
    if c["ragged"]:
        k, v = torch.where(valid, k, 0.0), torch.where(valid, v, 0.0)
    o = scale * _decayed(q, k, v, log_decay, init)
    o = torch.where(valid, o, 0.0) if c["ragged"] else o
    out = [o.transpose(1, 2).to(dtype)]
    # exponent of a row's decay to the end of its sequence
    left = (length[:, None] - 1 - t[None]).clamp(min=0)[:, None, :, None]                          # (bs, 1, L, 1)
    to_end = torch.exp(log_decay[None, :, None, None] * left)
    whole = torch.exp(log_decay[None, :] * length[:, None])[..., None, None]                       # (bs, H, 1, 1)
    if c["state"]:
        out.append(torch.matmul((k * to_end).transpose(-1, -2), v) + whole * init)
    if not c["step"]:
        return out if c["state"] else out[0]
    do = heads_first(s["do"])
    if c["ragged"]:
        q, do = torch.where(valid, q, 0.0), torch.where(valid, do, 0.0)
    if c["bits8"]:
        back = _values(*_codes(kept)).to(dtype)
        q, k, v = (heads_first(u) for u in back.unflatten(-1, (3, H, -1)).unbind(2))
    flip = lambda u: u.flip(2)                                                                     # noqa: E731
    dq = scale * _decayed(do, v, k, log_decay, init.transpose(-1, -2).contiguous() if c["state"] else None)
    dk = scale * flip(_decayed(flip(v), flip(do), flip(q), log_decay))
    dv = scale * flip(_decayed(flip(k), flip(q), flip(do), log_decay))
    if c["state"]:
        G = s["dstate"]
        dk = dk + torch.matmul(v * to_end, G.transpose(-1, -2).contiguous())
        dv = dv + torch.matmul(k * to_end, G)
        from_start = torch.exp(log_decay[:, None, None] * (t + 1)[None, :, None])[None]
        dinit = whole * G + scale * torch.matmul((q * from_start).transpose(-1, -2), do)
    if c["ragged"]:
        dq, dk, dv = (torch.where(valid, u, 0.0) for u in (dq, dk, dv))
    if c["packed"]:
        return out + [torch.stack([u.transpose(1, 2) for u in (dq, dk, dv)], 2).flatten(2).to(dtype)]
    return out + [u.transpose(1, 2).to(dtype) for u in (dq, dk, dv)] + ([dinit] if c["state"] else [])


# ---- the definitions in 64 bits ---------------------------------------------------------------------------

def exact(c, seed):
    """The operators from their definitions in 64 bits; linear attention token by token, by the state's recurrence forward
    and its adjoint backward."""
    def kept(x):
        """What the 8-bit checkpoint of x stands for (the scales are fp32 numbers by the format's definition)."""
        out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
        for at in range(0, x.shape[-1], BLOCK):
            v = x[..., at:at + BLOCK].double()
            top = v.abs().amax(-1, keepdim=True)
            scale = (top.float() * (1.0 / 127.0)).double()
            out[..., at:at + BLOCK] = torch.where(top > 0, torch.round(v * 127 / top.clamp(min=1e-30)) * scale, 0.0)
        return out

    def norm(s):
        x, w, b = s["x"].double(), s["w"].double(), s["b"].double()
        mean = x.sum(-1, keepdim=True) / c["width"]
        std = ((x * x).sum(-1, keepdim=True) / c["width"] - mean * mean + EPS).sqrt()
        y = (x - mean) / std * w + b
        if not c["step"]:
            return y
        xh = ((kept(s["x"]) if c["bits8"] else x) - mean) / std
        dy = s["dy"].double()
        g = dy * w / std
        dx = g - (g.sum(-1, keepdim=True) + xh * (g * xh).sum(-1, keepdim=True)) / c["width"]
        return [y, dx, (dy * xh).sum(0), dy.sum(0)]

    def token(s):
        q, k, v = (s[n].double() for n in "qkv")
        S = torch.exp(s["log_decay"].double())[:, None, None] * s["state"].double() + k[..., None] * v[..., None, :]
        return (q[..., None] * S).sum(-2) * c["dk"] ** -0.5, S

    def attn(s):
        bs, L, H = c["bs"], c["L"], c["heads"]
        if c["packed"]:
            q, k, v = (t.double() for t in s["features"].unflatten(-1, (3, H, -1)).unbind(2))
        else:
            q, k, v = (s[n].double() for n in "qkv")
        q = q * c["dk"] ** -0.5
        f = torch.exp(s["log_decay"].double())[:, None, None]
        length = torch.tensor(_lengths(c), device=q.device)[:, None, None, None]
        zero = torch.zeros(bs, H, c["dk"], c["dv"], dtype=torch.float64, device=q.device)
        S = s["initial_state"].double() if c["state"] else zero
        o = torch.zeros(bs, L, H, c["dv"], dtype=torch.float64, device=q.device)
        for t in range(L):
            S_t = torch.addcmul(f * S, k[:, t, :, :, None], v[:, t, :, None, :])
            S = torch.where(t < length, S_t, S) if c["ragged"] else S_t
            o[:, t] = (q[:, t, :, :, None] * S).sum(-2)
        inside = torch.arange(L, device=q.device)[None, :, None, None] < length
        out = [torch.where(inside, o, 0.0)] + ([S] if c["state"] else [])
        if not c["step"]:
            return out if c["state"] else out[0]
        do = s["do"].double()
        if c["bits8"]:
            back = kept(s["features"]).to(s["features"].dtype)
            q, k, v = (t.double() for t in back.unflatten(-1, (3, H, -1)).unbind(2))
            q = q * c["dk"] ** -0.5
        dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
        S = s["initial_state"].double() if c["state"] else zero
        G = s["dstate"].double() if c["state"] else zero
        for t in range(L):
            S = torch.addcmul(f * S, k[:, t, :, :, None], v[:, t, :, None, :])
            dq[:, t] = (S * do[:, t, :, None, :]).sum(-1)
        for t in reversed(range(L)):
            G_t = torch.addcmul(G, q[:, t, :, :, None], do[:, t, :, None, :])
            dk[:, t] = (G_t * v[:, t, :, None, :]).sum(-1)
            dv[:, t] = (G_t * k[:, t, :, :, None]).sum(-2)
            G = torch.where(t < length, f * G_t, G) if c["ragged"] else f * G_t
        grads = [torch.where(inside, u, 0.0) for u in (dq * c["dk"] ** -0.5, dk, dv)]
        if c["packed"]:
            return out + [torch.stack(grads, 2).flatten(2)]
        return out + grads + ([G] if c["state"] else [])

    if c["op"] == "attn" and c["L"] * (3 if c["step"] else 1) > 150000:
        return None
    with torch.no_grad():
        s = {n: t.detach() if isinstance(t, torch.Tensor) else t for n, t in prepare(c, seed).items()}
        return {"norm": norm, "pack": lambda s: kept(s["x"]), "attn": attn, "token": token}[c["op"]](s)


def work(c):
    """Each input read once and each output written once; an 8-bit checkpoint is written by the forward and read by the
    backward in its input's place.  Flops of linear attention: two products of dk x dv a token and head forward (update,
    read-out), five backward (the two states' updates, dq, dk, dv)."""
    n = BYTES[c["dtype"]]
    kept = 1 + 4 / BLOCK
    if c["op"] == "norm":
        e, step = c["rows"] * c["width"], c["step"]
        moved = 2 * n + (2 * n + (2 * kept if c["bits8"] else n) if step else 0)
        return {"bytes": moved * e + (4 if step else 2) * c["width"] * n, "flops": (20 if step else 8) * e}
    if c["op"] == "pack":
        e = c["rows"] * c["width"]
        return {"bytes": 2 * (n + kept) * e, "flops": 6 * e}
    state = 4 * c["bs"] * c["heads"] * c["dk"] * c["dv"]
    if c["op"] == "token":
        return {"bytes": 2 * state + n * c["bs"] * c["heads"] * 2 * (c["dk"] + c["dv"]), "flops": state * 5 / 4}
    tokens, step = sum(_lengths(c)) * c["heads"], c["step"]
    moved = n * 2 * (c["dk"] + c["dv"])
    if step:
        moved += n * (2 * c["dk"] + 2 * c["dv"]) + (2 * kept if c["bits8"] else n) * (2 * c["dk"] + c["dv"])
    return {"bytes": moved * tokens + (4 if step else 2) * state * c["state"],
            "flops": (14 if step else 4) * tokens * c["dk"] * c["dv"]}
