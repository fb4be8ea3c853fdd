"""Operators of a layer in 8-bit floating point around a recurrent mixer, as cases that can be timed and compared:
root-mean-square norm with the residual's addition (its output in the tensors' type or in 8 bits), products of tensors in 8 bits
with a scale for each block of 128, and a gated linear recurrence.

``run`` makes one pass: in plain torch operations, in 32 bits and rounded once at the end of an operator, or, where ``own`` is
set, through the package's entry points.  ``listed()`` holds the named cases, ``draw()`` makes more over the same ranges,
``exact()`` evaluates a case in 64 bits.

Fields: op ("norm", "product", "layer", "scan", "token"), dtype, and by op

* norm: rows, width, residual (it is added first, and the sum returned), step (forward and backward), bits8 (the output in
  8 bits, returned as the values it stands for, which bfloat16 holds)
* product: rows, width, out, step; y = x w^T with both operands in 8 bits.  Forward: the weight is in 8 bits already
* layer: rows, width, out, step; the norm of a residual sum, in 8 bits into the product with a weight
* scan: bs, L, width, gate, step, state (an initial state is given, the final one returned), ragged (every batch entry has a
  length of its own), packed (one (bs, L, 3 * width) features tensor instead of x, f, gate)
* token: bs, width; one token for every batch entry, the state updated in place
"""
import math

import torch

own = False

DEVICE = "cuda:0"
BYTES = {"float32": 4, "bfloat16": 2, "float16": 2}
EPS = 1e-6
BLOCK = 128                 # elements along a row that share a scale
TOP = 448.0                 # largest number of 8 bits with 4 of exponent


def _norm(rows, width, dtype, residual=True, step=False, bits8=False, **name):
    return dict(name, op="norm", rows=rows, width=width, dtype=dtype, residual=residual, step=step, bits8=bits8)


def _product(op, rows, width, out, dtype, step=False, **name):
    return dict(name, op=op, rows=rows, width=width, out=out, dtype=dtype, step=step)


def _scan(bs, L, width, dtype, step=False, gate=True, state=False, ragged=False, packed=False, **name):
    return dict(name, op="scan", bs=bs, L=L, width=width, dtype=dtype, step=step, gate=gate, state=state, ragged=ragged, packed=packed)


def _token(bs, width, dtype, **name):
    return dict(name, op="token", bs=bs, width=width, dtype=dtype)


def listed():
    return [
        # norm of a decoding batch's 8 tokens at the 7B width: hardly more than a launch
        _norm(8, 4096, "bfloat16", name="norm_token"),
        # norm of a 7B layer, training step on 2 sequences of 8192 tokens with the residual stream's gradient
        _norm(16384, 4096, "bfloat16", step=True, name="norm_step_7b"),
        # norm of a 40B layer's prompt, into the 8 bits that the projection reads
        _norm(16384, 8192, "bfloat16", bits8=True, name="norm_8bit_40b"),
        # one token through the 7B layer's projection to three times its width: the weight's bandwidth
        _product("product", 1, 4096, 12288, "bfloat16", name="product_token"),
        # the same projection of 2 prompts of 8192 tokens
        _product("product", 16384, 4096, 12288, "bfloat16", name="product_7b"),
        # training step of the 7B layer's output projection: three products, each operand quantised along what it is summed over
        _product("product", 8192, 4096, 4096, "bfloat16", step=True, name="product_step_7b"),
        # norm and projection of a short prompt to an odd number of outputs, in half precision
        _product("layer", 701, 2560, 7683, "float16", name="layer_prompt_ragged"),
        # training step of norm and projection on an odd batch and an odd width
        _product("layer", 5003, 2561, 7680, "bfloat16", step=True, name="layer_step_ragged"),
        # training step of the recurrent mixer at the 7B layer shape, from the projected features
        _scan(2, 8192, 4096, "bfloat16", step=True, packed=True, name="scan_step_7b"),
        # four prompts of different lengths go into the state that the decoding starts from
        _scan(4, 701, 2560, "float16", state=True, ragged=True, name="scan_prefill_ragged"),
        # long context on few channels (one tensor-parallel rank's share) in fp32: the sequence has to be split to fill the card
        _scan(1, 131072, 512, "float32", state=True, name="scan_forward_long"),
        # one token of a serving batch at the 40B width
        _token(64, 8192, "bfloat16", name="token_batch"),
    ]


def _loguniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: rows, widths, lengths and batches over their logarithm; at most 2^26 elements in a norm (2^27 into 8 bits) and
    a scan, 2^39 multiplications in a product's forward and 2^37 in one of a step."""
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    half = rng.choice(["bfloat16", "bfloat16", "float16"])
    op = rng.choice(["norm", "norm_step", "norm_8bit", "product", "product_step", "layer", "layer_step", "scan", "scan_step",
                     "scan_packed", "scan_long", "token"])
    if op.startswith("norm"):
        width = _loguniform(rng, 64, 12288)
        width = rng.choice([width, max(64, width // 64 * 64), max(128, width // 128 * 128)])
        rows = min(_loguniform(rng, 1, 65536), (1 << 26) // width)
        return _norm(rows, width, dtype, residual=rng.random() < 0.7, step=op == "norm_step", bits8=op == "norm_8bit")
    if op.startswith(("product", "layer")):
        step = op.endswith("step")
        width, out = _loguniform(rng, 64, 8192), _loguniform(rng, 64, 12288)
        width = rng.choice([width, max(128, width // 128 * 128)])
        out = rng.choice([out, max(64, out // 64 * 64)])
        rows = min(_loguniform(rng, 1, 16384), max(1, (1 << (37 if step else 39)) // (width * out)))
        return _product(op.split("_")[0], rows, width, out, half, step=step)
    width = _loguniform(rng, 16, 8192)
    width = rng.choice([width, max(16, width // 16 * 16), max(64, width // 64 * 64)])
    if op == "token":
        return _token(_loguniform(rng, 1, 256), width, dtype)
    if op == "scan_long":
        L = _loguniform(rng, 16384, 131072)
        return _scan(1, L, min(width, (1 << 26) // L), dtype, gate=rng.random() < 0.5, state=rng.random() < 0.5)
    bs = _loguniform(rng, 1, 8)
    L = min(_loguniform(rng, 1, 16384), max(1, (1 << 26) // (bs * width)))
    if op == "scan_packed":
        return _scan(bs, L, width, dtype, step=rng.random() < 0.7, packed=True)
    return _scan(bs, L, width, dtype, step=op == "scan_step", gate=rng.random() < 0.7, state=rng.random() < 0.5, ragged=rng.random() < 0.4)


def _lengths(c):
    """Lengths of the batch entries: of a ragged batch evenly spaced down from L."""
    return [max(1, c["L"] * (c["bs"] - i) // c["bs"]) if c["ragged"] else c["L"] for i in range(c["bs"])]


def _normal(shape, dtype, gen):
    return torch.empty(shape, dtype=dtype, device=DEVICE).normal_(generator=gen)


def _stream(rows, width, dtype, gen):
    """A residual stream: channels of different scale."""
    spread = torch.exp(0.5 * torch.randn(width, generator=gen, device=DEVICE)).to(dtype)
    return _normal((rows, width), dtype, gen).mul_(spread)


def prepare(c, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = getattr(torch, c["dtype"])
    s = {"case": c}
    if c["op"] in ("norm", "product", "layer"):
        R, D = c["rows"], c["width"]
        s["x"] = _stream(R, D, dtype, gen)
        leaves = ["x"]
        if c["op"] != "product":
            s["g"] = (1 + 0.2 * torch.randn(D, generator=gen, device=DEVICE)).to(dtype)
            s["residual"] = _stream(R, D, dtype, gen) if c.get("residual", True) else None
            leaves += ["residual", "g"] if s["residual"] is not None else ["g"]
        N = D
        if c["op"] != "norm":
            N = c["out"]
            s["w"] = _normal((N, D), dtype, gen).mul_(D ** -0.5)
            leaves.append("w")
            if not c["step"]:
                # the weight as a serving program keeps it: codes in rows of whole blocks, the scales in whole words
                codes, scales = _codes(s.pop("w").float())
                s["codes"], s["scales"] = codes, torch.nn.functional.pad(scales, (0, -scales.shape[-1] % 4), value=1.0).to(torch.float8_e8m0fnu)
        if c["step"]:
            s["dy"] = _normal((R, N), dtype, gen)
            if s.get("residual") is not None:
                s["dr"] = _normal((R, D), dtype, gen)
            s["leaves"] = [s[n].requires_grad_(True) for n in leaves]
        return s
    bs, D = c["bs"], c["width"]
    # memories spaced over the channels' logarithm, from 8 tokens to 4096
    s["bias"] = torch.log(torch.logspace(3, 12, D, base=2.0, device=DEVICE)) + 0.2 * torch.randn(D, generator=gen, device=DEVICE)
    if c["op"] == "token":
        s["x"], s["f"], s["gate"] = (_normal((bs, D), dtype, gen) for _ in range(3))
        s["state"] = _normal((bs, D), torch.float32, gen)
        return s
    L = c["L"]
    if c["packed"]:
        s["features"] = _normal((bs, L, 3 * D), dtype, gen)
        leaves = [s["features"], s["bias"]]
    else:
        s["x"], s["f"] = (_normal((bs, L, D), dtype, gen) for _ in range(2))
        s["gate"] = _normal((bs, L, D), dtype, gen) if c["gate"] else None
        leaves = [t for t in (s["x"], s["f"], s["gate"], s["bias"]) if t is not None]
    s["initial_state"] = _normal((bs, D), torch.float32, gen) if c["state"] else None
    s["lengths"] = torch.tensor(_lengths(c), dtype=torch.int32, device=DEVICE) if c["ragged"] else None
    if c["step"]:
        s["dy"] = _normal((bs, L, D), dtype, gen)
        if c["state"]:
            s["dstate"] = _normal((bs, D), torch.float32, gen)
            leaves.append(s["initial_state"])
        s["leaves"] = [t.requires_grad_(True) for t in leaves]
    return s


def run(s):
    if own:
        return _run_own(s)
    with torch.no_grad():
        return {"norm": _plain_norm, "product": _plain_product, "layer": _plain_layer, "scan": _plain_scan, "token": _plain_token}[s["case"]["op"]](s)


# ---- the package's entry points ---------------------------------------------------------------------------

def _run_own(s):
    from savanna_amd.operators.float8 import Float8, from_float8, linear_float8, norm_linear_float8
    from savanna_amd.operators.gated_recurrence import gated_recurrence, gated_recurrence_features, gated_recurrence_step
    from savanna_amd.operators.norm import rms_norm, rms_norm_float8

    c = s["case"]
    if c["op"] == "token":
        return gated_recurrence_step(s["x"], s["f"], s["state"], s["gate"], s["bias"]), s["state"]
    if c["op"] == "norm":
        if c["bits8"]:
            y = rms_norm_float8(s["x"], s["g"], EPS, residual=s["residual"])
            if s["residual"] is None:
                return from_float8(y, torch.bfloat16)
            return from_float8(y[0], torch.bfloat16), y[1]
        if not c["step"]:
            with torch.no_grad():
                return rms_norm(s["x"], s["g"], EPS, residual=s["residual"])
        y = rms_norm(s["x"], s["g"], EPS, residual=s["residual"])
        if s["residual"] is None:
            return [y.detach(), *torch.autograd.grad(y, s["leaves"], s["dy"])]
        return [y[0].detach(), y[1].detach(), *torch.autograd.grad(y, s["leaves"], [s["dy"], s["dr"]])]
    if c["op"] in ("product", "layer"):
        if not c["step"]:
            w = Float8(s["codes"], s["scales"], c["width"])
            with torch.no_grad():
                return linear_float8(s["x"], w) if c["op"] == "product" else norm_linear_float8(s["x"], s["g"], w, EPS, residual=s["residual"])
        if c["op"] == "product":
            y = linear_float8(s["x"], s["w"])
            return [y.detach(), *torch.autograd.grad(y, s["leaves"], s["dy"])]
        y, r = norm_linear_float8(s["x"], s["g"], s["w"], EPS, residual=s["residual"])
        return [y.detach(), r.detach(), *torch.autograd.grad([y, r], s["leaves"], [s["dy"], s["dr"]])]

    def call():
        if c["packed"]:
            return gated_recurrence_features(s["features"], s["bias"])
        return gated_recurrence(s["x"], s["f"], s["gate"], s["bias"], initial_state=s["initial_state"], lengths=s["lengths"],
                                output_final_state=c["state"])

    if not c["step"]:
        with torch.no_grad():
            return call()
    y = call()
    if c["state"]:
        return [y[0].detach(), y[1].detach(), *torch.autograd.grad(y, s["leaves"], [s["dy"], s["dstate"]])]
    return [y.detach(), *torch.autograd.grad(y, s["leaves"], s["dy"])]


# ---- plain forms ------------------------------------------------------------------------------------------

def _power(e):
    """2^e in fp32 for whole numbers e from -126 to 127, exactly."""
    return ((e + 127).int() << 23).view(torch.float32)


def _codes(x):
    """(codes, scales) of (rows, D) in fp32.  Blocks of 128 along a row share the smallest power of two (2^-127 at least) that brings
    their largest magnitude to at most 448; rows are filled with zeros to whole blocks."""
    v = torch.nn.functional.pad(x, (0, -x.shape[-1] % BLOCK)).unflatten(-1, (-1, BLOCK))
    part, power = torch.frexp(v.abs().amax(-1))                      # top = part * 2^power, part in [1/2, 1)
    power = torch.where(part > 0, power - 9 + (part > TOP / 512), 0).clamp(min=-127)
    codes = (v * _power(-power)[..., None]).to(torch.float8_e4m3fn)
    return codes.flatten(-2), _power(power + 1) * 0.5


def _values(x):
    """What x in 8 bits stands for."""
    codes, scales = _codes(x)
    return (codes.float().unflatten(-1, (-1, BLOCK)) * scales[..., None]).flatten(-2)[..., :x.shape[-1]]


def _weight(s):
    return (s["codes"].float().unflatten(-1, (-1, BLOCK)) * s["scales"].float()[:, :s["codes"].shape[-1] // BLOCK, None]).flatten(-2)[:, :s["case"]["width"]]


def _plain_norm_fwd(s):
    r = s["x"].float()
    if s["residual"] is not None:
        r = (r + s["residual"].float()).to(s["x"].dtype).float()
    rstd = torch.rsqrt(r.square().mean(-1, keepdim=True) + EPS)
    return r, rstd, r * rstd * s["g"].float()


def _plain_norm_bwd(s, r, rstd, dy):
    dtype, xh = s["x"].dtype, r * rstd
    g = dy * s["g"].float()
    dx = rstd * (g - xh * (g * xh).mean(-1, keepdim=True))
    dw = (dy * xh).sum(0).to(dtype)
    if s["residual"] is None:
        return [dx.to(dtype), dw]
    dx = (dx + s["dr"].float()).to(dtype)
    return [dx, dx, dw]


def _plain_norm(s):
    c, dtype = s["case"], s["x"].dtype
    r, rstd, y = _plain_norm_fwd(s)
    y = _values(y).to(torch.bfloat16) if c["bits8"] else y.to(dtype)
    out = [y] if s["residual"] is None else [y, r.to(dtype)]
    if c["step"]:
        return out + _plain_norm_bwd(s, r, rstd, s["dy"].float())
    return out[0] if s["residual"] is None else tuple(out)


def _plain_product_bwd(s, kept):
    """dx and dw of y = x w^T; kept: what the forward's 8 bits of x stand for."""
    dy, w = s["dy"].float(), s["w"].float()
    dx = torch.matmul(_values(dy), _values(w.t().contiguous()).t())
    dw = torch.matmul(_values(dy.t().contiguous()), _values(kept.t().contiguous()).t())
    return dx.to(s["x"].dtype), dw.to(s["x"].dtype)


def _plain_product(s):
    x = _values(s["x"].float())
    y = torch.matmul(x, (_values(s["w"].float()) if s["case"]["step"] else _weight(s)).t()).to(s["x"].dtype)
    return [y, *_plain_product_bwd(s, x)] if s["case"]["step"] else y


def _plain_layer(s):
    dtype = s["x"].dtype
    r, rstd, x = _plain_norm_fwd(s)
    x = _values(x)
    y = torch.matmul(x, (_values(s["w"].float()) if s["case"]["step"] else _weight(s)).t()).to(dtype)
    if not s["case"]["step"]:
        return y, r.to(dtype)
    dn, dw = _plain_product_bwd(s, x)
    return [y, r.to(dtype), *_plain_norm_bwd(s, r, rstd, dn.float()), dw]


def _plain_token(s):
    z, state = s["f"].float() + s["bias"], s["state"]
    a, b = torch.sigmoid(z), torch.sigmoid(-z)
    state.mul_(a).add_(b * s["x"].float())
    return (s["gate"].float() * state).to(s["x"].dtype), state


def _scanned(a, u):
    """h_t = a_t h_{t-1} + u_t along dimension 1, in steps of doubled reach."""
    reach = 1
    while reach < u.shape[1]:
        u = torch.cat([u[:, :reach], u[:, reach:] + a[:, reach:] * u[:, :-reach]], 1)
        a = torch.cat([a[:, :reach], a[:, reach:] * a[:, :-reach]], 1)
        reach *= 2
    return u


def _plain_scan(s):
    c, dtype = s["case"], getattr(torch, s["case"]["dtype"])
    if c["packed"]:
        x, f, gate = (t.float() for t in s["features"].unflatten(-1, (3, -1)).unbind(-2))
    else:
        x, f, gate = (t.float() if t is not None else None for t in (s["x"], s["f"], s["gate"]))
    z = f + s["bias"]
    a, b = torch.sigmoid(z), torch.sigmoid(-z)
    if c["ragged"]:     # rows behind a length pass the state on
        inside = (torch.arange(c["L"], device=x.device)[None] < s["lengths"][:, None])[..., None]
        a, b, x = torch.where(inside, a, 1.0), torch.where(inside, b, 0.0), torch.where(inside, x, 0.0)
    u = b * x
    if c["state"]:
        u = torch.cat([u[:, :1] + a[:, :1] * s["initial_state"][:, None], u[:, 1:]], 1)
    h = _scanned(a, u)
    y = gate * h if c["gate"] else h
    if c["ragged"]:
        y = torch.where(inside, y, 0.0)
    out = [y.to(dtype)] + ([h[:, -1].clone()] if c["state"] else [])
    if not c["step"]:
        return tuple(out) if c["state"] else out[0]
    dy = s["dy"].float()
    if c["ragged"]:
        dy = torch.where(inside, dy, 0.0)
    dh = gate * dy if c["gate"] else dy
    if c["state"]:
        dh = torch.cat([dh[:, :-1], dh[:, -1:] + s["dstate"][:, None]], 1)
    later = torch.cat([torch.zeros_like(a[:, :1]), a[:, 1:].flip(1)], 1)
    G = _scanned(later, dh.flip(1)).flip(1)
    first = s["initial_state"][:, None] if c["state"] else torch.zeros_like(h[:, :1])
    df = G * (torch.cat([first, h[:, :-1]], 1) - x) * a * b
    grads = [b * G, df] + ([dy * h] if c["gate"] else [])
    if c["packed"]:
        grads = [torch.cat(grads, -1)]
    grads = [t.to(dtype) for t in grads] + [df.sum((0, 1))]
    return out + grads + ([a[:, 0] * G[:, 0]] if c["state"] else [])


# ---- the definitions in 64 bits ---------------------------------------------------------------------------

def exact(c, seed):
    """The operators from their definitions in 64 bits: 8-bit numbers block after block, the recurrence token by token and its
    adjoint backward."""
    def power_of(e):
        return ((e + 1023).long() << 52).view(torch.float64)

    def number8(v):
        """The nearest number of 1 sign, 4 exponent and 3 fraction bits (ties to the even one) of magnitudes up to 448."""
        _, e = torch.frexp(v)
        step = power_of((e - 4).clamp(min=-9))
        return torch.round(v / step) * step

    def kept(x):
        """What x in 8 bits with a power of two for each block along its rows stands for."""
        out = torch.empty_like(x)
        for at in range(0, x.shape[-1], BLOCK):
            v = x[..., at:at + BLOCK]
            top = v.abs().amax(-1, keepdim=True)
            power = torch.ceil(torch.log2(top.clamp(min=1e-300) / TOP))
            power = power.clamp(min=-900)
            power = power + (top > TOP * power_of(power)).double() - (top <= TOP * power_of(power - 1)).double()
            scale = power_of(power.clamp(min=-127))
            out[..., at:at + BLOCK] = number8(v / scale) * scale
        return out

    def norm_fwd(s):
        r = s["x"].double()
        if s["residual"] is not None:
            r = (r + s["residual"].double()).to(s["x"].dtype).double()
        rms = ((r * r).sum(-1, keepdim=True) / c["width"] + EPS).sqrt()
        return r, rms, r / rms * s["g"].double()

    def norm_bwd(s, r, rms, dy):
        xh = r / rms
        g = dy * s["g"].double() / rms
        dx = g - xh * (g * xh).sum(-1, keepdim=True) / c["width"]
        dw = (dy * xh).sum(0)
        if s["residual"] is None:
            return [dx, dw]
        return [dx + s["dr"].double()] * 2 + [dw]

    def norm(s):
        r, rms, y = norm_fwd(s)
        out = [kept(y) if c["bits8"] else y] + ([r] if s["residual"] is not None else [])
        if c["step"]:
            return out + norm_bwd(s, r, rms, s["dy"].double())
        return tuple(out) if s["residual"] is not None else out[0]

    def weight(s):
        if c["step"]:
            return kept(s["w"].double())
        scale = s["scales"].double().repeat_interleave(BLOCK, -1)
        return s["codes"].double()[:, :c["width"]] * scale[:, :c["width"]]

    def product_bwd(s, x8):
        dy, w = s["dy"].double(), s["w"].double()
        return kept(dy) @ kept(w.t().contiguous()).t(), kept(dy.t().contiguous()) @ kept(x8.t().contiguous()).t()

    def product(s):
        x = kept(s["x"].double())
        y = x @ weight(s).t()
        return [y, *product_bwd(s, x)] if c["step"] else y

    def layer(s):
        r, rms, x = norm_fwd(s)
        x = kept(x)
        y = x @ weight(s).t()
        if not c["step"]:
            return y, r
        dn, dw = product_bwd(s, x)
        return [y, r, *norm_bwd(s, r, rms, dn), dw]

    def token(s):
        z = s["f"].double() + s["bias"].double()
        h = torch.sigmoid(z) * s["state"].double() + torch.sigmoid(-z) * s["x"].double()
        return s["gate"].double() * h, h

    def scan(s):
        bs, L, D = c["bs"], c["L"], c["width"]
        if c["packed"]:
            x, f, gate = (s["features"][..., i * D:(i + 1) * D].double() for i in range(3))
        else:
            x, f = s["x"].double(), s["f"].double()
            gate = s["gate"].double() if c["gate"] else torch.ones_like(x)
        a = 1 / (1 + torch.exp(-f - s["bias"].double()))
        b = 1 / (1 + torch.exp(f + s["bias"].double()))
        length = torch.tensor(_lengths(c), device=x.device)[:, None]
        h = s["initial_state"].double() if c["state"] else torch.zeros(bs, D, dtype=torch.float64, device=x.device)
        y, before = torch.zeros_like(x), torch.zeros_like(x) if c["step"] else None
        for t in range(L):
            if c["step"]:
                before[:, t] = h
            new = a[:, t] * h + b[:, t] * x[:, t]
            h = torch.where(t < length, new, h) if c["ragged"] else new
            y[:, t] = gate[:, t] * h
        inside = (torch.arange(L, device=x.device)[None] < length)[..., None]
        out = [torch.where(inside, y, 0.0)] + ([h] if c["state"] else [])
        if not c["step"]:
            return tuple(out) if c["state"] else out[0]
        G = s["dstate"].double() if c["state"] else torch.zeros_like(h)
        dy, dx, df = s["dy"].double(), torch.zeros_like(x), torch.zeros_like(x)
        for t in reversed(range(L)):
            here = G + gate[:, t] * dy[:, t]
            dx[:, t] = b[:, t] * here
            df[:, t] = here * (before[:, t] - x[:, t]) * a[:, t] * b[:, t]
            G = torch.where(t < length, a[:, t] * here, G) if c["ragged"] else a[:, t] * here
        dgate = dy * (a * before + b * x)
        dx, df, dgate = (torch.where(inside, t, 0.0) for t in (dx, df, dgate))
        grads = [torch.cat([dx, df, dgate], -1)] if c["packed"] else [dx, df] + ([dgate] if c["gate"] else [])
        return out + grads + [df.sum((0, 1))] + ([G] if c["state"] else [])

    with torch.no_grad():
        s = {n: t.detach() if isinstance(t, torch.Tensor) else t for n, t in prepare(c, seed).items()}
        return {"norm": norm, "product": product, "layer": layer, "scan": scan, "token": token}[c["op"]](s)


def work(c):
    """Each input read once and each output written once; what the forward keeps of its input in 8 bits is read by the backward in
    its place.  Flops: a product's 2 a multiplication (three products in a step), some tens an element elsewhere."""
    n = BYTES[c["dtype"]]
    kept = 1 + 1 / BLOCK
    if c["op"] == "norm":
        e, step, added = c["rows"] * c["width"], c["step"], c["residual"]
        moved = n * (4 if added else 2)
        if c["bits8"]:
            moved += 2 * kept + 2 - n
        if step:
            moved += n * (4 if added else 3)
        return {"bytes": moved * e + c["width"] * n * (2 if step else 1), "flops": (20 if step else 6) * e}
    if c["op"] in ("product", "layer"):
        R, K, N = c["rows"], c["width"], c["out"]
        moved = n * R * (K + N) + (n if c["step"] else kept) * N * K
        if c["op"] == "layer":
            moved += n * (2 * R * K + K)
        if c["step"]:
            moved += n * R * (K + N) + kept * R * K + n * N * K
            moved += n * (2 * R * K + K) if c["op"] == "layer" else 0
        return {"bytes": moved, "flops": 2 * R * K * N * (3 if c["step"] else 1)}
    if c["op"] == "token":
        e = c["bs"] * c["width"]
        return {"bytes": e * (4 * n + 8) + 4 * c["width"], "flops": 20 * e}
    e, step = sum(_lengths(c)) * c["width"], c["step"]
    moved = n * (4 if c["gate"] else 3) + (n * (7 if c["gate"] else 5) if step else 0)
    return {"bytes": moved * e + 4 * c["bs"] * c["width"] * c["state"] * (4 if step else 2), "flops": (60 if step else 20) * e}
