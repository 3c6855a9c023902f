"""Workloads of the operators around the quantized linear of a DiT block.

  linear    a linear with MXFP4 weights (E2M1 codes, one E8M0 scale per 32 inputs)
            on activations quantised to MXFP4 in the call, with the fused epilogue
            y = residual + gate * act(x . W^T + bias)
  quantize  a tensor to MXFP4 and back to the values it then stands for
  rotary    RMSNorm of q and k per head, then rotary positions with several axes
  norm      x' = c x + gate * norm(branch), n = norm(x') * (1 + scale) + shift
  entry     norm whose n leaves as MXFP4 and feeds a linear: the entry of a block

Each has a plain form in elementary torch operations on 32-bit values (own = False),
the framework's call (own = True) and a definition in 64 bits (exact).
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6
THETA = 10000.0
BLOCK = 32

# The costliest listed sizes; drawn cases stay below them.
MAX_PRODUCT = 16384 * 3072 * 12288
MAX_ELEMENTS = 16896 * 3072


def listed():
    return [
        # The modulation of one block and stream: one timestep embedding, six vectors of the hidden size.
        dict(name="linear modulation, one token", kind="linear", m=1, k=3072, n=18432, x="bf16", act="none", bias=True,
             gate=False, residual=False),
        # A vision tower's fused q/k/v on a few patches: small, ragged, half precision.
        dict(name="linear 37 patches", kind="linear", m=37, k=1152, n=3456, x="f16", act="none", bias=True, gate=False,
             residual=False),
        # Feed-forward entry of a 2048 x 2048 image's tokens with its activation: the largest product.
        dict(name="linear feed-forward up", kind="linear", m=16384, k=3072, n=12288, x="bf16", act="gelu_tanh", bias=True,
             gate=False, residual=False),
        # Feed-forward exit at 1024 x 1024 (image and text tokens): deep, with the gated residual.
        dict(name="linear feed-forward down", kind="linear", m=4352, k=12288, n=3072, x="bf16", act="none", bias=True,
             gate=True, residual=True),
        # A block's activations quantised on their own, e.g. once for two consumers.
        dict(name="quantize activations", kind="quantize", rows=16896, k=3072, x="bf16"),
        # A dense 32-bit weight quantised at load; the width fills no whole block.
        dict(name="quantize odd weight", kind="quantize", rows=1153, k=4307, x="f32"),
        # Joint image and text tokens of a 2048 x 2048 image: q and k out of the fused q/k/v.
        dict(name="rotary image", kind="rotary", batch=1, t=1, h=128, w=128, text=512, hq=24, hk=24, dim=128, rot_t=8,
             rot_h=28, rot_w=28, pairs="adjacent", ladder="own", norm=True, x="bf16"),
        # One new token of a text model with shared key heads: latency.
        dict(name="rotary one token", kind="rotary", batch=1, t=0, h=0, w=0, text=1, hq=32, hk=8, dim=128, rot_t=24,
             rot_h=20, rot_w=20, pairs="halves", ladder="shared", norm=True, x="bf16"),
        # Two clips of nine frames, odd width, part of each head left unrotated, no norm.
        dict(name="rotary video", kind="rotary", batch=2, t=9, h=30, w=53, text=7, hq=12, hk=12, dim=72, rot_t=8, rot_h=12,
             rot_w=12, pairs="halves", ladder="own", norm=False, x="f16"),
        # After attention at 2048 x 2048: norm of the branch, gate, residual, the feed-forward's norm.
        dict(name="norm image", kind="norm", groups=1, rows=16896, hidden=3072, x="bf16", branch="bf16", post="rms",
             pre="layer", gate=True, modulate=True, c=1.0),
        # Three odd sequences with their own modulation, 32-bit residual stream, scaled residual.
        dict(name="norm f32 stream", kind="norm", groups=3, rows=1031, hidden=1160, x="f32", branch="bf16", post="rms",
             pre="rms", gate=True, modulate=True, c=0.75),
        # Between two blocks at 1024 x 1024: the residual update and norm, then q/k/v in MXFP4.
        dict(name="entry q/k/v", kind="entry", groups=1, rows=4352, hidden=3072, n=9216, x="bf16", branch="bf16", post="rms",
             pre="layer", gate=True, modulate=True, c=1.0),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "quantize", "rotary", "norm", "entry"])
    x = rng.choice(["bf16", "bf16", "f16", "f32"])
    while True:
        if kind == "linear":
            c = dict(kind=kind, m=_spread(rng, 1, 16384), k=_spread(rng, 64, 12288), n=_spread(rng, 64, 18432), x=x,
                     act=rng.choice(["none", "gelu_tanh", "silu"]), bias=rng.random() < 0.7, gate=rng.random() < 0.4,
                     residual=rng.random() < 0.4)
            if c["m"] * c["k"] * c["n"] <= MAX_PRODUCT and c["m"] * max(c["n"], c["k"]) <= 4 * MAX_ELEMENTS:
                return c
        elif kind == "quantize":
            c = dict(kind=kind, rows=_spread(rng, 1, 40000), k=_spread(rng, 32, 16384), x=x)
            if c["rows"] * c["k"] <= MAX_ELEMENTS:
                return c
        elif kind == "rotary":
            dim = rng.choice([32, 64, 72, 80, 96, 128, 128, 256])
            pairs = rng.randint(3, dim // 2)
            a = rng.randint(1, pairs - 2)
            b = rng.randint(1, pairs - a - 1)
            hk = rng.choice([1, 2, 4, 8, 12, 24])
            c = dict(kind=kind, batch=rng.randint(1, 3), t=rng.randint(0, 12), h=_spread(rng, 1, 128), w=_spread(rng, 1, 128),
                     text=_spread(rng, 1, 2048), hq=hk * rng.choice([1, 1, 2, 4]), hk=hk, dim=dim, rot_t=a, rot_h=b,
                     rot_w=pairs - a - b, pairs=rng.choice(["adjacent", "halves"]), ladder=rng.choice(["own", "shared"]),
                     norm=rng.random() < 0.7, x=x)
            if c["batch"] * _tokens(c) * (c["hq"] + c["hk"]) * dim <= 2 * MAX_ELEMENTS:
                return c
        else:
            c = dict(kind=kind, groups=rng.randint(1, 4), rows=_spread(rng, 1, 16896), hidden=_spread(rng, 64, 8192), x=x,
                     branch=rng.choice([x, "bf16"]), post=rng.choice(["rms", "layer", "none"]),
                     pre=rng.choice(["rms", "layer"]), gate=rng.random() < 0.7, modulate=rng.random() < 0.7,
                     c=rng.choice([1.0, 0.5, 1.5]))
            if kind == "entry":
                c["n"] = _spread(rng, 64, 9216)
            rows = c["groups"] * c["rows"]
            if rows * max(c["hidden"], c.get("n", 0)) <= MAX_ELEMENTS:
                return c


# ---------------------------------------------------------------- inputs


def _tokens(c):
    return c["t"] * c["h"] * c["w"] + c["text"]


def _randn(g, shape, std=1.0, dtype=torch.float32):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def _activations(g, rows, k, dtype):
    """Gaussian rows with a few channels an order larger, as the inputs of transformer linears have."""
    channel = torch.exp(torch.randn((k,), generator=g, device="cuda") * 0.5)
    return (torch.randn((rows, k), generator=g, device="cuda") * channel).to(dtype)


def _positions(c):
    """int32 [tokens, 3]: the grid's (frame, row, column), rows and columns counted from the middle, then text tokens
    that count on along every axis."""
    t, h, w, text = c["t"], c["h"], c["w"], c["text"]
    ar = lambda n: torch.arange(n, dtype=torch.int32, device="cuda")  # noqa: E731
    grid = torch.stack([ar(t)[:, None, None].expand(t, h, w), (ar(h) - h // 2)[None, :, None].expand(t, h, w),
                        (ar(w) - w // 2)[None, None, :].expand(t, h, w)], -1).reshape(-1, 3)
    first = max(h, w) // 2 if t else 1500  # a lone text token is one far into its answer
    return torch.cat([grid, (first + ar(text))[:, None].expand(text, 3)]).contiguous()


def _norm_inputs(c, g):
    rows, hidden = c["groups"] * c["rows"], c["hidden"]
    vec = lambda std, mean=0.0: _randn(g, (c["groups"], hidden), std) + mean  # noqa: E731
    bf = torch.bfloat16
    s = dict(case=c, x=_randn(g, (rows, hidden), 2.0, DTYPES[c["x"]]),
             branch=_activations(g, rows, hidden, DTYPES[c["branch"]]),
             post_weight=(_randn(g, (hidden,), 0.1) + 1.0).to(bf) if c["post"] != "none" else None,
             pre_weight=(_randn(g, (hidden,), 0.1) + 1.0).to(bf) if c["pre"] == "rms" else None,
             gate=vec(0.5).to(bf) if c["gate"] else None, shift=vec(0.3).to(bf) if c["modulate"] else None,
             scale=vec(0.2).to(bf) if c["modulate"] else None)
    return s


def _weight(g, n, k):
    """A Gaussian weight in MXFP4, in the order that checkpoints store: codes uint8 [n, ceil(k / 32) * 16] (even columns in
    the low four bits), scales uint8 [n, ceil(k / 32)]."""
    codes, scales = _mx_codes(_randn(g, (n, k), 0.02))
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).contiguous(), scales.contiguous()


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    if c["kind"] == "quantize":
        s = dict(case=c, x=_activations(g, c["rows"], c["k"], DTYPES[c["x"]]))
    elif c["kind"] == "linear":
        m, k, n = c["m"], c["k"], c["n"]
        codes, scales = _weight(g, n, k)
        bf = torch.bfloat16
        s = dict(case=c, x=_activations(g, m, k, DTYPES[c["x"]]), codes=codes, scales=scales,
                 bias=_randn(g, (n,), 0.1, bf) if c["bias"] else None, gate=_randn(g, (n,), 0.5, bf) if c["gate"] else None,
                 residual=_randn(g, (m, n), 2.0, bf) if c["residual"] else None)
    elif c["kind"] == "rotary":
        b, tokens, hq, hk, d = c["batch"], _tokens(c), c["hq"], c["hk"], c["dim"]
        qkv = _randn(g, (b, tokens, hq + 2 * hk, d), 1.5, DTYPES[c["x"]])  # the fused projection's output
        rot = (c["rot_t"], c["rot_h"], c["rot_w"])
        s = dict(case=c, qkv=qkv, q=qkv[:, :, :hq], k=qkv[:, :, hq:hq + hk], positions=_positions(c),
                 q_weight=(_randn(g, (d,), 0.1) + 1.0).to(qkv.dtype) if c["norm"] else None,
                 k_weight=(_randn(g, (d,), 0.1) + 1.0).to(qkv.dtype) if c["norm"] else None,
                 axis=torch.tensor([a for a, n in enumerate(rot) for _ in range(n)], device="cuda"),
                 turns=_turns(c))
    else:
        s = _norm_inputs(c, g)
        if c["kind"] == "entry":
            s["codes"], s["scales"] = _weight(g, c["n"], c["hidden"])
            s["bias"] = _randn(g, (c["n"],), 0.1, torch.bfloat16)
    if own:  # the handles that a program keeps: the package, the layer, the axes
        import qwen_imager_b200 as lib
        s["lib"] = lib
        if "codes" in s:
            s["layer"] = lib.MxLinear(lib.MxTensor.from_packed(s["codes"], s["scales"], _inner(c)), s["bias"])
        if c["kind"] == "rotary":
            s["axes"] = lib.RotaryAxes((c["rot_t"], c["rot_h"], c["rot_w"]), theta=THETA, pairs=c["pairs"],
                                       ladder=c["ladder"], device="cuda")
    return s


def _inner(c):
    return c["k"] if c["kind"] == "linear" else c["hidden"]


def _frequencies(c):
    """Radians a position for each pair of a head, axis after axis."""
    rot = (c["rot_t"], c["rot_h"], c["rot_w"])
    if c["ladder"] == "shared":  # one ladder over all pairs
        return [THETA ** (-i / sum(rot)) for i in range(sum(rot))]
    return [THETA ** (-i / n) for n in rot for i in range(n)]


def _turns(c):
    """The frequencies in turns a position, as two 32-bit terms: 11 leading bits, whose product with a position below 2^13
    is exact, and the rest. Whole turns then drop out exactly, however far the position."""
    f = torch.tensor(_frequencies(c), dtype=torch.float64) / (2.0 * math.pi)
    m, e = torch.frexp(f)
    high = torch.ldexp(torch.round(m * 2048.0) / 2048.0, e)
    return high.float().cuda(), (f - high).float().cuda()


# ---------------------------------------------------------------- plain forms (32 bits)

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _mx_codes(x):
    """E2M1 codes uint8 [rows, 32 ceil(k / 32)] and E8M0 scales uint8 [rows, ceil(k / 32)]: the scale is the power of two
    that brings the block's largest magnitude to [4, 8), codes are the nearest (ties to the even code), past 6 they are 6; a
    block with an infinity or NaN has scale 255 (NaN)."""
    x = x.float()
    rows, k = x.shape
    blocks = -(-k // BLOCK)
    xb = torch.zeros((rows, blocks * BLOCK), device=x.device)
    xb[:, :k] = x
    xb = xb.view(rows, blocks, BLOCK)
    amax = xb.abs().amax(-1)
    e = torch.frexp(amax).exponent - 3 + 127  # amax = f * 2^exponent, f of [0.5, 1)
    e = torch.where(amax == 0, torch.zeros_like(e), e.clamp(0, 254))
    y = xb.abs() / _scale_values(e)[..., None]
    code = (y > 0.25).to(torch.uint8)
    code += y >= 0.75
    code += y > 1.25
    code += y >= 1.75
    code += y > 2.5
    code += y >= 3.5
    code += y > 5.0
    code |= torch.signbit(xb).to(torch.uint8) << 3
    bad = ~torch.isfinite(amax)
    code = torch.where(bad[..., None], torch.zeros_like(code), code)
    return code.view(rows, blocks * BLOCK), torch.where(bad, torch.full_like(e, 255), e).to(torch.uint8)


def _scale_values(e):
    """2^(e - 127) from its bits (e = 0 is the subnormal 2^-127); 255 is NaN."""
    e = e.to(torch.int32)
    bits = torch.where(e == 0, torch.full_like(e, 1 << 22), e << 23)
    return torch.where(e == 255, torch.full_like(e, 0x7FC00000), bits).view(torch.float32)


def _mx_values(codes, scales, k):
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=codes.device)
    rows, blocks = scales.shape
    v = table[codes.to(torch.int32)].view(rows, blocks, BLOCK) * _scale_values(scales)[..., None]
    return v.view(rows, blocks * BLOCK)[:, :k]


def _unpacked(packed):
    return torch.stack([packed & 15, packed >> 4], -1).reshape(packed.shape[0], -1)


def _product(values, s):
    c = s["case"]
    w = _mx_values(_unpacked(s["codes"]), s["scales"], _inner(c))
    t = values @ w.t()
    del w
    if s["bias"] is not None:
        t = t + s["bias"].float()
    if c.get("act") == "gelu_tanh":
        t = 0.5 * t * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (t + 0.044715 * t * t * t)))
    elif c.get("act") == "silu":
        t = t / (1.0 + torch.exp(-t))
    if s.get("gate") is not None and c["kind"] == "linear":
        t = t * s["gate"].float()
    if s.get("residual") is not None:
        t = t + s["residual"].float()
    return t.to(torch.bfloat16)


def _rotary_plain(x, weight, s):
    """x [batch, tokens, heads, dim] -> the same, rotated."""
    c = s["case"]
    t = x.float()
    if weight is not None:
        t = t * torch.rsqrt((t * t).mean(-1, keepdim=True) + EPS) * weight.float()
    at, (high, low) = s["positions"].float()[:, s["axis"]], s["turns"]  # [tokens, pairs]
    turn = at * high
    angle = 2.0 * math.pi * (turn - torch.round(turn) + at * low)
    cos, sin = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    p = angle.shape[-1]
    rot, rest = t[..., :2 * p], t[..., 2 * p:]
    if c["pairs"] == "adjacent":
        a, b = rot[..., 0::2], rot[..., 1::2]
        rot = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = rot[..., :p], rot[..., p:]
        rot = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([rot, rest], -1).to(x.dtype)


def _normed(t, how):
    if how == "layer":
        t = t - t.mean(-1, keepdim=True)
    return t * torch.rsqrt((t * t).mean(-1, keepdim=True) + EPS)


def _norm_plain(s):
    """(x', n), both in 32 bits."""
    c = s["case"]
    per_row = lambda v: v.float().repeat_interleave(c["rows"], 0)  # noqa: E731
    h = s["branch"].float()
    if c["post"] != "none":
        h = _normed(h, c["post"]) * s["post_weight"].float()
    if s["gate"] is not None:
        h = h * per_row(s["gate"])
    x = c["c"] * s["x"].float() + h
    n = _normed(x, c["pre"])
    if s["pre_weight"] is not None:
        n = n * s["pre_weight"].float()
    if s["scale"] is not None:
        n = n * (1.0 + per_row(s["scale"])) + per_row(s["shift"])
    return x, n


def _run_plain(s):
    c = s["case"]
    if c["kind"] == "linear":
        return _product(_mx_values(*_mx_codes(s["x"]), c["k"]), s)
    if c["kind"] == "quantize":
        return _mx_values(*_mx_codes(s["x"]), c["k"]).to(torch.bfloat16)
    if c["kind"] == "rotary":
        return _rotary_plain(s["q"], s["q_weight"], s), _rotary_plain(s["k"], s["k_weight"], s)
    x, n = _norm_plain(s)
    dtype = DTYPES[c["x"]]
    if c["kind"] == "norm":
        return x.to(dtype), n.to(dtype)
    return x.to(dtype), _product(_mx_values(*_mx_codes(n), c["hidden"]), s)


# ---------------------------------------------------------------- one pass


def run(state):
    if not own:
        return _run_plain(state)
    s, c, lib = state, state["case"], state["lib"]
    if c["kind"] == "linear":
        return s["layer"].forward_fused(s["x"], activation=c["act"], gate=s["gate"], residual=s["residual"])
    if c["kind"] == "quantize":
        return lib.mx_quantize(s["x"]).dequantize()
    if c["kind"] == "rotary":
        return lib.qk_norm_rotary(s["q"], s["k"], s["positions"], s["axes"], q_weight=s["q_weight"],
                                  k_weight=s["k_weight"], eps=EPS)
    x, n = lib.gated_residual_norm(s["x"], s["branch"], post=c["post"], post_weight=s["post_weight"], gate=s["gate"],
                                   residual_scale=c["c"], pre=c["pre"], pre_weight=s["pre_weight"], scale=s["scale"],
                                   shift=s["shift"], eps=EPS, quantize=c["kind"] == "entry")
    if c["kind"] == "norm":
        return x, n
    return x, s["layer"].forward_fused(n)


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
    c = case
    size = {"bf16": 2, "f16": 2, "f32": 4}
    if c["kind"] == "quantize":
        # the input in, 4-bit codes and a byte a block out, and back as 16-bit values
        return {"bytes": c["rows"] * c["k"] * (size[c["x"]] + 2) + c["rows"] * -(-c["k"] // BLOCK) * 17 * 2, "flops": 0}
    if c["kind"] == "rotary":
        e = c["batch"] * _tokens(c) * (c["hq"] + c["hk"]) * c["dim"]
        return {"bytes": 2 * e * size[c["x"]] + _tokens(c) * 12, "flops": (10 if c["norm"] else 6) * e}
    weight = lambda n, k: n * -(-k // BLOCK) * 17 + 2 * n  # noqa: E731
    if c["kind"] == "linear":
        m, k, n = c["m"], c["k"], c["n"]
        return {"bytes": m * k * size[c["x"]] + weight(n, k) + m * n * 2 * (2 if c["residual"] else 1), "flops": 2 * m * k * n}
    rows, h = c["groups"] * c["rows"], c["hidden"]
    b = rows * h * (2 * size[c["x"]] + size[c["branch"]])
    if c["kind"] == "norm":
        return {"bytes": b + rows * h * size[c["x"]], "flops": 20 * rows * h}
    return {"bytes": b + weight(c["n"], h) + 2 * rows * c["n"], "flops": 2 * rows * h * c["n"]}


# ---------------------------------------------------------------- the definitions in 64 bits


def _grid(v):
    """MXFP4 of each 32 values of a row, by rounding on the grid's local step."""
    rows, k = v.shape
    pad = -k % BLOCK
    b = torch.nn.functional.pad(v, (0, pad)).reshape(rows, -1, BLOCK)
    top = b.abs().amax(-1, keepdim=True)
    exponent = torch.where(top > 0, torch.frexp(top).exponent - 3, torch.full_like(top, -127, dtype=torch.int32)).clamp(min=-127)
    unit = torch.ldexp(torch.ones_like(top), exponent)
    y = b / unit
    step = torch.ldexp(torch.ones_like(y), (torch.frexp(y).exponent - 2).clamp(-1, 1))
    step = torch.where(y == 0, torch.ones_like(step), step)
    y = (torch.round(y / step) * step).clamp(-6.0, 6.0) * unit
    return y.reshape(rows, -1)[:, :k]


def _weight64(s, k):
    p = s["codes"].long()
    code = torch.empty((p.shape[0], 2 * p.shape[1]), dtype=torch.long, device=p.device)
    code[:, 0::2], code[:, 1::2] = p % 16, p // 16
    mag = code % 8
    v = torch.where(mag < 2, mag * 0.5, torch.exp2((mag // 2 - 1).double()) * (1.0 + 0.5 * (mag % 2)))
    v = torch.where(code >= 8, -v, v)
    return (v * torch.exp2(s["scales"].double() - 127.0).repeat_interleave(BLOCK, 1))[:, :k]


def _linear64(v, s):
    c = s["case"]
    t = _grid(v) @ _weight64(s, _inner(c)).t()
    if s["bias"] is not None:
        t += s["bias"].double()
    if c.get("act") == "gelu_tanh":
        t = t * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (t + 0.044715 * t ** 3))
    elif c.get("act") == "silu":
        t = t * torch.sigmoid(t)
    if c["kind"] == "linear":
        if s["gate"] is not None:
            t = t * s["gate"].double()
        if s["residual"] is not None:
            t = t + s["residual"].double()
    return t


def _rotary64(x, weight, s):
    c = s["case"]
    v = x.double()
    if weight is not None:
        v = v / (v.square().mean(-1, keepdim=True) + EPS).sqrt() * weight.double()
    rot = (c["rot_t"], c["rot_h"], c["rot_w"])
    p = sum(rot)
    theta = torch.tensor(_frequencies(c), dtype=torch.float64, device=x.device)
    angle = torch.cat([s["positions"][:, a:a + 1].double().expand(-1, n) for a, n in enumerate(rot)], 1) * theta
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    out = v.clone()
    first, second = (slice(0, 2 * p, 2), slice(1, 2 * p, 2)) if c["pairs"] == "adjacent" else (slice(0, p), slice(p, 2 * p))
    z = torch.complex(v[..., first], v[..., second]) * turn
    out[..., first], out[..., second] = z.real, z.imag
    return out


def _norm64(s):
    c = s["case"]

    def normed(v, how, weight):
        if how == "none":
            return v
        if how == "layer":
            var, mean = torch.var_mean(v, -1, correction=0, keepdim=True)
            v = (v - mean) / (var + EPS).sqrt()
        else:
            v = v / (v.square().mean(-1, keepdim=True) + EPS).sqrt()
        return v if weight is None else v * weight.double()

    groups = lambda v: v.reshape(c["groups"], c["rows"], c["hidden"])  # noqa: E731
    h = groups(normed(s["branch"].double(), c["post"], s["post_weight"]))
    if s["gate"] is not None:
        h = h * s["gate"].double()[:, None]
    x = groups(s["x"].double()) * c["c"] + h
    n = normed(x, c["pre"], s["pre_weight"])
    if s["scale"] is not None:
        n = n + n * s["scale"].double()[:, None] + s["shift"].double()[:, None]
    return x.reshape(-1, c["hidden"]), n.reshape(-1, c["hidden"])


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["kind"] == "linear":
        return _linear64(s["x"].double(), s)
    if c["kind"] == "quantize":
        return _grid(s["x"].double())
    if c["kind"] == "rotary":
        return _rotary64(s["q"], s["q_weight"], s), _rotary64(s["k"], s["k_weight"], s)
    x, n = _norm64(s)
    return (x, n) if c["kind"] == "norm" else (x, _linear64(n, s))
