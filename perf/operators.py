"""Measured cases of the cached-attention operators: rotary positions, the packed key/value cache
(written with rotation and quantisation, read back), attention over it, and attention of a batch
that shares a long prefix.

``run`` computes each in its plain form (elementary torch operations in 32 bits) or, where ``own``
is true, through the package's public calls. ``exact`` restates the definitions in 64 bits.

The cache's arithmetic, which both forms follow to the bit: a block of ``block`` values along the
head's axis has r = max|x| * (1 / QMAX) and the scale s = r rounded to bfloat16, or for E8M0 scales
the smallest power of two that is not below r; s is held within [2^-100, 2^100]. The code of x is
x * (1 / s) rounded to the nearest code, ties to even, and stands for code * s.
"""

from __future__ import annotations

import math

import torch

own = False

QMAX = {"int8": 127.0, "fp8e4m3": 448.0, "int4": 7.0, "fp4_e2m1": 6.0}
BITS = {"int8": 8, "fp8e4m3": 8, "int4": 4, "fp4_e2m1": 4}
DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
FP4 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
TINY, HUGE = 2.0 ** -100, 2.0 ** 100


# ---- cases -----------------------------------------------------------------------------------
def _rotary(name, **kw):
    base = dict(name=name, op="rotary", batch=1, tokens=1, heads=32, dim=128, rot=128, layout="half", dtype="bfloat16",
                positions=32768, base=10000.0, factor=1.0, order="bthd", grad=False)
    return {**base, **kw}


def _cache(name, **kw):
    base = dict(name=name, op="cache", tokens=1, heads=32, kv_heads=8, dim=128, rot=128, layout="half", dtype="bfloat16",
                positions=32768, base=10000.0, factor=1.0, format="int8", block=128, scales="bf16", page=64)
    return {**base, **kw}


def _attention(name, **kw):
    base = dict(name=name, op="attention", batch=1, queries=1, heads=32, kv_heads=8, dim=128, dtype="bfloat16",
                format="int8", block=128, scales="bf16", page=64, low=1, high=1, prefix=0, lse=False)
    return {**base, **kw}


def listed():
    return [
        # one token of a decode step of the 8B-shaped stack (32 query heads of 128)
        _rotary("rotary, one token", dtype="float16"),
        # a prompt of the 70B-shaped stack, neighbouring pairs in half of each head, positions stretched fourfold
        _rotary("rotary, a prompt", tokens=8192, heads=64, rot=64, layout="interleaved", factor=4.0),
        # a training step over sequences of odd length, heads before tokens, with the gradient
        _rotary("rotary, with its gradient", batch=3, tokens=1001, dtype="float32", order="bhtd", grad=True),
        # a decode step of 16 requests: one new token each, 4-bit cache
        _cache("cache, 16 new tokens", tokens=16, format="int4", dtype="float16"),
        # a prompt of odd length into a block-scaled 4-bit cache
        _cache("cache, 1999 tokens, FP4 blocks", tokens=1999, heads=64, format="fp4_e2m1", block=32, scales="e8m0", page=32),
        # a batch of prompts into an 8-bit cache
        _cache("cache, 32768 tokens, FP8", tokens=32768, format="fp8e4m3", factor=4.0),
        # a single request early in its answer: latency counts
        _attention("attention, one short request", low=257, high=257, dtype="float16"),
        # a full decode batch of the 70B-shaped stack with ragged lengths
        _attention("attention, 64 requests, FP4 blocks", batch=64, heads=64, format="fp4_e2m1", block=32, scales="e8m0",
                   low=2048, high=8192),
        # a chunk of a long prompt against what is cached of it and itself
        _attention("attention, a prompt's chunk", queries=1024, low=8192, high=8192, format="fp8e4m3"),
        # a few requests after a short system prompt
        _attention("prefix, 4 requests", batch=4, prefix=513, low=1, high=33, format="int4", dim=64, block=64, page=16, lse=True),
        # a serving batch behind a long document
        _attention("prefix, 32 requests", batch=32, prefix=8192, low=64, high=512),
        # many samples of one long prompt, 70B-shaped
        _attention("prefix, 128 requests", batch=128, heads=64, prefix=16384, low=1, high=1024, format="int4"),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    limit = [work(c) for c in listed()]
    most = {k: max(w[k] for w in limit) for k in ("bytes", "flops")}
    while True:
        op = rng.choice(("rotary", "cache", "attention", "prefix"))
        dim = rng.choice((64, 128, 128, 128, 256))
        rot = rng.choice((dim, dim, dim // 2))
        layout = rng.choice(("half", "interleaved"))
        factor = rng.choice((1.0, 1.0, 4.0))
        positions = _spread(rng, 2048, 131072)
        kv = rng.choice((1, 2, 4, 8, 8))
        heads = kv * rng.choice((1, 2, 4, 5, 8, 8))
        fmt = rng.choice(sorted(QMAX))
        block, scales = rng.choice(((dim, "bf16"), (dim, "e8m0"), (32, "e8m0"), (32, "bf16")))
        page = rng.choice((16, 32, 64, 128))
        half = rng.choice(("float16", "bfloat16"))
        if op == "rotary":
            c = _rotary("", batch=rng.choice((1, 1, 2, 5)), tokens=_spread(rng, 1, 16384), heads=heads, dim=dim, rot=rot,
                        layout=layout, dtype=rng.choice(sorted(DTYPES)), positions=max(16384, positions), factor=factor,
                        order=rng.choice(("bthd", "bhtd")), grad=rng.random() < 0.4)
        elif op == "cache":
            c = _cache("", tokens=_spread(rng, 1, 32768), heads=heads, kv_heads=kv, dim=dim, rot=rot, layout=layout,
                       dtype=half, positions=max(32768, positions), factor=factor, format=fmt, block=block, scales=scales,
                       page=page)
        else:
            high = _spread(rng, 1, 16384)
            queries = rng.choice((1, 1, 1, 2, 5, _spread(rng, 3, 2048))) if op == "attention" else 1
            c = _attention("", batch=_spread(rng, 1, 128), queries=queries, heads=heads, kv_heads=kv, dim=dim, dtype=half,
                           format=fmt, block=block, scales=scales, page=page, low=_spread(rng, 1, high), high=high,
                           prefix=_spread(rng, 64, 16384) if op == "prefix" else 0, lse=rng.random() < 0.3)
        del c["name"]
        w = work(c)
        # the plain form's products in 32 bits and its scores bound what a case may cost there
        plain = c["op"] != "attention" or (c["batch"] * c["kv_heads"] * c["high"] * c["dim"] < 6e8
                                           and c["batch"] * c["heads"] * c["queries"] * (c["high"] + c["prefix"]) < 3e8)
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"] and plain:
            return c


def work(case):
    c = case
    if c["op"] == "rotary":
        n, size = c["batch"] * c["tokens"] * c["heads"] * c["dim"], 4 if c["dtype"] == "float32" else 2
        passes = 2 if c["grad"] else 1
        tables = c["batch"] * c["tokens"] * (c["rot"] * 4 + 8)
        return {"bytes": passes * (2 * n * size + tables), "flops": passes * 3 * n * c["rot"] / c["dim"]}
    row = c["dim"] * BITS[c["format"]] / 8 + c["dim"] // c["block"] * (1 if c["scales"] == "e8m0" else 2)
    if c["op"] == "cache":
        kv, q = c["kv_heads"] * c["dim"], c["heads"] * c["dim"]
        per_token = 2 * 2 * q + 2 * 2 * kv + 2 * 2 * kv + 2 * 2 * c["kv_heads"] * row + 4 * c["rot"] + 16
        return {"bytes": c["tokens"] * per_token, "flops": c["tokens"] * (3 * (q + kv) + 12 * kv)}
    mean = (c["low"] + c["high"]) / 2
    keys = c["batch"] * mean + c["prefix"]
    own_pairs = sum(max(0.0, mean - j) for j in range(c["queries"])) * c["batch"]
    pairs = c["heads"] * (own_pairs + c["batch"] * c["queries"] * c["prefix"])
    rows = c["batch"] * c["queries"] * c["heads"]
    return {"bytes": keys * 2 * c["kv_heads"] * row + rows * c["dim"] * 4 + 4 * c["batch"], "flops": 4.0 * c["dim"] * pairs}


# ---- inputs ----------------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(1_000_003 * seed + 17)
    return g


def _angles(case, device):
    """The angle of each position and pair in 64 bits, and what multiplies cosine and sine. ``factor``
    stretches the positions: pairs that turn often within the original length keep their frequency,
    those that turn less than once are slowed by the factor, with a ramp between."""
    rot, base, factor = case["rot"], case["base"], case["factor"]
    i = torch.arange(rot // 2, dtype=torch.float64, device=device)
    freq = base ** (-2.0 * i / rot)
    gain = 1.0
    if factor != 1.0:
        original = case["positions"] / factor
        at = lambda beta: rot * math.log(original / (beta * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        low, high = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rot - 1)
        ramp = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
        freq = freq * (1 - ramp) + freq / factor * ramp
        gain = 0.1 * math.log(factor) + 1.0
    p = torch.arange(case["positions"], dtype=torch.float64, device=device)
    return p[:, None] * freq[None, :], gain


def _tables(case):
    a, gain = _angles(case, "cuda")
    return (a.cos() * gain).float(), (a.sin() * gain).float()


def _normal(shape, g, dtype):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _keys(shape, g, dtype):
    """Keys as projections give them: a few channels of each head several times larger."""
    x = torch.randn(shape, generator=g, device="cuda")
    gain = torch.ones(shape[-2:], device="cuda")
    gain[:, :: max(1, shape[-1] // 4)] = 5.0
    return (x * gain).to(dtype)


def _inputs(case, seed):
    """Every tensor of a case, from the seed alone."""
    c, g = case, _generator(seed)
    dtype = DTYPES[c["dtype"]]
    s = {"case": c}
    if c["op"] == "rotary":
        lead = (c["batch"], c["tokens"], c["heads"]) if c["order"] == "bthd" else (c["batch"], c["heads"], c["tokens"])
        view = (lambda t: t) if c["order"] == "bthd" else (lambda t: t.transpose(1, 2))
        s["x"] = view(_normal((*lead, c["dim"]), g, dtype))
        first = torch.randint(0, c["positions"] - c["tokens"] + 1, (c["batch"], 1), generator=g, device="cuda")
        s["positions"] = first + torch.arange(c["tokens"], device="cuda")
        if c["grad"]:
            s["dy"] = view(_normal((*lead, c["dim"]), g, dtype))
        return s
    if c["op"] == "cache":
        t, kv, d = c["tokens"], c["kv_heads"], c["dim"]
        # rows of one fused projection: queries, keys and values side by side
        qkv = _normal((t, (c["heads"] + 2 * kv) * d), g, dtype).view(t, c["heads"] + 2 * kv, d)
        s["q"], s["k"], s["v"] = qkv[:, : c["heads"]], qkv[:, c["heads"]: c["heads"] + kv], qkv[:, c["heads"] + kv:]
        s["pages"] = -(-t // c["page"]) + 8
        order = torch.randperm(s["pages"], generator=g, device="cuda")
        at = torch.arange(t, device="cuda")
        s["slots"] = order[at // c["page"]] * c["page"] + at % c["page"]
        s["positions"] = torch.randint(0, c["positions"], (t,), generator=g, device="cuda")
        return s
    b, kv, d, page = c["batch"], c["kv_heads"], c["dim"], c["page"]
    per, first = -(-c["high"] // page), -(-c["prefix"] // page)
    s["pages"] = b * per + first
    order = torch.randperm(s["pages"], generator=g, device="cuda").to(torch.int32)
    s["tables"], s["prefix"] = order[first:].view(b, per).contiguous(), order[:first].contiguous()
    s["lengths"] = torch.randint(c["low"], c["high"] + 1, (b,), generator=g, device="cuda").to(torch.int32)
    s["q"] = _normal((b, c["queries"], c["heads"], d), g, dtype)
    s["k"], s["k_scales"] = _quantise(_keys((s["pages"], page, kv, d), g, dtype).transpose(1, 2), c)
    s["v"], s["v_scales"] = _quantise(_normal((s["pages"], page, kv, d), g, dtype).transpose(1, 2), c)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    c = case
    if c["op"] != "attention":
        s["cos"], s["sin"] = _tables(c)
    if c["op"] == "cache" and not own:
        rows, blocks = (s["pages"], c["kv_heads"], c["page"]), c["dim"] // c["block"]
        s["kc"], s["vc"] = (torch.zeros((*rows, c["dim"] * BITS[c["format"]] // 8), dtype=torch.uint8, device="cuda") for _ in "kv")
        kind = torch.uint8 if c["scales"] == "e8m0" else torch.bfloat16
        s["ks"], s["vs"] = (torch.zeros((*rows, blocks), dtype=kind, device="cuda") for _ in "kv")
    if own:
        import tinygrad_dx12_b200 as tg

        s["tg"] = tg
        scale_dtype = torch.float8_e8m0fnu if c.get("scales") == "e8m0" else torch.bfloat16
        if c["op"] != "attention":
            s["table"] = tg.RotaryTable(s["cos"], s["sin"], c["layout"])
        if c["op"] == "cache":
            s["cache"] = tg.PackedCache.empty(s["pages"], c["page"], c["kv_heads"], c["dim"], c["format"],
                                              block_size=c["block"], scale_dtype=scale_dtype, device="cuda")
        if c["op"] == "attention":
            s["cache"] = tg.PackedCache(s["k"], s["v"], s["k_scales"].view(scale_dtype), s["v_scales"].view(scale_dtype),
                                        c["format"], c["dim"], c["block"])
        if c.get("grad"):
            s["x"].requires_grad_()
    return s


# ---- plain forms -----------------------------------------------------------------------------
def _rotate(x, cos, sin, layout, sign=1.0):
    """The first 2 * cos.shape[-1] values of each head turned by their pair's angle (the other way for sign -1)."""
    n = cos.shape[-1]
    x = x.float()
    cos, sin = cos.unsqueeze(-2), sin.unsqueeze(-2) * sign
    turn, rest = x[..., : 2 * n], x[..., 2 * n:]
    if layout == "half":
        a, b = turn[..., :n], turn[..., n:]
        return torch.cat((a * cos - b * sin, b * cos + a * sin, rest), -1)
    a, b = turn[..., 0::2], turn[..., 1::2]
    return torch.cat((torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2), rest), -1)


def _codes(y, fmt):
    """Nearest codes of y, ties to even: 8-bit ones as bytes, 4-bit ones in pairs, the first in the low bits."""
    q = QMAX[fmt]
    if fmt == "fp8e4m3":
        return y.clamp(-q, q).to(torch.float8_e4m3fn).view(torch.uint8)
    if fmt == "int8":
        return y.round().clamp(-q, q).to(torch.int8).view(torch.uint8)
    if fmt == "int4":
        n = y.round().clamp(-q, q).to(torch.int8) & 15
    else:
        m = y.abs()
        step = torch.where(m < 2, 0.5, torch.where(m < 4, 1.0, 2.0))
        m = ((m / step).round() * step).clamp(max=q)
        n = torch.where(m < 2, m * 2, torch.where(m < 4, m + 2, m / 2 + 4)).to(torch.int8) + (y.signbit().to(torch.int8) << 3)
    return (n[..., 0::2] | (n[..., 1::2] << 4)).view(torch.uint8)


def _quantise(x, c):
    """Codes and scales of x (..., dim)."""
    x = x.float().unflatten(-1, (-1, c["block"]))
    r = x.abs().amax(-1) * (1.0 / QMAX[c["format"]])
    if c["scales"] == "e8m0":
        e = ((r.view(torch.int32) + 0x7FFFFF) >> 23).clamp(27, 227)
        scales, s = e.to(torch.uint8), (e << 23).view(torch.float32)
    else:
        scales = r.to(torch.bfloat16).clamp(TINY, HUGE)
        s = scales.float()
    return _codes((x * s.reciprocal()[..., None]).flatten(-2), c["format"]), scales


def _dequantise(codes, scales, c):
    """The values (..., dim) in 32 bits that codes and scales stand for."""
    if c["format"] == "fp8e4m3":
        x = codes.view(torch.float8_e4m3fn).float()
    elif c["format"] == "int8":
        x = codes.view(torch.int8).float()
    else:
        n = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
        if c["format"] == "int4":
            x = ((n ^ 8).to(torch.int8) - 8).float()
        else:
            x = torch.tensor(FP4 + tuple(-v for v in FP4), device=codes.device)[n.int()]
    s = (scales.int() << 23).view(torch.float32) if scales.dtype == torch.uint8 else scales.float()
    return (x.unflatten(-1, (-1, c["block"])) * s[..., None]).flatten(-2)


def _plain_rotary(s):
    c = s["case"]
    cos, sin = s["cos"][s["positions"]], s["sin"][s["positions"]]
    y = _rotate(s["x"], cos, sin, c["layout"]).to(s["x"].dtype)
    return [y, _rotate(s["dy"], cos, sin, c["layout"], -1.0).to(s["x"].dtype)] if c["grad"] else [y]


def _plain_cache(s):
    c = s["case"]
    cos, sin = s["cos"][s["positions"]], s["sin"][s["positions"]]
    dtype, page, offset = s["k"].dtype, s["slots"] // c["page"], s["slots"] % c["page"]
    q = _rotate(s["q"], cos, sin, c["layout"]).to(dtype)
    kc, ks = _quantise(_rotate(s["k"], cos, sin, c["layout"]), c)
    vc, vs = _quantise(s["v"], c)
    s["kc"][page, :, offset], s["ks"][page, :, offset], s["vc"][page, :, offset], s["vs"][page, :, offset] = kc, ks, vc, vs
    k = _dequantise(s["kc"][page, :, offset], s["ks"][page, :, offset], c).to(dtype)
    v = _dequantise(s["vc"][page, :, offset], s["vs"][page, :, offset], c).to(dtype)
    return [q, k, v]


def _plain_attention(s):
    c = s["case"]
    b, n, kv, d = c["batch"], c["queries"], c["kv_heads"], c["dim"]
    group = c["heads"] // kv
    at = s["tables"].long()

    def own_rows(codes, scales):  # (batch, kv_heads, keys, dim)
        return _dequantise(codes[at].transpose(1, 2).flatten(2, 3), scales[at].transpose(1, 2).flatten(2, 3), c)

    def prefix_rows(codes, scales):  # (kv_heads, keys, dim)
        p = s["prefix"].long()
        return _dequantise(codes[p].transpose(0, 1).flatten(1, 2), scales[p].transpose(0, 1).flatten(1, 2), c)[:, : c["prefix"]]

    q = s["q"].float().unflatten(2, (kv, group)).permute(0, 2, 3, 1, 4) * (1.0 / math.sqrt(d))  # (batch, kv, group, queries, dim)
    k, v = own_rows(s["k"], s["k_scales"]), own_rows(s["v"], s["v_scales"])
    scores = (q.flatten(2, 3) @ k.transpose(-1, -2)).unflatten(2, (group, n))
    last = s["lengths"][:, None] - n + torch.arange(n, device="cuda")  # the last key that each query sees
    seen = torch.arange(k.shape[2], device="cuda") <= last[..., None]
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    if c["prefix"]:
        kp, vp = prefix_rows(s["k"], s["k_scales"]), prefix_rows(s["v"], s["v_scales"])
        rows = q.transpose(0, 1).flatten(1, 3)
        front = (rows @ kp.transpose(-1, -2)).unflatten(1, (b, group, n)).transpose(0, 1)
        scores = torch.cat((front, scores), -1)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = (scores - top).exp()
    total = p.sum(-1, keepdim=True)
    out = (p[..., c["prefix"]:].flatten(2, 3) @ v).unflatten(2, (group, n))
    if c["prefix"]:
        front = p[..., : c["prefix"]].transpose(0, 1).flatten(1, 3) @ vp
        out = out + front.unflatten(1, (b, group, n)).transpose(0, 1)
    out = torch.where(total > 0, out / total, 0.0)
    out = out.permute(0, 3, 1, 2, 4).flatten(2, 3).to(s["q"].dtype)
    if not c["lse"]:
        return [out]
    return [out, (total.log() + top).squeeze(-1).permute(0, 3, 1, 2).flatten(2, 3)]


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"rotary": _plain_rotary, "cache": _plain_cache, "attention": _plain_attention}[c["op"]](s)
    tg = s["tg"]
    if c["op"] == "rotary":
        y = tg.rotary(s["x"], s["table"], s["positions"])
        return [y.detach(), *torch.autograd.grad(y, s["x"], s["dy"])] if c["grad"] else [y]
    if c["op"] == "cache":
        q = tg.cache_write(s["cache"], s["k"], s["v"], s["slots"], s["table"], s["positions"], q=s["q"])
        return [q, *tg.cache_read(s["cache"], s["slots"], dtype=s["k"].dtype)]
    shared = dict(prefix=s["prefix"], prefix_length=c["prefix"]) if c["prefix"] else {}
    out = tg.cache_attention(s["q"], s["cache"], s["tables"], s["lengths"], return_lse=c["lse"], **shared)
    return list(out) if c["lse"] else [out]


# ---- definitions in 64 bits ------------------------------------------------------------------
def _exact_turn(x, angle, gain, layout, back=False):
    """x as complex numbers times gain * exp(i * angle), or its conjugate."""
    x, n = x.double(), angle.shape[-1]
    head, rest = x[..., : 2 * n], x[..., 2 * n:]
    pairs = head.unflatten(-1, (2, n)).transpose(-1, -2) if layout == "half" else head.unflatten(-1, (n, 2))
    w = torch.polar(torch.full_like(angle, gain), -angle if back else angle).unsqueeze(-2)
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * w)
    z = z.transpose(-1, -2) if layout == "half" else z
    return torch.cat((z.flatten(-2), rest), -1)


def _exact_values(x, c):
    """What the cache gives back for x (..., dim)."""
    x = x.double().unflatten(-1, (-1, c["block"]))
    r = x.abs().amax(-1, keepdim=True) / QMAX[c["format"]]
    if c["scales"] == "e8m0":
        s = torch.exp2(r.clamp(min=TINY).log2().ceil()).clamp(TINY, HUGE)
    else:
        s = r.to(torch.bfloat16).double().clamp(TINY, HUGE)
    y = x / s
    if c["format"].startswith("int"):
        y = y.round()
    else:  # floats of 3 or 1 mantissa bits, the smallest normal ones at 2^-6 and 1
        bits, least = (3, -6) if c["format"] == "fp8e4m3" else (1, 0)
        step = torch.exp2(y.abs().clamp(min=2.0 ** least).log2().floor() - bits)
        y = (y / step).round() * step
    return (y.clamp(-QMAX[c["format"]], QMAX[c["format"]]) * s).flatten(-2)


def _exact_decode(codes, scales, c):
    """The 64-bit values of stored codes and scales, through a table of all codes."""
    n = torch.arange(256 if BITS[c["format"]] == 8 else 16, dtype=torch.float64, device=codes.device)
    if c["format"] == "int8":
        values = n - 256 * (n > 127)
    elif c["format"] == "int4":
        values = n - 16 * (n > 7)
    else:
        e, m = (4, 3) if c["format"] == "fp8e4m3" else (2, 1)
        bias = 2 ** (e - 1) - 1
        sign = 1 - 2 * (n >= 2 ** (e + m)).double()
        exponent, fraction = (n % 2 ** (e + m)) // 2 ** m, n % 2 ** m / 2 ** m
        values = sign * torch.where(exponent > 0, (1 + fraction) * torch.exp2(exponent - bias), fraction * 2.0 ** (1 - bias))
    if BITS[c["format"]] == 4:
        codes = torch.stack((codes % 16, codes // 16), -1).flatten(-2)
    s = torch.exp2(scales.double() - 127) if scales.dtype == torch.uint8 else scales.double()
    return values[codes.int()] * s.repeat_interleave(c["block"], -1)


def exact(case, seed):
    s, c = _inputs(case, seed), case
    if c["op"] != "attention":
        angles, gain = _angles(c, "cuda")
        angles = angles[s["positions"]]
    if c["op"] == "rotary":
        y = _exact_turn(s["x"], angles, gain, c["layout"])
        return [y, _exact_turn(s["dy"], angles, gain, c["layout"], back=True)] if c["grad"] else [y]
    if c["op"] == "cache":
        return [_exact_turn(s["q"], angles, gain, c["layout"]),
                _exact_values(_exact_turn(s["k"], angles, gain, c["layout"]), c), _exact_values(s["v"], c)]
    if c["batch"] * c["queries"] * c["heads"] * (c["high"] + c["prefix"]) > 4e8:
        return None
    group, n = c["heads"] // c["kv_heads"], c["queries"]
    q = s["q"].double() / math.sqrt(c["dim"])
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    lse = torch.full(q.shape[:3], -math.inf, dtype=torch.float64, device="cuda")
    lengths = s["lengths"].tolist()
    p = s["prefix"].long()
    front = [_exact_decode(s[x][p], s[x + "_scales"][p], c).transpose(1, 2).flatten(0, 1)[: c["prefix"]] for x in "kv"]
    for b in range(c["batch"]):
        t = s["tables"][b].long()[: -(-lengths[b] // c["page"])]
        k, v = (torch.cat((front[i], _exact_decode(s[x][t], s[x + "_scales"][t], c).transpose(1, 2).flatten(0, 1)[: lengths[b]]))
                for i, x in enumerate("kv"))  # (keys, kv_heads, dim)
        place = torch.arange(k.shape[0], device="cuda")[None, :] - c["prefix"]
        hidden = place > torch.arange(n, device="cuda")[:, None] + (lengths[b] - n)
        hidden &= place >= 0
        x = torch.einsum("qhgd,thd->hgqt", q[b].unflatten(1, (c["kv_heads"], group)), k).masked_fill(hidden, -math.inf)
        w = torch.nan_to_num(torch.softmax(x, -1), nan=0.0)
        out[b] = torch.einsum("hgqt,thd->qhgd", w, v).flatten(1, 2)
        lse[b] = torch.logsumexp(x, -1).permute(2, 0, 1).flatten(1, 2)
    return [out, lse] if c["lse"] else [out]
