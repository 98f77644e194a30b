"""Measured cases of 8-bit activations between packed projections: the RMS norm that adds the residual and
quantises, the product of block-scaled activations with packed weights and its epilogue, the routing of
tokens to experts, and the experts' products.

``run`` computes each in its plain form (elementary torch operations in 32 bits, 64 for the choice of
experts) or, where ``own`` is true, through the package's public calls. ``exact`` restates the definitions
in 64 bits.

Block-scaled activations, which both forms follow to the bit: a block of 32 values along the last axis has
r = max|x| * (1 / 448) and as its scale s the smallest power of two that is not below r, held within
[2^-100, 2^100]; the code of x is x / s rounded to the nearest E4M3 value, ties to even, and stands for
code * s. Weights are FP4 E2M1 or FP6 codes with a power of two for every 32 of a row.
"""

from __future__ import annotations

import math

import torch

own = False

BLOCK, QMAX = 32, 448.0
DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
BITS = {"fp4_e2m1": 4, "fp6_e2m3": 6, "fp6_e3m2": 6}
MANTISSA = {"fp4_e2m1": (2, 1), "fp6_e2m3": (2, 3), "fp6_e3m2": (3, 2)}  # exponent bits, mantissa bits


# ---- cases -----------------------------------------------------------------------------------
def _norm(name, **kw):
    base = dict(name=name, op="norm", rows=1, cols=4096, dtype="bfloat16", residual=True, eight=True)
    return {**base, **kw}


def _linear(name, **kw):
    base = dict(name=name, op="linear", rows=1, out=4096, inner=4096, format="fp4_e2m1", bias=False, activation="none",
                gated=False, residual=False, dtype="bfloat16", eight=False)
    return {**base, **kw}


def _route(name, **kw):
    base = dict(name=name, op="route", rows=1, experts=64, k=8, scores="softmax", bias=False, groups=1, top_groups=1,
                group_best=1, renormalize=True, scale=1.0, dtype="float32")
    return {**base, **kw}


def _experts(name, **kw):
    base = dict(name=name, op="experts", rows=1, hidden=4096, inter=2048, experts=32, k=4, format="fp4_e2m1",
                activation="silu", dtype="bfloat16", residual=False, bias=False)
    return {**base, **kw}


def listed():
    return [
        # a decode step of the 70B-shaped stack: the norm before a projection
        _norm("norm, one token", cols=8192),
        # a prompt of odd length of the 8B-shaped stack, 16-bit output for what is not quantised
        _norm("norm, 1999 tokens, 16 bits", rows=1999, dtype="float16", eight=False),
        # a batch of prompts of the 70B-shaped stack
        _norm("norm, 16384 tokens", rows=16384, cols=8192),
        # a decode step: the 70B-shaped down projection, added to the residual stream
        _linear("linear, one token, residual", out=8192, inner=28672, residual=True),
        # a small decode batch through the 70B-shaped gate|up projections, quantised for the next product
        _linear("linear, 33 tokens, gated", rows=33, out=57344, inner=8192, activation="silu", gated=True, eight=True),
        # a prompt over 6-bit weights with a bias (the benchmark's prefill matrix)
        _linear("linear, 4096 tokens, FP6, bias", rows=4096, out=14336, inner=4096, format="fp6_e2m3", bias=True,
                activation="gelu", dtype="float16"),
        # a decode step's token: latency counts
        _route("route, one token", experts=128),
        # a prompt of odd length over groups of experts, with a balancing bias
        _route("route, 1999 tokens, groups", rows=1999, experts=256, scores="sigmoid", bias=True, groups=8, top_groups=4,
               group_best=2, scale=2.5),
        # a batch of prompts, weights as the softmax gives them
        _route("route, 32768 tokens", rows=32768, experts=64, k=6, renormalize=False, dtype="bfloat16"),
        # one request's token through its four experts
        _experts("experts, one token", residual=True),
        # a decode batch that touches nearly all experts
        _experts("experts, 64 tokens", rows=64, experts=128, k=8, inter=1024, residual=True),
        # a prompt's chunk
        _experts("experts, 4001 tokens", rows=4001, experts=64, k=8, format="fp6_e3m2"),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    limit = [work(c) for c in listed()]
    most = {k: max(w[k] for w in limit) for k in ("bytes", "flops")}
    while True:
        op = rng.choice(("norm", "linear", "route", "experts"))
        half, fmt = rng.choice(("float16", "bfloat16")), rng.choice(sorted(BITS))
        if op == "norm":
            c = _norm("", rows=_spread(rng, 1, 16384), cols=32 * _spread(rng, 2, 512), dtype=rng.choice(sorted(DTYPES)),
                      residual=rng.random() < 0.7, eight=rng.random() < 0.7)
        elif op == "linear":
            gated, eight = rng.random() < 0.4, rng.random() < 0.4
            step = (32 if eight else 1) * (2 if gated else 1)
            c = _linear("", rows=_spread(rng, 1, 8192), out=step * max(1, _spread(rng, 64, 57344) // step),
                        inner=128 * _spread(rng, 2, 224), format=fmt, bias=rng.random() < 0.4, gated=gated, eight=eight,
                        activation=rng.choice(("none", "relu", "silu", "gelu", "gelu_tanh")),
                        residual=not eight and rng.random() < 0.4, dtype=rng.choice((half, half, "float32")))
        elif op == "route":
            groups = rng.choice((1, 1, 2, 4, 8))
            experts = groups * _spread(rng, 2, 512 // groups)
            top_groups = rng.randint(1, groups)
            k = rng.randint(1, min(16, experts // groups * top_groups))
            c = _route("", rows=_spread(rng, 1, 32768), experts=experts, k=k, scores=rng.choice(("softmax", "sigmoid")),
                       bias=rng.random() < 0.5, groups=groups, top_groups=top_groups, group_best=rng.choice((1, 2)),
                       renormalize=rng.random() < 0.6, scale=rng.choice((1.0, 1.0, 2.5)), dtype=rng.choice(sorted(DTYPES)))
        else:
            experts = _spread(rng, 4, 256)
            c = _experts("", rows=_spread(rng, 1, 4096), hidden=128 * _spread(rng, 2, 56), inter=128 * _spread(rng, 1, 32),
                         experts=experts, k=rng.randint(1, min(8, experts)), format=fmt, dtype=half,
                         activation=rng.choice(("silu", "gelu", "gelu_tanh")), residual=rng.random() < 0.5,
                         bias=rng.random() < 0.3)
        del c["name"]
        w = work(c)
        # the plain form's weights and products in 32 bits bound what a case may cost there
        plain = {"linear": lambda: c["out"] * c["inner"] < 6e8 and c["rows"] * c["out"] < 3e8,
                 "experts": lambda: c["experts"] * c["hidden"] * c["inter"] < 1.2e9}.get(op, lambda: True)()
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"] and plain:
            return c


def _touched(c):
    """Experts that are chosen at least once when every token's choice is as good as any."""
    return c["experts"] * (1.0 - (1.0 - c["k"] / c["experts"]) ** c["rows"])


def work(case):
    c, size = case, 4 if case["dtype"] == "float32" else 2
    if c["op"] == "norm":
        n = c["rows"] * c["cols"]
        # 8-bit rows are written, and read back as the 16-bit values they stand for
        back = n * (2 * (1 + 1 / BLOCK) + 2) if c["eight"] else n * size
        return {"bytes": n * size * (3 if c["residual"] else 1) + back + 4 * c["cols"], "flops": 4.0 * n}
    if c["op"] == "linear":
        m, n, k = c["rows"], c["out"], c["inner"]
        y = m * (n // 2 if c["gated"] else n)
        out = y * (2 * (1 + 1 / BLOCK) + 2) if c["eight"] else y * size
        weights = n * k * (BITS[c["format"]] / 8 + 1 / BLOCK)
        return {"bytes": weights + m * k * (1 + 1 / BLOCK) + out + (y * size if c["residual"] else 0) + (2 * n if c["bias"] else 0),
                "flops": 2.0 * m * n * k}
    if c["op"] == "route":
        return {"bytes": c["rows"] * (c["experts"] * size + c["k"] * 12) + 4 * c["experts"],
                "flops": 8.0 * c["rows"] * c["experts"]}
    per = 3 * c["hidden"] * c["inter"]
    weights = _touched(c) * per * (BITS[c["format"]] / 8 + 1 / BLOCK)
    rows = c["rows"] * c["hidden"] * (1 + 1 / BLOCK + 2 + (2 if c["residual"] else 0)) + c["rows"] * c["k"] * 8
    return {"bytes": weights + rows, "flops": 2.0 * c["rows"] * c["k"] * per}


# ---- inputs ----------------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(1_000_003 * seed + 29)
    return g


def _normal(shape, g, dtype):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _stream(shape, g, dtype):
    """Rows of a residual stream: a few channels many times larger than the others."""
    gain = torch.ones(shape[-1], device="cuda")
    gain[:: max(1, shape[-1] // 8)] = 20.0
    return (torch.randn(shape, generator=g, device="cuda") * gain).to(dtype)


def _packed(shape, fmt, g):
    """Random codes of ``shape`` back to back, and scale bytes that keep products of unit rows near one."""
    codes = torch.randint(0, 256, (math.prod(shape) * BITS[fmt] // 8,), dtype=torch.uint8, device="cuda", generator=g)
    size = {"fp4_e2m1": 2.9, "fp6_e2m3": 3.4, "fp6_e3m2": 9.6}[fmt]  # root mean square of random codes
    middle = round(-math.log2(size * math.sqrt(shape[-1])))
    scales = torch.randint(middle - 1, middle + 2, (*shape[:-1], shape[-1] // BLOCK), device="cuda", generator=g)
    return codes, (scales + 127).to(torch.uint8)


def _inputs(case, seed):
    """Every tensor of a case, from the seed alone."""
    c, g = case, _generator(seed)
    dtype = DTYPES[c["dtype"]]
    s = {"case": c}
    if c["op"] == "norm":
        s["x"] = _normal((c["rows"], c["cols"]), g, dtype)
        s["weight"] = 1.0 + 0.1 * torch.randn(c["cols"], generator=g, device="cuda")
        if c["residual"]:
            s["residual"] = _stream((c["rows"], c["cols"]), g, dtype)
    elif c["op"] == "linear":
        m, n, k = c["rows"], c["out"], c["inner"]
        s["x"], s["x_scales"] = _quantise(_normal((m, k), g, torch.float32))
        s["w"], s["w_scales"] = _packed((n, k), c["format"], g)
        if c["bias"]:
            s["bias"] = _normal((n,), g, torch.bfloat16)
        if c["residual"]:
            s["residual"] = _stream((m, n // 2 if c["gated"] else n), g, dtype)
    elif c["op"] == "route":
        s["logits"] = (torch.randn((c["rows"], c["experts"]), generator=g, device="cuda") * 1.5).to(dtype)
        if c["bias"]:
            s["bias"] = torch.randn(c["experts"], generator=g, device="cuda") * 0.05
    else:
        t, h, i, e = c["rows"], c["hidden"], c["inter"], c["experts"]
        s["x"], s["x_scales"] = _quantise(_normal((t, h), g, torch.float32))
        s["up"], s["up_scales"] = _packed((e, 2 * i, h), c["format"], g)
        s["down"], s["down_scales"] = _packed((e, h, i), c["format"], g)
        # some experts are more popular than others
        taste = torch.randn(e, generator=g, device="cuda") * 0.5
        logits = torch.randn((t, e), generator=g, device="cuda") + taste
        chosen = torch.topk(logits, c["k"], dim=-1)
        s["indices"] = chosen.indices.to(torch.int32)
        s["weights"] = torch.softmax(chosen.values, -1)
        s["most"] = int(torch.bincount(s["indices"].flatten().long(), minlength=e).max())
        if c["bias"]:
            s["up_bias"], s["down_bias"] = _normal((e, 2 * i), g, torch.bfloat16), _normal((e, h), g, torch.bfloat16)
        if c["residual"]:
            s["residual"] = _stream((t, h), g, dtype)
    return s


def prepare(case, seed):
    return _inputs(case, seed)


# ---- plain forms -----------------------------------------------------------------------------
def _quantise(x):
    """E4M3 codes (..., dim) and scale bytes (..., dim / 32) of x."""
    x = x.float().unflatten(-1, (-1, BLOCK))
    r = x.abs().amax(-1) * (1.0 / QMAX)
    e = ((r.view(torch.int32) + 0x7FFFFF) >> 23).clamp(27, 227)
    y = x * (e << 23).view(torch.float32).reciprocal()[..., None]
    return y.clamp(-QMAX, QMAX).to(torch.float8_e4m3fn).flatten(-2), e.to(torch.uint8)


def _values(codes, scales):
    """The values (..., dim) in 32 bits that activations' codes and scale bytes stand for."""
    s = (scales.int() << 23).view(torch.float32)
    return (codes.float().unflatten(-1, (-1, BLOCK)) * s[..., None]).flatten(-2)


def _weights(codes, scales, shape, fmt):
    """The values of ``shape`` in 32 bits that packed codes and scale bytes stand for."""
    if BITS[fmt] == 4:
        n = torch.stack((codes & 15, codes >> 4), -1)
    else:
        b = codes.view(-1, 3).int()
        word = b[:, 0] | (b[:, 1] << 8) | (b[:, 2] << 16)
        n = torch.stack((word & 63, (word >> 6) & 63, (word >> 12) & 63, word >> 18), -1)
    ebits, mbits = MANTISSA[fmt]
    every = torch.arange(2 ** BITS[fmt], dtype=torch.float32, device=codes.device)
    sign = 1 - 2 * (every >= 2 ** (ebits + mbits)).float()
    exponent = (every % 2 ** (ebits + mbits)).div(2 ** mbits, rounding_mode="floor")
    fraction = every % 2 ** mbits / 2 ** mbits
    bias = 2 ** (ebits - 1) - 1
    table = sign * torch.where(exponent > 0, (1 + fraction) * torch.exp2(exponent - bias), fraction * 2.0 ** (1 - bias))
    s = (scales.int() << 23).view(torch.float32)
    return (table[n.int()].view(*shape[:-1], -1, BLOCK) * s[..., None]).view(shape)


def _activate(v, name):
    if name == "relu":
        return v.clamp(min=0)
    if name == "silu":
        return v / (1 + torch.exp(-v))
    if name == "gelu":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))
    return v


def _epilogue(v, c):
    """Activation and gate of a product's columns."""
    if not c.get("gated", True):
        return _activate(v, c["activation"])
    gate, up = v.chunk(2, -1)
    return _activate(gate, c["activation"]) * up


def _plain_norm(s):
    c, x = s["case"], s["x"]
    total = (x.float() + s["residual"].float()).to(x.dtype) if c["residual"] else x
    t = total.float()
    y = t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-6) * s["weight"]
    y = _values(*_quantise(y)).to(torch.bfloat16) if c["eight"] else y.to(x.dtype)
    return [y, total] if c["residual"] else [y]


def _plain_linear(s):
    c = s["case"]
    v = _values(s["x"], s["x_scales"]) @ _weights(s["w"], s["w_scales"], (c["out"], c["inner"]), c["format"]).T
    if c["bias"]:
        v = v + s["bias"].float()
    v = _epilogue(v, c)
    if c["residual"]:
        v = v + s["residual"].float()
    return [_values(*_quantise(v)).to(torch.bfloat16) if c["eight"] else v.to(DTYPES[c["dtype"]])]


def _rank(v, k):
    """The k largest of each row, ties to the lowest index."""
    order = torch.sort(v, dim=-1, descending=True, stable=True)
    return order.values[..., :k], order.indices[..., :k]


def _choose(c, scores, choice):
    """Chosen experts of each row and their weights."""
    if c["groups"] > 1:
        size = c["experts"] // c["groups"]
        grouped = choice.unflatten(-1, (c["groups"], size))
        best = _rank(grouped, min(c["group_best"], size))[0].sum(-1)
        kept = torch.zeros_like(best, dtype=torch.bool).scatter_(-1, _rank(best, c["top_groups"])[1], True)
        choice = torch.where(kept[..., None], grouped, -math.inf).flatten(-2)
    indices = _rank(choice, c["k"])[1]
    weights = scores.gather(-1, indices)
    if c["renormalize"]:
        weights = weights / weights.sum(-1, keepdim=True)
    return indices, weights * c["scale"]


def _plan(indices, experts):
    """Where each expert's pairs begin, and the pairs in the order of their experts."""
    flat = indices.flatten()
    rows = torch.sort(flat, stable=True).indices
    count = torch.zeros(experts + 1, dtype=torch.int64, device=flat.device)
    count[1:].index_add_(0, flat.long(), torch.ones_like(flat, dtype=torch.int64))
    return count.cumsum(0).int(), rows.int()


def _plain_route(s):
    c = s["case"]
    x = s["logits"].double()
    if c["scores"] == "softmax":
        e = (x - x.amax(-1, keepdim=True)).exp()
        scores = e / e.sum(-1, keepdim=True)
    else:
        scores = 1 / (1 + (-x).exp())
    # without a bias or a sum of scores the choice is the logits' own
    choice = scores + s["bias"].double() if c["bias"] else scores if c["groups"] > 1 and c["group_best"] > 1 else x
    indices, weights = _choose(c, scores, choice)
    offsets, rows = _plan(indices, c["experts"])
    return [indices.int(), weights.float(), offsets, rows]


def _plain_experts(s):
    """Every expert's tokens side by side, as many places for each as the most popular one has."""
    c = s["case"]
    t, h, i, e, k, most = c["rows"], c["hidden"], c["inter"], c["experts"], c["k"], s["most"]
    offsets, rows = _plan(s["indices"], e)
    expert = s["indices"].flatten()[rows.long()].long()
    place = torch.arange(t * k, device="cuda") - offsets[expert]
    x = torch.zeros((e, most, h), device="cuda")
    x[expert, place] = _values(s["x"], s["x_scales"])[rows.long() // k]
    v = x @ _weights(s["up"], s["up_scales"], (e, 2 * i, h), c["format"]).transpose(1, 2)
    if c["bias"]:
        v = v + s["up_bias"].float()[:, None]
    v = _values(*_quantise(_epilogue(v, c)))
    y = v @ _weights(s["down"], s["down_scales"], (e, h, i), c["format"]).transpose(1, 2)
    if c["bias"]:
        y = y + s["down_bias"].float()[:, None]
    pairs = torch.empty((t * k, h), device="cuda")
    pairs[rows.long()] = y[expert, place]
    out = (pairs.view(t, k, h) * s["weights"][..., None]).sum(1)
    if c["residual"]:
        out = out + s["residual"].float()
    return [out.to(DTYPES[c["dtype"]])]


# ---- the framework's calls -------------------------------------------------------------------
def _handles(s):
    """The framework's own objects over a state's tensors, made once as a program that serves would."""
    import tinygrad_dx12_b200 as tg

    c, e8 = s["case"], torch.float8_e8m0fnu
    s["tg"] = tg
    if "x_scales" in s:
        s["own_x"] = tg.BlockScaled(s["x"], s["x_scales"].view(e8))
    if c["op"] == "linear":
        s["own_w"] = tg.PackedTensor(s["w"], c["format"], (c["out"], c["inner"]), s["w_scales"].view(e8), BLOCK)
    if c["op"] == "experts":
        e, h, i = c["experts"], c["hidden"], c["inter"]
        s["own_up"] = tg.PackedTensor(s["up"], c["format"], (e, 2 * i, h), s["up_scales"].view(e8), BLOCK)
        s["own_down"] = tg.PackedTensor(s["down"], c["format"], (e, h, i), s["down_scales"].view(e8), BLOCK)


def _own(s):
    if "tg" not in s:
        _handles(s)
    tg, c = s["tg"], s["case"]
    activation = None if c.get("activation") == "none" else c.get("activation")
    if c["op"] == "norm":
        y = tg.rms_norm(s["x"], s["weight"], eps=1e-6, residual=s.get("residual"),
                        dtype=torch.float8_e4m3fn if c["eight"] else s["x"].dtype)
        y, *total = y if c["residual"] else (y,)
        return [y.values(torch.bfloat16) if c["eight"] else y, *total]
    if c["op"] == "linear":
        y = tg.scaled_linear(s["own_x"], s["own_w"], bias=s.get("bias"), activation=activation, gated=c["gated"],
                             residual=s.get("residual"), dtype=torch.float8_e4m3fn if c["eight"] else DTYPES[c["dtype"]])
        return [y.values(torch.bfloat16) if c["eight"] else y]
    if c["op"] == "route":
        r = tg.route_experts(s["logits"], c["k"], scores=c["scores"], bias=s.get("bias"), groups=c["groups"],
                             top_groups=c["top_groups"], group_best=c["group_best"], renormalize=c["renormalize"],
                             scale=c["scale"])
        return [r.indices, r.weights, r.offsets, r.rows]
    routing = tg.plan_experts(s["indices"], s["weights"], c["experts"])
    return [tg.expert_mlp(s["own_x"], s["own_up"], s["own_down"], routing, activation=activation, gated=True,
                          up_bias=s.get("up_bias"), down_bias=s.get("down_bias"), residual=s.get("residual"),
                          dtype=DTYPES[c["dtype"]])]


def run(state):
    if own:
        return _own(state)
    plain = {"norm": _plain_norm, "linear": _plain_linear, "route": _plain_route, "experts": _plain_experts}
    return plain[state["case"]["op"]](state)


# ---- definitions in 64 bits ------------------------------------------------------------------
def _exact_quantised(x):
    """What block-scaled E4M3 gives back for x (..., dim)."""
    x = x.reshape(*x.shape[:-1], -1, BLOCK)
    r = x.abs().amax(-1, keepdim=True) / QMAX
    s = torch.exp2(r.clamp(min=2.0 ** -100).log2().ceil()).clamp(2.0 ** -100, 2.0 ** 100)
    y = x / s
    step = torch.exp2(y.abs().clamp(min=2.0 ** -6).log2().floor() - 3)  # three mantissa bits, subnormal below 2^-6
    return (((y / step).round() * step).clamp(-QMAX, QMAX) * s).flatten(-2)


def _exact_values(codes, scales):
    n = torch.arange(256, dtype=torch.float64, device=codes.device)
    exponent, fraction = n % 128 // 8, n % 8 / 8
    table = torch.where(exponent > 0, (1 + fraction) * torch.exp2(exponent - 7), fraction * 2.0 ** -6) * torch.where(n > 127, -1.0, 1.0)
    return table[codes.view(torch.uint8).int()] * torch.exp2(scales.double() - 127).repeat_interleave(BLOCK, -1)


def _exact_weights(codes, scales, fmt):
    """Values (..., K) of codes as bytes (..., K * bits / 8), bit by bit."""
    bits, (ebits, mbits) = BITS[fmt], MANTISSA[fmt]
    stream = (codes[..., None] >> torch.arange(8, dtype=torch.uint8, device=codes.device)) & 1
    stream = stream.flatten(-2).unflatten(-1, (-1, bits)).double()
    at = lambda low, high: (stream[..., low:high] * 2.0 ** torch.arange(high - low, device=codes.device)).sum(-1)  # noqa: E731
    fraction, exponent, bias = at(0, mbits) / 2 ** mbits, at(mbits, mbits + ebits), 2 ** (ebits - 1) - 1
    v = torch.where(exponent > 0, (1 + fraction) * torch.exp2(exponent - bias), fraction * 2.0 ** (1 - bias))
    return v * (1 - 2 * stream[..., -1]) * torch.exp2(scales.double() - 127).repeat_interleave(BLOCK, -1)


def _exact_activation(v, name):
    if name == "relu":
        return torch.where(v > 0, v, 0.0)
    if name == "silu":
        return v * torch.sigmoid(v)
    if name == "gelu":
        return v * torch.special.ndtr(v)
    if name == "gelu_tanh":
        return v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v))
    return v


def _exact_gate(v, name):
    half = v.shape[-1] // 2
    return _exact_activation(v[..., :half], name) * v[..., half:]


def _by_rows(codes, rows):
    return codes.view(rows, -1)


def _exact_linear(s, c):
    x, out = _exact_values(s["x"], s["x_scales"]), []
    codes = _by_rows(s["w"], c["out"])
    for first in range(0, c["out"], 4096):  # some rows of the matrix at a time: its bits as numbers are large
        out.append(x @ _exact_weights(codes[first:first + 4096], s["w_scales"][first:first + 4096], c["format"]).T)
    v = torch.cat(out, -1)
    if c["bias"]:
        v = v + s["bias"].double()
    v = _exact_gate(v, c["activation"]) if c["gated"] else _exact_activation(v, c["activation"])
    if c["residual"]:
        v = v + s["residual"].double()
    return _exact_quantised(v) if c["eight"] else v


def _exact_experts(s, c):
    x = _exact_values(s["x"], s["x_scales"])
    up, down = (s[n].view(c["experts"], r, -1) for n, r in (("up", 2 * c["inter"]), ("down", c["hidden"])))
    out = s["residual"].double() if c["residual"] else torch.zeros_like(x)
    for e in range(c["experts"]):
        token, slot = (s["indices"] == e).nonzero(as_tuple=True)
        if not len(token):
            continue
        v = x[token] @ _exact_weights(up[e], s["up_scales"][e], c["format"]).T
        v = v + s["up_bias"][e].double() if c["bias"] else v
        v = _exact_quantised(_exact_gate(v, c["activation"])) @ _exact_weights(down[e], s["down_scales"][e], c["format"]).T
        v = v + s["down_bias"][e].double() if c["bias"] else v
        out = out.index_add(0, token, v * s["weights"][token, slot].double()[:, None])
    return out


def _exact_route(s, c):
    x = s["logits"].double()
    scores = torch.softmax(x, -1) if c["scores"] == "softmax" else torch.sigmoid(x)
    summed = c["groups"] > 1 and c["group_best"] > 1
    choice = scores + s["bias"].double() if c["bias"] else scores if summed else x
    size = c["experts"] // c["groups"]
    order = lambda v: torch.argsort(-v, dim=-1, stable=True)  # noqa: E731
    if c["groups"] > 1:
        part = choice.view(-1, c["groups"], size)
        best = part.gather(-1, order(part)[..., :c["group_best"]]).sum(-1)
        place = torch.argsort(order(best), dim=-1)  # how many groups come before each
        choice = choice.masked_fill((place >= c["top_groups"]).repeat_interleave(size, -1), -math.inf)
    indices = order(choice)[:, :c["k"]]
    weights = torch.gather(scores, 1, indices)
    if c["renormalize"]:
        weights = weights / weights.sum(1, keepdim=True)
    flat = indices.flatten()
    offsets = torch.searchsorted(torch.sort(flat).values, torch.arange(c["experts"] + 1, device="cuda"))
    return [indices.int(), weights * c["scale"], offsets.int(), torch.argsort(flat, stable=True).int()]


def exact(case, seed):
    s, c = _inputs(case, seed), case
    if c["op"] == "norm":
        total = s["x"].double() + s["residual"].double() if c["residual"] else s["x"].double()
        t = total.to(s["x"].dtype).double()  # the stream is held in its own type, and the norm is of what it holds
        y = t / (t.square().mean(-1, keepdim=True) + 1e-6).sqrt() * s["weight"].double()
        y = _exact_quantised(y) if c["eight"] else y
        return [y, total] if c["residual"] else [y]
    if c["op"] == "linear":
        return [_exact_linear(s, c)]
    if c["op"] == "route":
        return _exact_route(s, c)
    return [_exact_experts(s, c)]
