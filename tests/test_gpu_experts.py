"""Routing to experts, its plan, and the experts' products, against their formulas in 64 bits."""

import math

import pytest
import torch

import scaled_helpers as H

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def tg():
    import tinygrad_dx12_b200 as tg

    return tg


# ---- routing -----------------------------------------------------------------------------------
def ranked(v, n):
    """Indices of the n largest of each row, ties to the lowest index."""
    return torch.sort(v, dim=-1, descending=True, stable=True).indices[..., :n]


def route64(logits, k, scores="softmax", bias=None, groups=1, top_groups=1, group_best=1, renormalize=True, scale=1.0, live=None):
    x = logits.double()
    x = torch.where(x.isnan(), -math.inf, x).clamp(max=torch.finfo(torch.float32).max)
    dead = x == -math.inf
    if scores == "softmax":
        top = torch.where(dead, -1e300, x).amax(-1, keepdim=True)
        e = torch.where(dead, 0.0, torch.exp(x - top))
        s = e / e.sum(-1, keepdim=True)
    else:
        s = torch.where(dead, 0.0, 1 / (1 + torch.exp(-x)))
    choice = x
    if bias is not None:
        b = bias.double().clamp(max=torch.finfo(torch.float32).max)
        dead = dead | b.isnan() | (b == -math.inf)
        choice = s + torch.where(b.isnan(), 0.0, b)
    elif groups > 1 and group_best == 2:
        choice = s
    choice = torch.where(dead, -math.inf, choice)
    if groups > 1:
        part = choice.unflatten(-1, (groups, -1))
        two = part.gather(-1, ranked(part, group_best))
        some = (two > -math.inf).any(-1)
        best = torch.where(two > -math.inf, two, 0.0).sum(-1) if group_best == 2 else two[..., 0]
        best = torch.where(some, best, -math.inf)
        kept = torch.zeros_like(some).scatter_(-1, ranked(best, top_groups), True) & some
        choice = torch.where(kept.repeat_interleave(part.shape[-1], -1), choice, -math.inf)
    at = ranked(choice, k)
    can = choice.gather(-1, at) > -math.inf
    w, chosen = torch.where(can, s.gather(-1, at), 0.0), torch.where(can, x.gather(-1, at), -math.inf)
    if renormalize:  # in logarithms, for scores too small for 64 bits
        log = chosen if scores == "softmax" else chosen - torch.nn.functional.softplus(chosen)
        log = torch.where(can, log, -math.inf)
        top = torch.where(can, log, -1e300).amax(-1, keepdim=True)
        w = torch.where(can, torch.exp(log - top), 0.0)
        w = torch.where(can, w / w.sum(-1, keepdim=True), 0.0)
    at = torch.where(can, at, -1)
    if live is not None:
        at[live:], w[live:] = -1, 0.0
    return at.int(), w * scale


def check_plan(r, first=0):
    flat = r.indices.flatten().long() - first
    bins = torch.where((flat >= 0) & (flat < r.experts), flat, r.experts)
    assert torch.equal(r.rows.long(), torch.sort(bins, stable=True).indices)
    count = torch.bincount(bins, minlength=r.experts + 1)[: r.experts]
    assert torch.equal(r.offsets.long(), torch.cat((count.new_zeros(1), count.cumsum(0))))


def check_route(tg, logits, k, live=None, **kw):
    alive = None if live is None else torch.tensor([live], dtype=torch.int32, device="cuda")
    r = tg.route_experts(logits, k, live=alive, **kw)
    at, w = route64(logits, k, live=live, **kw)
    assert torch.equal(r.indices, at)
    # fp32: the exponential's 2 ulp and its argument's half (|x| 2^-24 of the score, up to 128 either way), sums of at
    # most 32 rounds and a tree, a division or two
    tol = w.abs() * (128 + 48) * 2.0 ** -23 + 2.0 ** -126
    assert bool(((r.weights.double() - w).abs() <= tol).all())
    check_plan(r)
    return r


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,k", [(1, 1), (3, 2), (32, 4), (33, 32), (64, 6), (128, 8), (200, 1), (256, 8), (512, 16), (1000, 10), (1024, 32)])
def test_route(tg, experts, k, scores, dtype):
    g = H.generator(experts)
    for tokens in (1, 5, 300):
        x = (torch.randn((tokens, experts), device="cuda", generator=g) * 3).to(dtype)
        for renormalize in (True, False):
            check_route(tg, x, k, scores=scores, renormalize=renormalize, scale=1.0 if renormalize else 2.5)
        check_route(tg, x, k, scores=scores, bias=torch.randn(experts, device="cuda", generator=g) * 0.1)


@pytest.mark.parametrize("experts,groups,top_groups,k", [(64, 8, 3, 8), (256, 8, 4, 8), (12, 3, 1, 4), (96, 32, 5, 6), (64, 64 // 2, 32, 10),
                                                         (40, 4, 4, 7), (1024, 16, 2, 32)])
@pytest.mark.parametrize("group_best", [1, 2])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_route_groups(tg, experts, groups, top_groups, k, group_best, scores):
    g = H.generator(experts + groups)
    x = torch.randn((257, experts), device="cuda", generator=g) * 2
    kw = dict(scores=scores, groups=groups, top_groups=top_groups, group_best=group_best)
    check_route(tg, x, k, **kw)
    check_route(tg, x, k, bias=torch.randn(experts, device="cuda", generator=g) * 0.05, **kw)
    x[3], x[4, ::2], x[5, 1:] = -math.inf, math.nan, -math.inf  # few experts or none left
    check_route(tg, x, k, **kw)


def test_route_ties(tg):
    """Equal logits: the lowest indices, in order; ties of groups too."""
    x = torch.zeros((3, 64), device="cuda")
    x[1, 10], x[1, 50], x[2, 63] = 1.0, 1.0, -0.0
    r = check_route(tg, x, 4)
    assert r.indices.tolist() == [[0, 1, 2, 3], [10, 50, 0, 1], [0, 1, 2, 3]]
    r = check_route(tg, x, 4, groups=8, top_groups=2, group_best=2, scores="sigmoid", bias=torch.zeros(64, device="cuda"))
    assert r.indices.tolist()[0] == [0, 1, 2, 3]
    g = H.generator(5)
    y = torch.randint(-2, 3, (500, 96), device="cuda", generator=g).to(torch.bfloat16)
    check_route(tg, y, 9)
    check_route(tg, y, 9, groups=6, top_groups=2)
    check_route(tg, y, 9, scores="sigmoid", bias=torch.randint(-1, 2, (96,), device="cuda", generator=g).float())


def test_route_near_ties_are_ordered_in_64_bits(tg):
    """Scores that fp32 cannot tell apart."""
    x = torch.full((1, 64), -20.0, device="cuda")
    x[0, 40], x[0, 7] = 18.000002, 18.0  # sigmoids of 1 - 1.5e-8: one fp32 number
    r = check_route(tg, x, 2, scores="sigmoid", bias=torch.zeros(64, device="cuda"))
    assert r.indices.tolist() == [[40, 7]]


def test_route_odd_logits(tg):
    """Infinities, NaN, the largest values; rows with fewer choices than k; scores that vanish in 32 bits."""
    big = torch.finfo(torch.float32).max
    x = torch.zeros((10, 40), device="cuda")
    x[0] = -math.inf
    x[1, 3:] = -math.inf
    x[2, ::2] = math.nan
    x[3, 5] = math.inf
    x[4, 5], x[4, 9] = math.inf, math.inf
    x[5], x[5, 2] = -big, big
    x[6] = math.nan
    x[7] = torch.linspace(-300, -200, 40)
    x[8] = torch.linspace(-1e30, -9e29, 40)
    x[9] = math.inf
    for scores in ("softmax", "sigmoid"):
        for kw in (dict(), dict(bias=torch.zeros(40, device="cuda")), dict(renormalize=False), dict(groups=4, top_groups=2)):
            r = check_route(tg, x, 6, scores=scores, **kw)
            assert not r.weights.isnan().any() and r.indices[0].eq(-1).all() and r.indices[6].eq(-1).all()
    b = torch.zeros(40, device="cuda")
    b[0], b[1], b[2], b[3] = -math.inf, math.nan, math.inf, -big
    check_route(tg, x, 6, bias=b)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_route_odd_logits_of_16_bits(tg, dtype):
    """Infinities above the type's largest value, zeros of both signs, subnormals, equal rows."""
    f = torch.finfo(dtype)
    x = torch.zeros((8, 70), device="cuda", dtype=dtype)
    x[0, 3], x[0, 60] = f.max, math.inf
    x[1, 3], x[1, 60], x[1, 61] = math.inf, f.max, -math.inf
    x[2], x[2, 5] = -f.max, -math.inf
    x[3, ::2] = -0.0
    x[4] = torch.arange(70, device="cuda") * f.smallest_normal / 128
    x[5] = -x[4]
    x[6, 10:] = math.nan
    x[7, 69], x[7, 0] = 1.0, 1.0
    for scores in ("softmax", "sigmoid"):
        for kw in (dict(), dict(renormalize=False), dict(groups=7, top_groups=3), dict(groups=7, top_groups=3, group_best=2),
                   dict(bias=torch.linspace(0, 1e-3, 70, device="cuda"))):
            check_route(tg, x, 6, scores=scores, **kw)


@pytest.mark.parametrize("live", [0, 1, 77, 100, 500])
def test_route_live(tg, live):
    g = H.generator(live)
    r = check_route(tg, torch.randn((100, 64), device="cuda", generator=g), 8, live=live)
    assert r.indices[live:].eq(-1).all() and int(r.offsets[-1]) == min(live, 100) * 8


def test_route_strides_and_empty(tg):
    g = H.generator(8)
    x = torch.randn((50, 200), device="cuda", generator=g)
    check_route(tg, x[:, 17:81], 5)
    check_route(tg, x[::3, :64], 5)
    check_route(tg, x.T[:, :32], 5)
    r = tg.route_experts(x[:0], 3)
    assert r.indices.shape == (0, 3) and r.offsets.eq(0).all()


@pytest.mark.parametrize("tokens,k,experts", [(1, 1, 1), (1000, 8, 64), (1025, 8, 1024), (9000, 1, 3), (40000, 8, 256), (70000, 16, 100)])
def test_plan(tg, tokens, k, experts):
    g = H.generator(tokens)
    at = torch.randint(-2, experts + 9, (tokens, k), device="cuda", generator=g, dtype=torch.int32)
    w = torch.rand((tokens, k), device="cuda", generator=g)
    check_plan(tg.plan_experts(at, w, experts))
    check_plan(tg.plan_experts(at, w, max(1, experts // 3), first=experts // 2), first=experts // 2)
    check_plan(tg.plan_experts(torch.full_like(at, experts - 1), w, experts))  # the same expert for all
    at[:, 0] = torch.iinfo(torch.int32).min
    at[:, -1] = torch.iinfo(torch.int32).max
    check_plan(tg.plan_experts(at, w, experts))


# ---- products ----------------------------------------------------------------------------------
def some_routing(tg, tokens, k, experts, g, holes=True, first=0):
    at = torch.rand((tokens, experts + first), device="cuda", generator=g).argsort(-1)[:, :k].to(torch.int32)
    if holes:
        at[torch.rand((tokens, k), device="cuda", generator=g) < 0.1] = -1
    return tg.plan_experts(at, torch.rand((tokens, k), device="cuda", generator=g), experts, first)


def pairs64(x, w, r, bias, **kw):
    """(results, tolerances) of every pair (tokens, k, columns); zeros without an expert."""
    cols = w.shape[1] // (2 if kw.get("gated") else 1)
    v = torch.zeros((r.tokens * r.k, cols), dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(v)
    ww, flat = H.weights(w), r.indices.flatten() - r.first
    per_pair = x.shape[0] != r.tokens
    for e in range(r.experts):
        at = (flat == e).nonzero().flatten()
        if len(at):
            v[at], tol[at] = H.product(x[at if per_pair else at // r.k], ww[e], None if bias is None else bias[e], **kw)
    return v, tol


@pytest.mark.parametrize("general", [True, False])
@pytest.mark.parametrize("fmt", sorted(H.BITS))
@pytest.mark.parametrize("tokens,k,experts,n,cols", [(1, 1, 4, 128, 128), (1, 4, 8, 200, 256), (7, 3, 5, 256, 128), (64, 8, 32, 320, 256),
                                                     (300, 2, 3, 192, 256)])
def test_expert_linear(tg, fmt, tokens, k, experts, n, cols, general):
    from tinygrad_dx12_b200 import experts as E

    g = H.generator(tokens + n)
    r = some_routing(tg, tokens, k, experts, g)
    w = H.make_weights((experts, n, cols), fmt, g)
    bias = torch.randn((experts, n), device="cuda", generator=g).bfloat16()
    x = tg.quantize(torch.randn((tokens, cols), device="cuda", generator=g))
    xx = H.values(x.codes, x.scales)
    for kw in (dict(), dict(bias=bias, activation="gelu"), dict(gated=True, activation="silu", bias=bias)):
        v, tol = pairs64(xx, w, r, **{"bias": None, **kw})
        H.check(E.expert_linear(x, w, r, dtype=torch.float32, _general=general, **kw), v, tol)
        H.check(E.expert_linear(x, w, r, dtype=torch.float16, _general=general, **kw), v, tol)
        if v.shape[1] % 32 == 0:
            H.check8(E.expert_linear(x, w, r, dtype=E4M3, _general=general, **kw), v, tol)
    if k > 1:
        x = tg.quantize(torch.randn((tokens * k, cols), device="cuda", generator=g))
        v, tol = pairs64(H.values(x.codes, x.scales), w, r, None)
        H.check(E.expert_linear(x, w, r, dtype=torch.bfloat16, _general=general), v, tol)


@pytest.mark.parametrize("general", [True, False])
@pytest.mark.parametrize("indices", [[[2, 2, 5]], [[1] * 20], [[0, 3, 0, -1, 3, 3]], [[2, 2], [2, 1]], [[4]]])
def test_the_same_expert_twice(tg, indices, general):
    """A token may name an expert more than once: each of its pairs is answered."""
    from tinygrad_dx12_b200 import experts as E

    g = H.generator(len(indices[0]))
    at = torch.tensor(indices, dtype=torch.int32, device="cuda")
    r = tg.plan_experts(at, torch.rand(at.shape, device="cuda", generator=g), 6)
    up, down = H.make_weights((6, 256, 256), "fp4_e2m1", g), H.make_weights((6, 256, 128), "fp6_e2m3", g)
    x = tg.quantize(torch.randn((len(indices), 256), device="cuda", generator=g))
    xx = H.values(x.codes, x.scales)
    for kw in (dict(), dict(gated=True, activation="silu")):
        v, tol = pairs64(xx, up, r, None, **kw)
        H.check(E.expert_linear(x, up, r, dtype=torch.float32, _general=general, **kw), v, tol)
    y = E.expert_mlp(x, up, down, r, dtype=torch.float32, _general=general)
    H.check(y, *mlp64(xx, up, down, r, "silu", True, None, None, None))


@pytest.mark.parametrize("count", [0, 1, 15, 16, 17, 112, 113, 224, 225, 500])
def test_expert_token_counts(tg, count):
    """One expert has ``count`` tokens, its neighbours none or the others."""
    g = H.generator(count)
    at = torch.full((512, 1), 2, dtype=torch.int32, device="cuda")
    at[count:] = 5
    r = tg.plan_experts(at, torch.ones((512, 1), device="cuda"), 7)
    w = H.make_weights((7, 256, 256), "fp4_e2m1", g)
    x = tg.quantize(torch.randn((512, 256), device="cuda", generator=g))
    for kw in (dict(), dict(gated=True)):
        v, tol = pairs64(H.values(x.codes, x.scales), w, r, None, **kw)
        H.check(tg.expert_linear(x, w, r, dtype=torch.float32, **kw), v, tol)


@pytest.mark.parametrize("tokens,k,experts,n,cols", [(900, 4, 12, 2048, 384), (2000, 1, 3, 4096, 640), (130, 8, 100, 512, 256)])
def test_expert_waves(tg, tokens, k, experts, n, cols):
    """Several tiles of tokens an expert and several tiles a CTA."""
    g = H.generator(tokens)
    r = some_routing(tg, tokens, k, experts, g, holes=False)
    w = H.make_weights((experts, n, cols), "fp4_e2m1", g)
    x = tg.quantize(torch.randn((tokens, cols), device="cuda", generator=g))
    xx = H.values(x.codes, x.scales)
    for kw in (dict(), dict(gated=True, activation="silu")):
        y = tg.expert_linear(x, w, r, dtype=torch.float32, **kw)
        H.check(y, *pairs64(xx, w, r, None, **kw))
        assert torch.equal(y, tg.expert_linear(x, w, r, dtype=torch.float32, **kw))


def mlp64(x, up, down, r, activation, gated, up_bias, down_bias, residual):
    """(result, tolerance). What lies between is quantised from values known to ``tol``: a code lies within half a step
    (2^-4 of the value, 2^-10 scales) of them, on either side, so the second product is of the 64-bit values and
    every term may move by that much, tol included."""
    v, tol = pairs64(x, up, r, up_bias, activation=activation, gated=gated)
    codes, scales = H.quantise(v.float())
    h = H.values(codes, scales)
    # values whose code the fp32 sums may turn over: their distance to a border is below tol (and fp32's rounding of v)
    s = torch.exp2(scales.double() - 127).repeat_interleave(32, -1)
    step = torch.maximum(torch.exp2(v.abs().clamp(min=1e-300).log2().floor() - 3), s * 2.0 ** -9)
    near = tol + v.abs() * 2.0 ** -23
    frac = (v.abs() / step) % 1.0
    border = (frac - 0.5).abs() * step <= near * 1.01
    top = v.abs().unflatten(-1, (-1, 32)).amax(-1, keepdim=True)
    ttop = near.unflatten(-1, (-1, 32)).amax(-1, keepdim=True)
    sb = s.unflatten(-1, (-1, 32))[..., :1]
    scale_border = ((top - 448 * sb).abs() <= ttop * 1.01) | ((top - 224 * sb).abs() <= ttop * 1.01)
    moved = torch.where(border, step, 0.0)
    moved = torch.maximum(moved, torch.where(scale_border.expand(*sb.shape[:-1], 32).flatten(-2), 2 * step, 0.0))
    out = torch.zeros((r.tokens, down.shape[1]), dtype=torch.float64, device="cuda")
    err = torch.zeros_like(out)
    y, ty = pairs64(h, down, r, down_bias)
    dd, flat = H.weights(down).abs(), r.indices.flatten() - r.first
    for e in range(r.experts):
        at = (flat == e).nonzero().flatten()
        if len(at):
            ty[at] += moved[at] @ dd[e].T
    w = torch.where((flat >= 0) & (flat < r.experts), r.weights.flatten(), 0.0).double()[:, None]
    out = (y * w).view(r.tokens, r.k, -1).sum(1)
    err = ((ty + y.abs() * (r.k + 2) * 2.0 ** -24) * w).view(r.tokens, r.k, -1).sum(1)
    if residual is not None:
        out = out + residual.double()
        err = err + out.abs() * 2.0 ** -23
    return out, err


@pytest.mark.parametrize("general", [False, True])
@pytest.mark.parametrize("tokens,k,experts,hidden,inner", [(1, 4, 32, 256, 128), (33, 2, 4, 384, 256), (64, 8, 16, 128, 64), (200, 1, 3, 256, 128)])
def test_expert_mlp(tg, tokens, k, experts, hidden, inner, general):
    from tinygrad_dx12_b200 import experts as E

    g = H.generator(tokens)
    r = some_routing(tg, tokens, k, experts, g)
    x = tg.quantize(torch.randn((tokens, hidden), device="cuda", generator=g))
    res = torch.randn((tokens, hidden), device="cuda", generator=g).bfloat16()
    for fmt, gated, activation, bias, residual, dtype in (("fp4_e2m1", True, "silu", False, res, torch.bfloat16),
                                                          ("fp6_e3m2", False, "gelu", True, None, torch.float32),
                                                          ("fp6_e2m3", True, "gelu_tanh", True, res, torch.float16)):
        up = H.make_weights((experts, inner * (2 if gated else 1), hidden), fmt, g)
        down = H.make_weights((experts, hidden, inner), fmt, g)
        ub = torch.randn(up.shape[:2], device="cuda", generator=g).half() if bias else None
        db = torch.randn(down.shape[:2], device="cuda", generator=g) if bias else None
        y = E.expert_mlp(x, up, down, r, activation, gated, ub, db, residual, dtype, _general=general)
        H.check(y, *mlp64(H.values(x.codes, x.scales), up, down, r, activation, gated, ub, db, residual))
        assert torch.equal(y, E.expert_mlp(x, up, down, r, activation, gated, ub, db, residual, dtype, _general=general))


def test_tokens_without_experts(tg):
    """Padded rows and tokens whose experts are another rank's: the residual, or zeros."""
    g = H.generator(21)
    x = tg.quantize(torch.randn((20, 256), device="cuda", generator=g))
    up, down = H.make_weights((4, 256, 256), "fp4_e2m1", g), H.make_weights((4, 256, 128), "fp4_e2m1", g)
    res = torch.randn((20, 256), device="cuda", generator=g)
    at = torch.full((20, 2), -1, dtype=torch.int32, device="cuda")
    at[5], at[6, 1] = torch.tensor([1, 3], dtype=torch.int32), 7
    w = torch.ones((20, 2), device="cuda")
    w[0] = math.nan  # of no expert: not read into a result
    r = tg.plan_experts(at, w, 4)
    y = tg.expert_mlp(x, up, down, r, residual=res, dtype=torch.float32)
    assert torch.equal(torch.cat((y[:5], y[6:])), torch.cat((res[:5], res[6:]))) and not torch.equal(y[5], res[5])
    z = tg.expert_mlp(x, up, down, r, dtype=torch.float32)
    assert z[:5].eq(0).all() and z[6:].eq(0).all()
    p = tg.expert_linear(x, up, r, dtype=torch.float32)
    assert p[:10].eq(0).all() and p[12:].eq(0).all()
    none = tg.plan_experts(torch.full_like(at, -1), w, 4)
    assert tg.expert_mlp(x, up, down, none).eq(0).all() and tg.expert_linear(x, up, none).eq(0).all()


def test_shards_of_experts_add_up(tg):
    """Two ranks' experts, each with its own plan: their sums are the whole's."""
    g = H.generator(22)
    x = tg.quantize(torch.randn((40, 256), device="cuda", generator=g))
    up, down = H.make_weights((8, 256, 256), "fp4_e2m1", g), H.make_weights((8, 256, 128), "fp4_e2m1", g)
    whole = tg.route_experts(torch.randn((40, 8), device="cuda", generator=g), 3)
    y = tg.expert_mlp(x, up, down, whole, dtype=torch.float32)
    parts = []
    for first in (0, 4):
        cut = lambda w: tg.PackedTensor(w.data.view(8, -1)[first:first + 4].reshape(-1).clone(), w.format, (4, *w.shape[1:]),  # noqa: E731
                                        w.scales.view(torch.uint8)[first:first + 4].clone().view(torch.float8_e8m0fnu), 32)
        r = tg.plan_experts(whole.indices, whole.weights, 4, first)
        parts.append(tg.expert_mlp(x, cut(up), cut(down), r, dtype=torch.float32))
    assert torch.allclose(parts[0] + parts[1], y, rtol=0, atol=float(y.abs().max()) * 2.0 ** -21)


def test_block_of_a_decoder(tg):
    """Norm, router, experts and residual as a layer has them, eager and recorded: other tokens, other experts, a shorter
    batch at replay."""
    g = H.generator(23)
    hidden, inner, experts, k = 512, 256, 16, 4
    up, down = H.make_weights((experts, 2 * inner, hidden), "fp4_e2m1", g), H.make_weights((experts, hidden, inner), "fp4_e2m1", g)
    router = torch.randn((experts, hidden), device="cuda", generator=g) * 0.05
    weight = 1 + 0.1 * torch.randn(hidden, device="cuda", generator=g)

    def block(h, y, live):
        x8, h2 = tg.rms_norm(y, weight, residual=h, dtype=E4M3)
        logits = tg.rms_norm(h2, weight, dtype=torch.float32) @ router.T
        r = tg.route_experts(logits, k, live=live)
        return tg.expert_mlp(x8, up, down, r, residual=h2), r.indices

    def inputs(live):
        return (torch.randn((48, hidden), device="cuda", generator=g).bfloat16(), torch.randn((48, hidden), device="cuda", generator=g).bfloat16(),
                torch.tensor([live], dtype=torch.int32, device="cuda"))

    sets = [inputs(n) for n in (48, 31, 0, 1)]
    want = [block(*s) for s in sets]
    step, other = tg.GraphStep(block, *sets[0]), tg.GraphStep(block, *sets[1])
    side = torch.cuda.Stream()
    for s, (y, at) in zip(sets, want):
        a, b = step(*s)
        assert torch.equal(a, y) and torch.equal(b, at)
        live = int(s[2])
        h2 = (s[0].float() + s[1].float()).bfloat16()
        assert torch.equal(a[live:], h2[live:]) and (live == 0 or not torch.equal(a[:live], h2[:live]))
    torch.cuda.synchronize()
    for _ in range(20):
        a = step(*sets[1])
        with torch.cuda.stream(side):
            c = other(*sets[3])
            d = block(*sets[0])
    torch.cuda.synchronize()
    assert torch.equal(a[0], want[1][0]) and torch.equal(c[0], want[3][0]) and torch.equal(d[0], want[0][0])
