"""Plain restatements for the tests of 8-bit activations and experts, from their formulas: values and sums in
float64; the quantisation's own operations in float32, where each is one IEEE rounding."""

from __future__ import annotations

import math

import torch

QMAX = 448.0
BITS = {"fp4_e2m1": 4, "fp6_e2m3": 6, "fp6_e3m2": 6}
SHAPE = {"fp4_e2m1": (2, 1, 1), "fp6_e2m3": (2, 3, 1), "fp6_e3m2": (3, 2, 3)}  # exponent, mantissa, bias


def quantise(x):
    """(E4M3 codes, scale bytes) of x (..., dim) in float32."""
    x = x.float().unflatten(-1, (-1, 32))
    top = x.abs().amax(-1)
    r = top * torch.tensor(1.0 / QMAX, dtype=torch.float32, device=x.device)
    e = ((r.view(torch.int32) + 0x7FFFFF) >> 23).clamp(27, 227)
    nan = x.isnan().any(-1)
    y = (x * torch.exp2(127.0 - e.double()).float()[..., None]).clamp(-QMAX, QMAX)
    y = torch.where(nan[..., None], 0.0, y)
    return y.to(torch.float8_e4m3fn).flatten(-2), torch.where(nan, 255, e).to(torch.uint8)


def values(codes, scales):
    """What codes and scale bytes stand for, float64."""
    s = torch.exp2(scales.view(torch.uint8).double() - 127)
    s = torch.where(scales.view(torch.uint8) == 255, math.nan, s)
    return (codes.double().unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)


def decode(codes, fmt):
    """float64 values of packed codes (..., bytes)."""
    bits, (ebits, mbits, bias) = BITS[fmt], SHAPE[fmt]
    if bits == 4:
        n = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).int()
    else:
        b = codes.unflatten(-1, (-1, 3)).int()
        word = b[..., 0] | (b[..., 1] << 8) | (b[..., 2] << 16)
        n = torch.stack([(word >> (6 * i)) & 63 for i in range(4)], -1).flatten(-2)
    e, f = (n >> mbits) & (2 ** ebits - 1), (n & (2 ** mbits - 1)).double() / 2 ** mbits
    v = torch.where(e > 0, (1 + f) * torch.exp2(e.double() - bias), f * 2.0 ** (1 - bias))
    return torch.where((n >> (bits - 1)) > 0, -v, v)


def weights(w):
    """float64 values of a PackedTensor with E8M0 scales."""
    rows = math.prod(w.shape[:-1])
    raw = w.data[: rows * w.shape[-1] * BITS[w.format] // 8]
    v = decode(raw.view(*w.shape[:-1], -1), w.format)
    b = w.scales.view(torch.uint8)
    s = torch.where(b == 255, math.nan, torch.exp2(b.double() - 127))
    return (v.unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)


def make_weights(shape, fmt, g, device="cuda", low=-6, high=-2):
    import tinygrad_dx12_b200 as tg

    data = torch.randint(0, 256, (math.prod(shape) * BITS[fmt] // 8,), dtype=torch.uint8, device=device, generator=g)
    e = torch.randint(low, high + 1, (*shape[:-1], shape[-1] // 32), device=device, generator=g)
    return tg.PackedTensor(data, fmt, shape, (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu), 32)


def activate(v, name):
    if name == "relu":
        return v.clamp(min=0)
    if name == "silu":
        return v * torch.sigmoid(v)
    if name == "gelu":
        return v * torch.special.ndtr(v)
    if name == "gelu_tanh":
        return v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))
    return v


# No activation here is steeper than this: gelu's slope is at most 1.13, its tanh form's too, silu's 1.10.
SLOPE = 1.14


def product(x, w, bias=None, activation=None, gated=False, residual=None):
    """(result, how far fp32 sums may be from it), both float64: x (rows, K), w (N, K).

    The products of codes and powers of two are exact. A tensor-core instruction adds 32 of them to the
    accumulator; whatever the order and rounding inside, its error is below 2^-21 of the magnitudes that go in,
    at most sum|x||w|: (K / 32 + 16) 2^-21 of that over all of them, 16 for joined parts. The activation's
    functions, the gate's product and the additions round to fp32: 2^-20 of each one's magnitude."""
    v, size = x @ w.T, x.abs() @ w.abs().T
    tol = (x.shape[-1] / 32 + 16) * 2.0 ** -21 * size
    if bias is not None:
        v = v + bias.double()
        tol = tol + 2.0 ** -20 * v.abs()
    if gated:
        (g, u), (tg_, tu) = v.chunk(2, -1), tol.chunk(2, -1)
        a = activate(g, activation)
        ta = SLOPE * tg_ + 2.0 ** -20 * g.abs()
        v, tol = a * u, ta * (u.abs() + tu) + a.abs() * tu + 2.0 ** -20 * (a * u).abs()
    elif activation is not None:
        v, tol = activate(v, activation), SLOPE * tol + 2.0 ** -20 * v.abs()
    if residual is not None:
        v = v + residual.double()
        tol = tol + 2.0 ** -20 * v.abs()
    return v, tol


def half_step(v, dtype):
    """Half a step of the type at v: a rounding's largest error (fp16's subnormals have 2^-25)."""
    tiny = {torch.float16: 2.0 ** -25}.get(dtype, 0.0)
    return v.abs() * torch.finfo(dtype).eps / 2 + tiny


def check(y, v, tol):
    """y (a tensor) within tol and its type's rounding of v, everywhere."""
    d = (y.double() - v).abs()
    bound = half_step(v, y.dtype) * (1 + 2.0 ** -6) + tol
    bad = ~(d <= bound)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}: {d[bad].max():.3e} over {bound[bad].min():.3e}"


def check8(y, v, tol):
    """Block-scaled y within tol and E4M3's rounding of v, and no scale larger or smaller than it may be."""
    got = values(y.codes, y.scales)
    s = torch.exp2(y.scales.view(torch.uint8).double() - 127)
    top = (v.abs() + tol).unflatten(-1, (-1, 32)).amax(-1)
    least = (v.abs() - tol).unflatten(-1, (-1, 32)).amax(-1)
    assert bool((s >= (least / QMAX) * (1 - 2.0 ** -22)).all()), "a scale clips its block"
    assert bool(((s <= 2 * top / QMAX * (1 + 2.0 ** -22)) | (s <= 2.0 ** -100)).all()), "a scale is larger than its block needs"
    # half a step: 2^-4 of a normal value, 2^-10 scales below 2^-6 of them
    bound = torch.maximum(v.abs() * 2.0 ** -4, (s * 2.0 ** -10).repeat_interleave(32, -1)) + 1.07 * tol
    d = (got - v).abs()
    bad = ~(d <= bound)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}: {d[bad].max():.3e} over {bound[bad].min():.3e}"


def generator(seed, device="cuda"):
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    return g
