"""Plain restatements for the cached-attention tests: rotary positions, quantisation, reading back and
attention, from their formulas. Values and sums in float64 on the CPU; the quantisation's own
operations in float32, where each is one IEEE rounding and codes have to agree to the bit."""

from __future__ import annotations

import math

import torch

QMAX = {"int8": 127.0, "fp8e4m3": 448.0, "int4": 7.0, "fp4_e2m1": 6.0}
FP4 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def turn(x, cos, sin, positions, layout, transpose=False):
    """x (..., tokens, heads, dim) with pairs turned; in x's precision (pass float64 or float32)."""
    c, s = cos[positions].to(x.dtype).unsqueeze(-2), sin[positions].to(x.dtype).unsqueeze(-2)
    if transpose:
        s = -s
    n = cos.shape[1]
    y = x.clone()
    first, second = (slice(0, n), slice(n, 2 * n)) if layout == "half" else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    a, b = x[..., first], x[..., second]
    y[..., first] = a * c - b * s
    y[..., second] = b * c + a * s
    return y


def quantise(x, fmt, block, e8m0):
    """(values of the codes (..., dim), scales (..., dim / block)) of float32 x; float32 throughout."""
    x = x.float().unflatten(-1, (-1, block))
    r = x.abs().amax(-1) * torch.tensor(1.0 / QMAX[fmt], dtype=torch.float32)
    if e8m0:
        e = ((r.view(torch.int32) + 0x7FFFFF) >> 23).clamp(27, 227)
        s = (e << 23).view(torch.float32)
        s = torch.where(r.isnan(), r, s)
    else:
        s = r.to(torch.bfloat16).float().clamp(2.0 ** -100, 2.0 ** 100)
    y = x * (1.0 / s)[..., None]
    q = QMAX[fmt]
    if fmt.startswith("int"):
        y = y.round().clamp(-q, q)
    elif fmt == "fp8e4m3":
        y = y.clamp(-q, q).to(torch.float8_e4m3fn).float()
    else:
        m = y.abs()
        step = torch.where(m < 2, 0.5, torch.where(m < 4, 1.0, 2.0))
        y = ((m / step).round() * step).clamp(max=q).copysign(y)
    return y.flatten(-2), s


def read_back(codes, scales, block):
    """float32 values of codes and scales: one product each."""
    return (codes.unflatten(-1, (-1, block)) * scales[..., None]).flatten(-2)


def attend(q, k, v, scale, queries_end=None):
    """Rows q (n, heads, dim) over k, v (keys, kv_heads, dim), float64; row i sees ``queries_end[i]``
    keys (None: all). Returns (out, lse, spread): spread bounds what rounding of weights and scores
    to fp16 products and fp32 sums may move (see ``tolerance``)."""
    n, heads, dim = q.shape
    group = heads // k.shape[1]
    kk, vv = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    s = torch.einsum("nhd,thd->hnt", q, kk) * scale
    size = torch.einsum("nhd,thd->hnt", q.abs(), kk.abs()) * abs(scale)
    if queries_end is not None:
        hidden = torch.arange(k.shape[0])[None, :] >= torch.as_tensor(queries_end)[:, None]
        s = s.masked_fill(hidden[None], -math.inf)
        size = size.masked_fill(hidden[None], 0.0)
    lse = torch.logsumexp(s, -1) if k.shape[0] else torch.full((heads, n), -math.inf, dtype=q.dtype)
    w = torch.nan_to_num(torch.exp(s - torch.where(lse == -math.inf, 0.0, lse)[..., None]), nan=0.0)
    out = torch.einsum("hnt,thd->nhd", w, vv)
    mag = torch.einsum("hnt,thd->nhd", w, vv.abs())
    top = size.amax(-1) if k.shape[0] else torch.zeros((heads, n), dtype=q.dtype)
    return out, lse.transpose(0, 1), (mag, top.transpose(0, 1))


def tolerance(out, spread, dtype, dim, blocked=False):
    """How far a result may be from ``attend``'s, element by element.

    * rounding to the output type: half a unit in the last place, 2^-11 (fp16) or 2^-8 (bf16) of |out|
      (fp16 also 2^-25 for subnormals);
    * weights are rounded to fp16 (2^-11 relative each, 2^-25 absolute below 2^-14) and, in block-scaled
      caches, codes times scales too (2^-11): 2^-10 of the weighted mean of |v|;
    * scores: products are exact, sums over dim terms in fp32 on the tensor core (not round-to-nearest:
      2^-22 of the sum of magnitudes a term), scales and the exponential 2^-20: a score moves by
      e = (dim * 2^-22 + 2^-18) * sum|q||k|, its weight by that share, numerator and denominator both;
    * block-scaled keys: code times scale rounded to fp16, 2^-11 a term, taken at its worst: 2^-11 of
      sum|q||k| on top."""
    mag, size = spread
    e = size * (dim * 2.0 ** -22 + 2.0 ** -18 + (2.0 ** -11 if blocked else 0.0)) + 2.0 ** -18
    unit = 2.0 ** -11 if dtype == torch.float16 else 2.0 ** -8
    return out.abs() * unit + 2.0 ** -24 + mag * (2.0 ** -10 + 2 * e[..., None])
