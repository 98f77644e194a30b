"""Attention over keys whose values are zero: padded tokens, rows of zeros under ordinary keys, and
cells that were never written. They have weight without a value, so results shrink and logarithms
grow by what the formula says. A block of zeros is stored with the scale 2^-100, an unwritten cell
has the scale 0: the denominator, which divides weights by their row's scale, has to bear any number
of either. Tolerances: tests/cache_helpers.py."""

from __future__ import annotations

import math

import pytest
import torch

import tinygrad_dx12_b200 as tg
from tests import cache_helpers as ref
from tests.test_gpu_cache import Case, randn

pytestmark = pytest.mark.gpu

FORMATS = ["int8", "fp8e4m3", "int4", "fp4_e2m1"]
QUERIES = {"few": 1, "many": 20, "two tiles": 75}  # of four heads to a key head: 4, 80 and 300 query rows


def hide(c, slots, kind):
    """Give the cells ``slots`` values of zero: as padding (keys of zero too), under small keys, or unwritten."""
    n, (kv, dim) = len(slots), c.k.shape[1:]
    if kind == "unwritten":
        page, at = slots // c.page, slots % c.page
        for t in (c.cache.k, c.cache.v, c.cache.k_scales.view(torch.uint8), c.cache.v_scales.view(torch.uint8)):
            t[page.cuda(), :, at.cuda()] = 0
    else:
        k = randn((n, kv, dim), 300) * (0.05 if kind == "values" else 0.0)
        tg.cache_write(c.cache, k.cuda(), torch.zeros(n, kv, dim, device="cuda"), slots.cuda())
    k, v = tg.cache_read(c.cache, torch.arange(c.cache.pages * c.page, device="cuda"), dtype=torch.float32)
    c.k, c.v = k.cpu().double(), v.cpu().double()
    assert (c.v[slots] == 0).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("blocked,e8", [(False, False), (True, False), (True, True)])
@pytest.mark.parametrize("rows", list(QUERIES))
@pytest.mark.parametrize("n,kind,before,behind", [(32, "padding", 0, 40), (128, "unwritten", 0, 100), (128, "values", 70, 75),
                                                  (1, "unwritten", 100, 0), (4096, "padding", 0, 90), (4096, "values", 100, 10),
                                                  (4096, "unwritten", 0, 0), (160, "padding", 0, 0)])
def test_zero_values(fmt, blocked, e8, rows, n, kind, before, behind):
    queries = QUERIES[rows]
    c = Case([before + n + behind, 9], queries=queries, heads=4, kv=1, fmt=fmt, blocked=blocked, e8=e8, page=64, seed=301)
    hide(c, c.own[0][before:before + n], kind)
    c.check()
    if before + behind == 0:  # nothing but zero values: zeros, and the logarithm of the number of equal scores
        out, lse = c.run()
        assert (out[0] == 0).all()
        ends = torch.tensor([float(max(0, n - queries + i + 1)) for i in range(queries)], dtype=torch.float64)
        assert ((lse[0].cpu().double() - ends.log()[:, None]).abs()[ends > 0] <= 2.0 ** -16).all()


@pytest.mark.parametrize("fmt,blocked", [("int8", False), ("int4", False), ("fp4_e2m1", True)])
@pytest.mark.parametrize("dim,heads,kv", [(64, 8, 2), (256, 8, 1), (128, 16, 1)])
def test_zero_values_dims(fmt, blocked, dim, heads, kv):
    c = Case([2000, 300, 40], heads=heads, kv=kv, dim=dim, fmt=fmt, blocked=blocked, page=32, dtype=torch.float16, seed=302)
    hide(c, torch.cat([c.own[0][:1500], c.own[1][100:], c.own[2]]), "padding")
    c.check()


@pytest.mark.parametrize("fmt,blocked", [("int8", False), ("fp8e4m3", True), ("int4", False), ("fp4_e2m1", True)])
@pytest.mark.parametrize("batch", [3, 40])  # 12 and 160 query rows over the prefix
@pytest.mark.parametrize("where", ["prefix", "own", "half the prefix", "both"])
def test_zero_values_behind_a_prefix(fmt, blocked, batch, where):
    lengths = [(37 * i) % 150 for i in range(batch)]
    c = Case(lengths, heads=4, kv=1, fmt=fmt, blocked=blocked, prefix=700, page=16, seed=303)
    cells = {"prefix": c.shared, "half the prefix": c.shared[:350], "own": torch.cat(c.own),
             "both": torch.cat([c.shared, *c.own])}[where]
    hide(c, cells, "padding")
    c.check()


@pytest.mark.parametrize("fmt,blocked", [("int8", False), ("int4", True)])
@pytest.mark.parametrize("queries", [1, 40])
@pytest.mark.parametrize("size", [2.0 ** -60, 2.0 ** 20])
def test_zero_values_beside_small_and_large_ones(fmt, blocked, queries, size):
    """Values far from one: the results follow them, whatever the denominator's own scale."""
    c = Case([600], queries=queries, heads=4, kv=1, fmt=fmt, blocked=blocked, page=32, seed=304)
    v = randn((600, 1, 128), 305) * size
    v[200:400] = 0
    tg.cache_write(c.cache, randn((600, 1, 128), 306).cuda(), v.cuda(), c.own[0].cuda())
    k, v = tg.cache_read(c.cache, torch.arange(c.cache.pages * 32, device="cuda"), dtype=torch.float32)
    c.k, c.v = k.cpu().double(), v.cpu().double()
    out, lse = c.run()
    ends = [600 - queries + i + 1 for i in range(queries)]
    r, rl, spread = ref.attend(c.q[0].double(), c.k[c.own[0]], c.v[c.own[0]], c.scale, ends)
    # the helper's absolute term is a subnormal fp16's: here bf16 follows the size of the values
    tol = ref.tolerance(r, spread, torch.bfloat16, 128, blocked) - 2.0 ** -24
    assert ((out[0].cpu().double() - r).abs() <= tol).all()
    assert ((lse[0].cpu().double() - rl).abs() <= 2.0 ** -9).all() and math.isfinite(lse.sum().item())


@pytest.mark.parametrize("fmt,blocked", [("int8", False), ("fp4_e2m1", True)])
@pytest.mark.parametrize("rows", ["few", "many"])
@pytest.mark.parametrize("zero", [False, True])
def test_two_million_keys(fmt, blocked, rows, zero):
    """One page named 2^15 times: the result of the page alone, its logarithm larger by that of 2^15."""
    page, times = 64, 1 << 15
    cache = tg.PackedCache.empty(2, page, 1, 128, fmt, block_size=32 if blocked else 128)
    k, v = randn((page, 1, 128), 310).cuda(), randn((page, 1, 128), 311).cuda() * (0.0 if zero else 1.0)
    tg.cache_write(cache, k, v, torch.arange(page, 2 * page).cuda())
    batch = 2 if rows == "few" else 40
    q = randn((batch, 4, 128), 312, torch.bfloat16).cuda()
    one = torch.ones((batch, times), dtype=torch.int32, device="cuda")
    none = torch.zeros(batch, dtype=torch.int32, device="cuda")

    def attend(n):
        if rows == "few":
            return tg.cache_attention(q, cache, one, none + n, return_lse=True)
        return tg.cache_attention(q, cache, one, none, prefix=one[0], prefix_length=n, return_lse=True)

    (a, la), (b, lb) = attend(page), attend(page * times)
    # both round once to bfloat16 (2^-8); sums of up to 2^14 terms a lane in fp32 (2^-24 each)
    assert ((a.double() - b.double()).abs() <= 2.0 ** -7 * a.double().abs() + 2.0 ** -9 * a.double().abs().max()).all()
    assert ((lb.double() - la.double() - math.log(times)).abs() <= 2.0 ** -9).all()
    assert not zero or (b == 0).all()
