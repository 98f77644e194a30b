"""Rotary positions, the packed key/value cache and attention over it on the GPU, against plain
restatements (tests/cache_helpers.py): every format, head size and scale type, lengths from none to
many pages, shapes and strides off the fast paths, masks that leave nothing, NaN and infinities where
they are and are not looked at, and the refusals."""

from __future__ import annotations

import math

import pytest
import torch

import tinygrad_dx12_b200 as tg
from tests import cache_helpers as ref
from tinygrad_dx12_b200 import _lib

pytestmark = pytest.mark.gpu

FORMATS = ["int8", "fp8e4m3", "int4", "fp4_e2m1"]
E8 = torch.float8_e8m0fnu
BF = torch.bfloat16


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(shape, seed, dtype=torch.float32):
    return torch.randn(shape, generator=gen(seed)).to(dtype)


def status(clear=True):
    import ctypes

    v = ctypes.c_uint32()
    torch.cuda.synchronize()
    _lib.call("b200_device_status", torch.cuda.current_device(), ctypes.byref(v), int(clear))
    return v.value


@pytest.fixture(autouse=True)
def clean_status():
    status()
    yield
    status()


# ---- rotary ---------------------------------------------------------------------------------------
def tables(rot, rows, seed=0):
    t = tg.RotaryTable.build(rot, rows)
    return t.cos.cpu(), t.sin.cpu()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [torch.float16, BF, torch.float32])
@pytest.mark.parametrize("tokens,heads,dim,rot", [(1, 1, 64, 64), (1, 32, 128, 128), (7, 5, 128, 64), (33, 3, 80, 80),
                                                  (9, 2, 96, 20), (5, 4, 64, 2), (700, 24, 128, 128), (3, 1, 256, 256)])
def test_rotary(layout, dtype, tokens, heads, dim, rot):
    table = tg.RotaryTable.build(rot, 5000, layout=layout)
    x = randn((tokens, heads, dim), 1, dtype)
    pos = torch.randint(0, 5000, (tokens,), generator=gen(2))
    r = ref.turn(x.double(), table.cos.cpu(), table.sin.cpu(), pos, layout)
    y = tg.rotary(x.cuda(), table, pos.cuda())
    # two fp32 products and a sum (2^-23 of |a| + |b| <= 2 * max), then one rounding to the type
    unit = {torch.float16: 2.0 ** -11, BF: 2.0 ** -8, torch.float32: 2.0 ** -24}[dtype]
    tol = unit * r.abs() + 2.0 ** -22 * x.double().abs().max() + 2.0 ** -25
    assert ((y.cpu().double() - r).abs() <= tol).all()
    assert torch.equal(y.cpu()[..., rot:], x[..., rot:])
    if dtype == torch.float32:  # the formula's own roundings: the same bits as fp32 products and sums
        assert torch.equal(y.cpu(), ref.turn(x, table.cos.cpu(), table.sin.cpu(), pos, layout))
    back = tg.rotary(x.cuda(), table, pos.to(torch.int32).cuda(), transpose=True)
    rb = ref.turn(x.double(), table.cos.cpu(), table.sin.cpu(), pos, layout, transpose=True)
    assert ((back.cpu().double() - rb).abs() <= unit * rb.abs() + 2.0 ** -22 * x.double().abs().max() + 2.0 ** -25).all()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("view", ["heads_first", "every_other_head", "misaligned", "in_place", "transposed_dim", "rows_of_one"])
def test_rotary_strides(layout, view):
    table = tg.RotaryTable.build(64, 100, layout=layout)
    pos = torch.randint(0, 100, (2, 9), generator=gen(3))
    base = randn((2, 9, 6, 130), 4, BF).cuda()
    if view == "heads_first":
        x = randn((2, 6, 9, 128), 4, BF).cuda().transpose(1, 2)
    elif view == "every_other_head":
        x = base[:, :, ::2, :128]
    elif view == "misaligned":
        x = base[..., 1:129]
    elif view == "transposed_dim":
        x = randn((2, 9, 128, 6), 4, BF).cuda().transpose(2, 3)
    elif view == "rows_of_one":
        x, pos = base[:, :1, :, :128], pos[:, :1]
    else:
        x = base[..., :128].contiguous()
    r = ref.turn(x.cpu().float(), table.cos.cpu(), table.sin.cpu(), pos, layout).to(BF)
    y = tg.rotary(x, table, pos.cuda(), out=x if view == "in_place" else None)
    assert torch.equal(y.cpu(), r)
    if view == "in_place":
        assert y is x


def test_rotary_gradient():
    """Against the formula (the transposed map) and against differences; broadcast input."""
    table = tg.RotaryTable.build(32, 50, layout="interleaved", scaling="by_parts", factor=4.0)
    pos = torch.arange(6).cuda() * 7
    x = randn((6, 1, 64), 5).cuda().requires_grad_()
    dy = randn((6, 3, 64), 6).cuda()
    y = tg.rotary(x.expand(6, 3, 64), table, pos)
    (gx,) = torch.autograd.grad(y, x, dy)
    r = ref.turn(dy.cpu().double(), table.cos.cpu(), table.sin.cpu(), pos.cpu(), "interleaved", True).sum(1, keepdim=True)
    assert ((gx.cpu().double() - r).abs() <= 2.0 ** -21 * dy.abs().max().item() * 3).all()
    # the map is linear: a central difference of step 1 is exact up to rounding
    for i in (0, 17, 40):
        e = torch.zeros(6, 1, 64, device="cuda")
        e[2, 0, i] = 1.0
        with torch.no_grad():
            d = (tg.rotary((x + e).expand(6, 3, 64), table, pos) - tg.rotary((x - e).expand(6, 3, 64), table, pos)) / 2
        num = (d.double() * dy.double()).sum().item()
        assert abs(num - gx[2, 0, i].item()) <= 2.0 ** -18 * dy.abs().sum().item()
    # twice differentiable: the gradient of the gradient is the map itself
    v = torch.ones_like(dy, requires_grad=True)
    (g1,) = torch.autograd.grad(tg.rotary(x.expand(6, 3, 64), table, pos), x, v, create_graph=True)
    (g2,) = torch.autograd.grad(g1, v, torch.ones_like(g1))
    assert torch.equal(g2, tg.rotary(torch.ones(6, 3, 64, device="cuda"), table, pos))


def test_rotary_outside_and_empty():
    table = tg.RotaryTable.build(64, 10)
    x = randn((4, 2, 128), 7, BF).cuda()
    y = tg.rotary(x, table, torch.tensor([0, 10, -1, 9]).cuda())
    assert status() == 2
    assert y[1:3, :, :64].isnan().all() and not y[0].isnan().any() and not y[3].isnan().any()
    assert torch.equal(y[..., 64:], x[..., 64:])
    assert tg.rotary(x[:0], table, torch.zeros(0, dtype=torch.int64).cuda()).shape == (0, 2, 128)


def test_rotary_tables():
    """The stretched forms against their formulas in plain Python."""
    rot, rows, base, f = 64, 4096, 10000.0, 8.0
    freq = [base ** (-2 * i / rot) for i in range(rot // 2)]
    for scaling in (None, "linear", "base", "by_parts"):
        t = tg.RotaryTable.build(rot, rows, base, scaling=scaling, factor=f, original=512)
        gain, want = 1.0, list(freq)
        if scaling == "linear":
            want = [w / f for w in freq]
        elif scaling == "base":
            want = [(base * f ** (rot / (rot - 2))) ** (-2 * i / rot) for i in range(rot // 2)]
        elif scaling == "by_parts":
            at = lambda turns: rot * math.log(512 / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
            lo, hi = math.floor(at(32)), math.ceil(at(1))
            want = [w * (1 - min(max((i - lo) / (hi - lo), 0), 1)) + w / f * min(max((i - lo) / (hi - lo), 0), 1)
                    for i, w in enumerate(freq)]
            gain = 0.1 * math.log(f) + 1
        for p in (0, 1, 777, rows - 1):
            for i in (0, 5, 13, 31):
                # a float64 angle of up to 4096 (2^-41) and one rounding to fp32
                assert abs(t.cos[p, i].item() - gain * math.cos(p * want[i])) <= 2.0 ** -23
                assert abs(t.sin[p, i].item() - gain * math.sin(p * want[i])) <= 2.0 ** -23


# ---- writing and reading ----------------------------------------------------------------------------
def make_cache(fmt="int8", dim=128, block=None, e8=False, pages=6, page=16, heads=2, order="heads"):
    return tg.PackedCache.empty(pages, page, heads, dim, fmt, block_size=block, scale_dtype=E8 if e8 else BF, order=order)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("blocked,e8", [(False, False), (False, True), (True, False), (True, True)])
@pytest.mark.parametrize("dtype", [torch.float16, BF, torch.float32])
def test_cache_round_trip(fmt, dim, blocked, e8, dtype):
    """Codes agree to the bit with the formula; the turned queries with rotary()."""
    block = 32 if blocked else dim
    layout, order = ("half", "heads") if blocked else ("interleaved", "tokens")
    table = tg.RotaryTable.build(dim // 2, 500, layout=layout)
    cache = make_cache(fmt, dim, block, e8, order=order)
    n, heads, kv = 37, 6, 2
    rows = randn((n, heads + 2 * kv, dim), 11)
    rows[:, :, 3] *= 20.0
    rows[5, :, :] *= 1e-6
    rows[6] = 0.0
    rows = rows.to(dtype).cuda()
    q, k, v = rows[:, :heads], rows[:, heads:heads + kv], rows[:, heads + kv:]
    slots = torch.randperm(6 * 16, generator=gen(12))[:n]
    pos = torch.randint(0, 500, (n,), generator=gen(13))
    qt = tg.cache_write(cache, k, v, slots.cuda(), table, pos.cuda(), q=q)
    cos, sin = table.cos.cpu(), table.sin.cpu()
    assert torch.equal(qt, tg.rotary(q, table, pos.cuda()))
    for i, x in enumerate((ref.turn(k.cpu().float(), cos, sin, pos, layout), v.cpu().float())):
        codes, scales = ref.quantise(x, fmt, block, e8)
        want = ref.read_back(codes, scales, block)
        for out in (torch.float32, dtype):
            got = tg.cache_read(cache, slots.to(torch.int32).cuda(), dtype=out)[i]
            assert torch.equal(got.cpu(), want.to(out)), (i, out)
    unused = torch.tensor([s for s in range(96) if s not in set(slots.tolist())])
    assert all((t == 0).all() for t in tg.cache_read(cache, unused.cuda()))
    assert status() == 0


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("e8", [False, True])
def test_cache_extremes(fmt, e8):
    """NaN poisons its block, infinities and huge values are held at the largest, tiny ones vanish."""
    cache = make_cache(fmt, 64, 32, e8, heads=1)
    x = randn((6, 1, 64), 14)
    x[0, 0, 3] = math.nan
    x[1, 0, 40] = math.inf
    x[2, 0, 5] = -math.inf
    x[3] = 3e38
    x[4] = 1e-38
    v = x.clone()
    slots = torch.arange(6)
    tg.cache_write(cache, x.cuda(), v.cuda(), slots.cuda())
    k, got = tg.cache_read(cache, slots.cuda(), dtype=torch.float32)
    codes, scales = ref.quantise(x, fmt, 32, e8)
    want = ref.read_back(codes, scales, 32)
    k = k.cpu()
    assert k[0, 0, :32].isnan().all() and torch.equal(k[0, 0, 32:], want[0, 0, 32:])
    assert torch.equal(k[1:], want[1:]) and torch.equal(got.cpu()[1:], want[1:])
    assert k[1, 0, 40].item() == ref.QMAX[fmt] * 2.0 ** 100 and (k[4] == 0).all()


def test_cache_slots():
    """Negative slots store and read nothing; those beyond the cache too, and are reported."""
    cache = make_cache("int8", 64, heads=1)
    x = randn((4, 1, 64), 15, BF).cuda()
    tg.cache_write(cache, x, x, torch.tensor([-1, 3, 96, 95]).cuda())
    assert status() == 2
    k, _ = tg.cache_read(cache, torch.tensor([0, 3, 95]).cuda())
    assert (k[0] == 0).all() and (k[1] != 0).any() and (k[2] != 0).any()
    assert status() == 0
    k, v = tg.cache_read(cache, torch.tensor([-5, 96, 3]).cuda())
    assert status() == 2 and (k[:2] == 0).all() and (v[:2] == 0).all() and (k[2] != 0).any()
    tg.cache_write(cache, x[:0], x[:0], torch.zeros(0, dtype=torch.int32).cuda())
    assert tg.cache_read(cache, torch.zeros(0, dtype=torch.int32).cuda())[0].shape == (0, 1, 64)


def test_cache_many_tokens():
    """More tokens than the few-token launch, odd rotary size, misaligned rows."""
    table = tg.RotaryTable.build(20, 3000)
    cache = make_cache("fp4_e2m1", 64, 32, True, pages=100, page=32, heads=3)
    n = 2999
    rows = randn((n, 3 * 5 * 64 + 1), 16, torch.float16).cuda()[:, 1:].view(n, 15, 64)
    q, k, v = rows[:, :9], rows[:, 9:12], rows[:, 12:]
    slots, pos = torch.randperm(3200, generator=gen(17))[:n], torch.randint(0, 3000, (n,), generator=gen(18))
    qt = tg.cache_write(cache, k, v, slots.cuda(), table, pos.cuda(), q=q)
    assert torch.equal(qt, tg.rotary(q, table, pos.cuda()))
    got = tg.cache_read(cache, slots.cuda(), dtype=torch.float32)
    for x, y in zip((ref.turn(k.cpu().float(), table.cos.cpu(), table.sin.cpu(), pos, "half"), v.cpu().float()), got):
        assert torch.equal(y.cpu(), ref.read_back(*ref.quantise(x, "fp4_e2m1", 32, True), 32))


# ---- attention --------------------------------------------------------------------------------------
class Case:
    """A filled cache with shuffled pages, and the plain result."""

    def __init__(self, lengths, queries=1, heads=8, kv=2, dim=128, fmt="int8", blocked=False, e8=False, page=16,
                 dtype=BF, prefix=0, order="heads", seed=0, poison=True, q_gain=1.0, spread=1.0, per=None):
        block = 32 if blocked else dim
        per = per if per is not None else max(1, -(-max(lengths, default=1) // page)) + 1
        first = -(-prefix // page)
        pages = len(lengths) * per + first + 1
        self.cache = tg.PackedCache.empty(pages, page, kv, dim, fmt, block_size=block, scale_dtype=E8 if e8 else BF, order=order)
        n = pages * page
        k, v = randn((n, kv, dim), seed + 1), randn((n, kv, dim), seed + 2)
        k[..., 1] *= 6.0
        v *= torch.exp2(torch.randn((n, 1, 1), generator=gen(seed + 3)) * spread)
        self.perm = torch.randperm(pages, generator=gen(seed + 4))
        self.tables = self.perm[first:first + len(lengths) * per].view(len(lengths), per)
        self.prefix = self.perm[:first]
        self.lengths, self.queries, self.page, self.n_prefix = lengths, queries, page, prefix
        slots = torch.arange(n)
        self.own = [self._slots(self.tables[b], min(x, per * page)) for b, x in enumerate(lengths)]
        self.shared = self._slots(self.prefix, prefix)
        if poison:  # what no request holds is NaN
            held = torch.cat([self.shared, *self.own])
            free = torch.ones(n, dtype=torch.bool)
            free[held] = False
            k[free], v[free] = math.nan, math.nan
        tg.cache_write(self.cache, k.cuda(), v.cuda(), slots.cuda())
        kk, vv = tg.cache_read(self.cache, slots.cuda(), dtype=torch.float32)
        self.k, self.v = kk.cpu().double(), vv.cpu().double()
        self.q = (randn((len(lengths), queries, heads, dim), seed + 5) * q_gain).to(dtype)
        self.scale = 1.0 / math.sqrt(dim)
        self.dim, self.dtype, self.blocked = dim, dtype, blocked

    def _slots(self, pages, n):
        i = torch.arange(n)
        return pages[i // self.page] * self.page + i % self.page

    def run(self, **kw):
        shared = dict(prefix=self.prefix.to(torch.int32).cuda(), prefix_length=self.n_prefix) if self.n_prefix else {}
        return tg.cache_attention(self.q.cuda(), self.cache, self.tables.to(torch.int32).cuda(),
                                  torch.tensor(self.lengths, dtype=torch.int32).cuda(), return_lse=True, **shared, **kw)

    def check(self, out=None, lse=None, scale=None):
        if out is None:
            out, lse = self.run() if scale is None else self.run(scale=scale)
        out, lse = out.cpu().double(), lse.cpu().double()
        for b, s in enumerate(self.own):
            at = torch.cat([self.shared, s])
            ends = [len(self.shared) + max(0, len(s) - self.queries + i + 1) for i in range(self.queries)]
            r, rl, spread = ref.attend(self.q[b].double(), self.k[at], self.v[at], self.scale if scale is None else scale, ends)
            tol = ref.tolerance(r, spread, self.dtype, self.dim, self.blocked)
            bad = (out[b] - r).abs() > tol
            assert not bad.any() and not out[b].isnan().any(), (b, ((out[b] - r).abs() / tol).max().item())
            assert torch.equal(lse[b] == -math.inf, rl == -math.inf)
            fine = rl != -math.inf
            ltol = spread[1] * (self.dim * 2.0 ** -22 + 2.0 ** -18 + (2.0 ** -11 if self.blocked else 0)) + 2.0 ** -16
            assert ((lse[b] - rl).abs()[fine] <= ltol[fine]).all(), (lse[b] - rl).abs()[fine].max()
            assert (out[b][~fine] == 0).all()
        assert status() == 0


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("blocked,e8", [(False, False), (False, True), (True, False), (True, True)])
@pytest.mark.parametrize("heads,kv,dtype", [(4, 2, torch.float16), (24, 2, BF)])
def test_attention_formats(fmt, dim, blocked, e8, heads, kv, dtype):
    Case([1, 0, 16, 17, 95, 200], heads=heads, kv=kv, dim=dim, fmt=fmt, blocked=blocked, e8=e8, dtype=dtype,
         order="tokens" if e8 else "heads").check()


@pytest.mark.parametrize("heads,kv", [(1, 1), (5, 1), (8, 8), (7, 7), (16, 1), (33, 3), (40, 1), (64, 8)])
@pytest.mark.parametrize("page", [16, 64])
def test_attention_groups(heads, kv, page):
    Case([3, 130, 31], heads=heads, kv=kv, page=page, fmt="int4", dtype=torch.float16, seed=20).check()


@pytest.mark.parametrize("queries", [2, 3, 5, 17, 64, 150])
@pytest.mark.parametrize("heads,kv,dim,blocked", [(8, 2, 128, False), (3, 3, 64, True), (4, 1, 256, False)])
def test_attention_queries(queries, heads, kv, dim, blocked):
    """Causal from the end; requests shorter than their queries leave rows without a key."""
    Case([queries, queries + 100, max(0, queries - 2), 0, 1], queries=queries, heads=heads, kv=kv, dim=dim, fmt="fp8e4m3",
         blocked=blocked, seed=30).check()


@pytest.mark.parametrize("prefix", [1, 16, 37, 700, 3000])
@pytest.mark.parametrize("queries,heads,kv,dim,fmt,blocked", [(1, 8, 2, 128, "int4", False), (1, 16, 1, 64, "fp4_e2m1", True),
                                                               (3, 6, 2, 128, "int8", False), (1, 8, 1, 256, "fp8e4m3", True)])
def test_attention_prefix(prefix, queries, heads, kv, dim, fmt, blocked):
    Case([5, 0, 77, queries], queries=queries, heads=heads, kv=kv, dim=dim, fmt=fmt, blocked=blocked, prefix=prefix,
         seed=40).check()


@pytest.mark.parametrize("batch", [1, 40, 150])
def test_attention_prefix_batches(batch):
    lengths = torch.randint(0, 90, (batch,), generator=gen(50)).tolist()
    Case(lengths, heads=8, kv=2, fmt="int8", prefix=260, page=32, seed=51).check()


def test_attention_long_and_ragged():
    """One request cut over many CTAs beside short ones; twice the same bits."""
    c = Case([20000, 1, 0, 333, 4097], heads=8, kv=2, fmt="int8", page=64, seed=60)
    a, b = c.run(), c.run()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    c.check(*a)


def test_attention_many_requests():
    lengths = torch.randint(0, 40, (5000,), generator=gen(61)).tolist()
    Case(lengths, heads=2, kv=1, dim=64, fmt="int4", seed=62).check()


@pytest.mark.parametrize("fmt,blocked", [("int8", False), ("fp4_e2m1", True)])
def test_attention_value_ranges(fmt, blocked):
    """Values whose scales span 2^40 from key to key, and scores far apart."""
    Case([300, 40], heads=8, kv=2, fmt=fmt, blocked=blocked, e8=True, spread=10.0, q_gain=8.0, seed=70).check()


def test_attention_scale_and_large_queries():
    c = Case([100, 7], heads=4, kv=2, q_gain=1e5, seed=71)
    c.check(scale=1e-5 / math.sqrt(128))
    Case([100, 7], heads=4, kv=2, q_gain=1e-4, dtype=torch.float16, seed=72).check()
    c = Case([50], heads=4, kv=2, seed=73)
    c.check(scale=0.0)
    c.check(scale=-0.3)


def test_attention_nan_and_inf_where_seen():
    """A NaN key spoils the rows that see it and no others; so does an infinite query."""
    c = Case([40, 40], queries=4, heads=4, kv=2, seed=74)
    x = randn((1, 2, 128), 75).cuda()
    x[0, 0, 5] = math.nan
    tg.cache_write(c.cache, x, x, c.own[0][38:39].cuda())  # request 0: key 38, seen by queries 2 and 3
    out, lse = c.run()
    o = out.cpu()
    assert o[0, 2:, :2].isnan().all() and not o[0, :2].isnan().any() and not o[0, :, 2:].isnan().any()
    assert not o[1].isnan().any() and lse.cpu()[0, 2:, :2].isnan().all()
    c = Case([40, 40], heads=4, kv=2, seed=76)
    c.q[0, 0, 1, 3] = math.inf
    o = c.run()[0].cpu()
    assert o[0, 0, 1].isnan().all() and not o[0, 0, 0].isnan().any() and not o[1].isnan().any()


def test_attention_pages_outside():
    """Pages that the cache does not have hold no keys; lengths beyond the table end with it."""
    c = Case([64, 64], heads=4, kv=2, poison=False, seed=77)
    good, _ = c.run()
    t = c.tables.to(torch.int32)
    t[0, 1], t[0, 2] = -1, 10 ** 6
    out, lse = tg.cache_attention(c.q.cuda(), c.cache, t.cuda(), torch.tensor([64, 64], dtype=torch.int32).cuda(), return_lse=True)
    assert status() == 2
    assert torch.equal(out[1], good[1])
    keep = torch.cat([c.own[0][:16], c.own[0][48:]])
    r, _, spread = ref.attend(c.q[0].double(), c.k[keep], c.v[keep], c.scale)
    assert ((out[0].cpu().double() - r).abs() <= ref.tolerance(r, spread, BF, 128)).all()
    long = tg.cache_attention(c.q.cuda(), c.cache, c.tables.to(torch.int32)[:, :4].cuda(),
                              torch.tensor([2 ** 31 - 1, -7], dtype=torch.int32).cuda())
    assert torch.equal(long[0], good[0]) and (long[1] == 0).all()
    none = tg.cache_attention(c.q.cuda(), c.cache, c.tables.to(torch.int32)[:, :0].cuda(), torch.tensor([3, 4], dtype=torch.int32).cuda())
    assert (none == 0).all() and status() == 0


def test_attention_strides_out_and_shapes():
    c = Case([33, 80], heads=4, kv=2, seed=78)
    good, lse = c.run()
    t, n = c.tables.to(torch.int32).cuda(), torch.tensor(c.lengths, dtype=torch.int32).cuda()
    q3 = c.q.cuda()[:, 0]
    assert torch.equal(tg.cache_attention(q3, c.cache, t, n), good[:, 0])
    wide = torch.randn(2, 9, 200, device="cuda").to(BF)
    wide[:, 1:9:2, 3:131] = q3
    assert torch.equal(tg.cache_attention(wide[:, 1:9:2, 3:131], c.cache, t, n), good[:, 0])
    flipped = q3.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(tg.cache_attention(flipped, c.cache, t, n), good[:, 0])
    out = torch.empty_like(q3)
    assert tg.cache_attention(q3, c.cache, t, n, out=out) is out and torch.equal(out, good[:, 0])
    spaced = torch.zeros(2, 2 * t.shape[1], dtype=torch.int32, device="cuda")
    spaced[:, ::2] = t
    assert torch.equal(tg.cache_attention(q3, c.cache, spaced[:, ::2], n), good[:, 0])
    assert tg.cache_attention(q3[:0], c.cache, t[:0], n[:0]).shape == (0, 4, 128)
    assert tg.cache_attention(c.q.cuda()[:, :0], c.cache, t, n).shape == (2, 0, 4, 128)


def test_cache_beyond_32_bits():
    """Cells whose byte offsets pass 2^32."""
    pages, page = 2 ** 32 // (64 * 2 * 256) + 64, 64
    cache = tg.PackedCache.empty(pages, page, 2, 256, "int8")
    k, v = randn((100, 2, 256), 80, BF), randn((100, 2, 256), 81, BF)
    table = torch.tensor([[pages - 1, pages - 2, 0]], dtype=torch.int32)
    at = torch.arange(100)
    slots = table[0].long()[at // page] * page + at % page
    tg.cache_write(cache, k.cuda(), v.cuda(), slots.cuda())
    kk, vv = (x.cpu() for x in tg.cache_read(cache, slots.cuda(), dtype=torch.float32))
    codes, scales = ref.quantise(k.float(), "int8", 256, False)
    assert torch.equal(kk, ref.read_back(codes, scales, 256))
    q = randn((1, 4, 256), 82, BF)
    out = tg.cache_attention(q.cuda(), cache, table.cuda(), torch.tensor([100], dtype=torch.int32).cuda())
    r, _, spread = ref.attend(q.double(), kk.double(), vv.double(), 1 / 16)
    assert ((out.cpu().double() - r).abs() <= ref.tolerance(r, spread, BF, 256)).all()


def test_side_streams_and_graph():
    """Calls on streams of their own, and a recorded step replayed with other lengths."""
    c = Case([900, 30], heads=8, kv=2, page=64, prefix=200, seed=83, per=20)
    good, _ = c.run()
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    outs = []
    for s in streams:
        with torch.cuda.stream(s):
            for _ in range(3):
                outs.append(c.run()[0])
    torch.cuda.synchronize()
    assert all(torch.equal(o, good) for o in outs)
    t, p = c.tables.to(torch.int32).cuda(), c.prefix.to(torch.int32).cuda()
    step = tg.GraphStep(lambda q, n: tg.cache_attention(q, c.cache, t, n, prefix=p, prefix_length=200), c.q.cuda(),
                        torch.tensor([900, 30], dtype=torch.int32).cuda())
    assert torch.equal(step(), good)
    c.lengths, c.own = [17, 640], [c.own[0][:17], c._slots(c.tables[1], 640)]
    # (the second request's further keys are NaN in the cache: give them values)
    k, v = randn((640, 2, 128), 84).cuda(), randn((640, 2, 128), 85).cuda()
    tg.cache_write(c.cache, k, v, c.own[1].cuda())
    kk, vv = tg.cache_read(c.cache, torch.arange(c.cache.pages * 64).cuda(), dtype=torch.float32)
    c.k, c.v = kk.cpu().double(), vv.cpu().double()
    out = step(c.q.cuda(), torch.tensor([17, 640], dtype=torch.int32).cuda()).clone()
    _, lse = c.run()
    c.check(out, lse)


def test_first_call_captured():
    """A stream whose first call is captured has no workspace yet: the same result, less parallel."""
    c = Case([2000, 3, 0], heads=4, kv=2, page=64, seed=86)
    good, _ = c.run()
    q, t, n = c.q.cuda(), c.tables.to(torch.int32).cuda(), torch.tensor(c.lengths, dtype=torch.int32).cuda()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        out = tg.cache_attention(q, c.cache, t, n)
    graph.replay()
    torch.cuda.synchronize()
    c.check(out, c.run()[1])
    assert good.shape == out.shape


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("e8", [False, True])
@pytest.mark.parametrize("queries,prefix", [(1, 300), (40, 0), (70, 130)])
def test_attention_without_logarithms(fmt, e8, queries, prefix):
    """Results alone: key codes may take their scales before the products then, rounded to fp16 (2^-11 a
    term, like a block-scaled cache's)."""
    c = Case([200, queries, 5, 0], queries=queries, heads=16, kv=2, fmt=fmt, e8=e8, prefix=prefix, seed=90)
    c.blocked = True
    _, lse = c.run()
    shared = dict(prefix=c.prefix.to(torch.int32).cuda(), prefix_length=prefix) if prefix else {}
    out = tg.cache_attention(c.q.cuda(), c.cache, c.tables.to(torch.int32).cuda(),
                             torch.tensor(c.lengths, dtype=torch.int32).cuda(), **shared)
    c.check(out, lse)


@pytest.mark.parametrize("rows", ["few", "many"])
@pytest.mark.parametrize("fmt,blocked", [("int8", False), ("fp4_e2m1", True), ("int4", False), ("fp8e4m3", True)])
def test_attention_outliers_that_are_not_seen(rows, fmt, blocked):
    """Keys and values 2^40 times the others', infinite or NaN, behind what most queries see: theirs are as
    without them."""
    queries = 1 if rows == "few" else 24
    c = Case([150, 150], queries=queries, heads=4, kv=1, fmt=fmt, blocked=blocked, seed=91, per=10, page=16)
    good, _ = c.run()
    big = torch.randn(1, 1, 128) * 2.0 ** 40
    bad = big.clone()
    bad[0, 0, 7], bad[0, 0, 50] = math.inf, math.nan
    last = c.own[0][149:150].cuda()  # request 0's last key: its last query alone sees it
    for x in (big, bad):
        tg.cache_write(c.cache, x.cuda(), x.cuda(), last)
        out, lse = c.run()
        if queries > 1:
            assert torch.equal(out[1], good[1])
            tol = 2.0 ** -7 * good[0, :-1].abs() + 2.0 ** -9 * good[0, :-1].abs().max()  # two runs' roundings
            assert ((out[0, :-1].float() - good[0, :-1].float()).abs() <= tol.float()).all()
        else:  # one query sees it: beyond the length instead
            n = torch.tensor([149, 150], dtype=torch.int32).cuda()
            o = tg.cache_attention(c.q.cuda(), c.cache, c.tables.to(torch.int32).cuda(), n)
            assert not o.isnan().any() and torch.equal(o[1], good[1])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("blocked,e8", [(False, False), (False, True), (True, False), (True, True)])
@pytest.mark.parametrize("queries,heads,kv", [(17, 8, 2), (33, 12, 2)])
def test_attention_many_rows_formats(fmt, dim, blocked, e8, queries, heads, kv):
    """68 and 198 query rows of a key head; lengths that end inside the block, before it and behind it."""
    Case([queries, 0, 200, 3, 129], queries=queries, heads=heads, kv=kv, dim=dim, fmt=fmt, blocked=blocked, e8=e8,
         order="tokens" if e8 else "heads", seed=93).check()


@pytest.mark.parametrize("queries,heads,kv", [(1, 16, 1), (1, 17, 1), (16, 4, 1), (13, 5, 1), (32, 4, 1), (43, 3, 1), (4, 16, 1)])
@pytest.mark.parametrize("prefix", [0, 1, 131])
def test_attention_rows_where_kernels_change(queries, heads, kv, prefix):
    Case([queries + 2, 0, 140, 31], queries=queries, heads=heads, kv=kv, dim=64, fmt="int8", prefix=prefix, seed=94).check()


@pytest.mark.parametrize("fmt,dim,lengths", [("int4", 64, [4096, 300]), ("int8", 128, [129, 1025, 0, 2047]), ("fp8e4m3", 256, [700])])
def test_attention_segments_cut_to_single_rounds(fmt, dim, lengths):
    c = Case(lengths, heads=8, kv=2, dim=dim, fmt=fmt, page=64, seed=95)
    a, b = c.run(), c.run()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    c.check(*a)


def test_attention_prefix_over_many_launches():
    """More requests than one launch takes, behind a prefix whose segments are cut."""
    lengths = torch.randint(0, 20, (4500,), generator=gen(96)).tolist()
    Case(lengths, heads=2, kv=1, dim=64, fmt="int4", prefix=600, seed=97).check()


def test_attention_prefix_follows_its_inputs():
    """Queries, keys and lengths that the launches right before have written: the same bits as when each
    call waits for everything before it."""
    c = Case([90, 33, 64, 2] * 12, heads=16, kv=2, fmt="int8", prefix=1500, seed=98)
    tables, prefix = c.tables.to(torch.int32).cuda(), c.prefix.to(torch.int32).cuda()
    last = torch.stack([o[n - 1] for o, n in zip(c.own, c.lengths)]).cuda()
    qs = [torch.randn(c.q.shape, generator=gen(i)).to(c.q.dtype).cuda() for i in range(8)]
    xs = [randn((len(c.lengths), 2, 128), 200 + i).cuda() for i in range(8)]
    ns = [torch.tensor([max(0, n - i) for n in c.lengths], dtype=torch.int32).cuda() for i in range(8)]
    q, n = torch.empty_like(qs[0]), torch.empty_like(ns[0])

    def step(i, wait):
        q.copy_(qs[i]), n.copy_(ns[i])
        tg.cache_write(c.cache, xs[i], xs[i], last)
        if wait:
            torch.cuda.synchronize()
        out = tg.cache_attention(q, c.cache, tables, n, prefix=prefix, prefix_length=1500)
        if wait:
            torch.cuda.synchronize()
        return out

    good = [step(i, True) for i in range(8)]
    for _ in range(10):
        fast = [step(i, False) for i in range(8)]
        assert all(torch.equal(a, b) for a, b in zip(fast, good))
    assert not torch.equal(good[0], good[1])


@pytest.mark.parametrize("blocked", [False, True])
def test_attention_many_rows_value_ranges(blocked):
    """Scales that span 2^40 from key to key under many query rows."""
    Case([400], queries=40, heads=8, kv=2, fmt="int8", blocked=blocked, e8=True, spread=10.0, q_gain=8.0, seed=92).check()


# ---- refusals ---------------------------------------------------------------------------------------
def test_refusals():
    cache = make_cache("int8", 128, heads=2)
    table = tg.RotaryTable.build(128, 10)
    x = torch.zeros(3, 2, 128, dtype=BF, device="cuda")
    pos = torch.zeros(3, dtype=torch.int64, device="cuda")
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    bad = [
        (lambda: tg.rotary(x[0], table, pos[:2]), "takes"),
        (lambda: tg.rotary(x.double(), table, pos), "float16"),
        (lambda: tg.rotary(x, table, pos[:2]), "shape"),
        (lambda: tg.rotary(x, table, pos.float()), "int32 or int64"),
        (lambda: tg.rotary(x, table, pos.cpu()), "must be on"),
        (lambda: tg.rotary(x[..., :64], table, pos), "does not fit"),
        (lambda: tg.rotary(x, table, pos, out=x.float()), "out must"),
        (lambda: tg.cache_write(cache, x[:, :1], x, pos), "must have shape"),
        (lambda: tg.cache_write(cache, x, x[:2], pos), "same tokens"),
        (lambda: tg.cache_write(cache, x, x.float(), pos), "share a type"),
        (lambda: tg.cache_write(cache, x, x, pos, table), "go together"),
        (lambda: tg.cache_write(cache, x, x, pos, q=x), "needs table"),
        (lambda: tg.cache_write(cache, x, x, pos[:1]), "shape"),
        (lambda: tg.cache_read(cache, pos, dtype=torch.int8), "float16"),
        (lambda: tg.cache_read(cache, pos[None]), "one-dimensional"),
        (lambda: tg.cache_attention(x.float(), cache, i32(3, 1), i32(3)), "float16 or bfloat16"),
        (lambda: tg.cache_attention(x[..., :64], cache, i32(3, 1), i32(3)), "must have shape"),
        (lambda: tg.cache_attention(x[:, :1], cache, i32(3, 1), i32(3)), "evenly"),
        (lambda: tg.cache_attention(x, cache, i32(2, 1), i32(3)), "tables"),
        (lambda: tg.cache_attention(x, cache, i32(3, 1).long(), i32(3)), "tables"),
        (lambda: tg.cache_attention(x, cache, i32(3, 1), i32(2)), "lengths"),
        (lambda: tg.cache_attention(x, cache, i32(3, 1), i32(3).cpu()), "must be on"),
        (lambda: tg.cache_attention(x, cache, i32(3, 1), i32(3), prefix_length=4), "needs"),
        (lambda: tg.cache_attention(x, cache, i32(3, 1), i32(3), prefix=i32(1), prefix_length=17), "hold"),
        (lambda: tg.cache_attention(x, cache, i32(3, 1), i32(3), out=x.float()), "out must"),
    ]
    for call, msg in bad:
        with pytest.raises(ValueError, match=msg):
            call()
    with pytest.raises(_lib.B200Error, match="injected"):
        _lib.lib().b200_inject_failure(1, -5)
        tg.cache_attention(x, cache, i32(3, 1), i32(3))
