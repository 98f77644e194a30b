"""Block-scaled rows, the RMS norm that makes them, and their products with packed weights, against their
formulas in 64 bits. Tolerances: ``scaled_helpers``."""

import ctypes
import math

import pytest
import torch

import scaled_helpers as H

pytestmark = pytest.mark.gpu
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


@pytest.fixture(scope="module")
def tg():
    import tinygrad_dx12_b200 as tg

    return tg


def rows(shape, g, dtype=torch.float32, gain=1.0):
    return (torch.randn(shape, device="cuda", generator=g) * gain).to(dtype)


# ---- block-scaled rows -------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(1, 32), (3, 96), (5, 1, 64), (2, 8192), (700, 4096), (2, 32800), (1, 65536)])
def test_quantize_to_the_bit(tg, shape, dtype):
    g = H.generator(1)
    x = rows(shape, g, dtype, 3.0) * torch.exp2(torch.randint(-12, 12, (*shape[:-1], 1), device="cuda", generator=g).to(dtype))
    y = tg.quantize(x)
    codes, scales = H.quantise(x)
    assert torch.equal(y.codes.view(torch.uint8), codes.view(torch.uint8))
    assert torch.equal(y.scales.view(torch.uint8), scales)
    for out in (torch.float32, torch.bfloat16):
        assert torch.equal(y.values(out).double(), H.values(codes, scales))


def test_quantize_borders(tg):
    """Zeros, subnormals, the largest values, infinities, NaN, magnitudes on either side of a power of two."""
    x = torch.zeros((16, 64), device="cuda")
    x[1, 0] = 448.0
    x[2, 0] = math.nextafter(448.0, 1e9) * (1 + 2.0 ** -23)
    x[3, 1] = 1e-40
    x[4, 2] = 3.4e38
    x[5, 3] = math.inf
    x[5, 4] = -math.inf
    x[6, 5] = math.nan
    x[6, 6] = 7.0
    x[7] = torch.linspace(-448, 448, 64)
    x[8] = torch.exp2(torch.arange(64, device="cuda").float() - 50)
    x[9, :32] = 2.0 ** -120
    x[10, 0], x[10, 1] = -0.0, 1.0
    x[11, 0] = 448.0 * 2.0 ** 100
    x[12, 0] = -448.0 * 2.0 ** 101
    y = tg.quantize(x)
    codes, scales = H.quantise(x)
    assert torch.equal(y.scales.view(torch.uint8), scales)
    assert torch.equal(y.codes.view(torch.uint8), codes.view(torch.uint8))
    v = y.values(torch.float32)
    assert v[6, :32].isnan().all() and v[6, 32:].eq(0).all() and not v[5].isnan().any()


def test_values_of_any_scale_byte(tg):
    codes = torch.arange(256, device="cuda").to(torch.uint8).view(E4M3).repeat(32, 1)
    scales = torch.arange(256, device="cuda").to(torch.uint8).view(32, 8).view(E8M0)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        want = H.values(codes, scales).to(dtype)
        got = tg.BlockScaled(codes, scales).values(dtype)
        assert torch.equal(got.isnan(), want.isnan())
        # fp32 holds no product below 2^-149: those of the lowest scale bytes are rounded there
        far = want.abs().double() >= 2.0 ** -126
        assert torch.equal(got[far], want[far])


def test_rows_of_views(tg):
    g = H.generator(2)
    x = rows((6, 5, 256), g, torch.bfloat16)
    for v in (x[::2], x[:, 1:4], x.transpose(0, 1), x[..., 32:96], x[..., ::2], x[..., 1:65]):
        codes, scales = H.quantise(v)
        y = tg.quantize(v)
        assert torch.equal(y.codes.view(torch.uint8), codes.view(torch.uint8)) and torch.equal(y.scales.view(torch.uint8), scales)
    y = tg.quantize(x)
    part = tg.BlockScaled(y.codes[:, ::2], y.scales[:, ::2])
    assert torch.equal(part.values(), y.values()[:, ::2])


# ---- the norm ----------------------------------------------------------------------------------
def norm64(t, weight, eps):
    y = t / (t.square().mean(-1, keepdim=True) + eps).sqrt()
    return y if weight is None else y * weight.double()


# fp32: the sum of squares has a relative error below (cols / 1024 + 40) 2^-24 (a thread's own terms, the tree, the
# division, the root's 2 ulp), its root half of that; two products round
def norm_tol(y, cols):
    return y.abs() * ((cols / 1024 + 40) / 2 + 4) * 2.0 ** -24


@pytest.mark.parametrize("shape", [(1, 8192), (1, 64), (3, 96), (2, 3, 4096), (700, 1024), (301, 8192), (5, 1000), (4, 7),
                                   (2, 16384), (3, 40000), (1, 32768), (600, 2048), (1, 1)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("residual", [False, True])
def test_norm(tg, shape, dtype, residual):
    g = H.generator(3)
    cols = shape[-1]
    x, weight = rows(shape, g, dtype, 2.0), 1 + 0.2 * rows((cols,), g)
    r = rows(shape, g, dtype, 5.0) if residual else None
    t = (x.float() + r.float()).to(dtype) if residual else x
    want = norm64(t.double(), weight, 1e-5)
    for out in [dtype, torch.float32] + ([E4M3] if cols % 32 == 0 else []):
        y = tg.rms_norm(x, weight, eps=1e-5, residual=r, dtype=out)
        if residual:
            y, total = y
            assert torch.equal(total, t)
        (H.check8 if out == E4M3 else H.check)(y, want, norm_tol(want, cols))


@pytest.mark.parametrize("wdtype", [None, torch.float16, torch.bfloat16, torch.float32])
def test_norm_weights_and_types(tg, wdtype):
    """A weight of each type or none; residuals of another type than x."""
    g = H.generator(4)
    x = rows((9, 512), g, torch.bfloat16)
    weight = None if wdtype is None else rows((512,), g, wdtype)
    y = tg.rms_norm(x, weight)
    want = norm64(x.double(), weight, 1e-6)
    H.check(y, want, norm_tol(want, 512))
    r = rows((9, 512), g, torch.float32)
    y, total = tg.rms_norm(x, weight, residual=r, dtype=E4M3)
    assert total.dtype == torch.float32 and torch.equal(total, x.float() + r)
    want = norm64(total.double(), weight, 1e-6)
    H.check8(y, want, norm_tol(want, 512))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cols", [256, 8192, 1000])
def test_norm_of_sums_in_32_bits(tg, dtype, cols):
    """fp32 partial sums added into a 16-bit stream, in place."""
    g = H.generator(cols)
    x, h = rows((21, cols), g, torch.float32, 3.0), rows((21, cols), g, dtype)
    t = (x + h.float()).to(dtype)
    for out in [dtype] + ([E4M3] if cols % 32 == 0 else []):
        into = h.clone()
        y, total = tg.rms_norm(x, residual=into, total=into, dtype=out)
        assert total is into and torch.equal(into, t)
        want = norm64(t.double(), None, 1e-6)
        (H.check8 if out == E4M3 else H.check)(y, want, norm_tol(want, cols))


def test_norm_in_place_and_views(tg):
    g = H.generator(5)
    x, h = rows((33, 4096), g, torch.bfloat16), rows((33, 4096), g, torch.bfloat16)
    t = (x.float() + h.float()).bfloat16()
    y, total = tg.rms_norm(x, residual=h, total=h)
    assert total is h and torch.equal(h, t)
    wide = rows((33, 3 * 512), g, torch.float16)
    for v in (wide[:, 512:1024], wide[::2, :512], wide[:, 3:515], wide.T[:, :32]):
        want = norm64(v.double(), None, 1e-6)
        H.check(tg.rms_norm(v), want, norm_tol(want, v.shape[-1]))


def test_norm_of_odd_rows(tg):
    """Zeros, infinities and NaN stay in their rows."""
    x = torch.ones((5, 128), device="cuda")
    x[1] = 0
    x[2, 3] = math.inf
    x[3, 4] = math.nan
    y, y8 = tg.rms_norm(x), tg.rms_norm(x, dtype=E4M3).values(torch.float32)
    assert y[1].eq(0).all() and y8[1].eq(0).all()
    assert y[2, 3].isnan() and y[2, 4] == 0 and y[3].isnan().all() and y8[3].isnan().all()
    assert torch.equal(y[4], y[0]) and not y[0].isnan().any()
    assert tg.rms_norm(x[:0]).shape == (0, 128) and tg.rms_norm(x[:0], dtype=E4M3).shape == (0, 128)


# ---- products ----------------------------------------------------------------------------------
def activations(tg, m, k, g):
    x = rows((m, k), g)
    x = x * torch.exp2(torch.randint(-2, 3, (m, k // 32), device="cuda", generator=g).float()).repeat_interleave(32, -1)
    return tg.quantize(x)


def run(tg, x, w, general=False, **kw):
    from tinygrad_dx12_b200 import scaled

    y = scaled.scaled_linear(x, w, _general=general, **kw)
    v, tol = H.product(H.values(x.codes, x.scales), H.weights(w), **{k: kw[k] for k in kw if k != "dtype"})
    (H.check8 if kw.get("dtype") == E4M3 else H.check)(y, v, tol)
    return y


@pytest.mark.parametrize("general", [True, False])
@pytest.mark.parametrize("fmt", sorted(H.BITS))
@pytest.mark.parametrize("m,n,k", [(1, 128, 128), (1, 1, 128), (3, 100, 256), (16, 256, 384), (17, 130, 128), (33, 513, 640)])
def test_linear_small(tg, fmt, m, n, k, general):
    g = H.generator(m * 1000 + n)
    x, w = activations(tg, m, k, g), H.make_weights((n, k), fmt, g)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        run(tg, x, w, general, dtype=dtype)


@pytest.mark.parametrize("m", [1, 2, 15, 16, 31, 32, 48, 111, 112, 113, 128, 129, 160, 223, 224, 225, 449, 700])
def test_linear_token_counts(tg, m):
    g = H.generator(m)
    x, w = activations(tg, m, 512, g), H.make_weights((384, 512), "fp4_e2m1", g)
    run(tg, x, w, dtype=torch.float32)
    run(tg, x, w, dtype=torch.float32, gated=True, activation="silu")


@pytest.mark.parametrize("n,k", [(8192, 256), (20000, 128), (128, 8192), (640, 5120), (1, 16384), (9472, 1024)])
@pytest.mark.parametrize("m", [1, 40, 300])
def test_linear_splits(tg, n, k, m):
    """Runs of several tiles, tiles of several runs, and both."""
    g = H.generator(n + k)
    x, w = activations(tg, m, k, g), H.make_weights((n, k), "fp6_e3m2", g)
    a = run(tg, x, w, dtype=torch.float32)
    assert torch.equal(a, tg.scaled_linear(x, w, dtype=torch.float32))


@pytest.mark.parametrize("m,n,k", [(300, 20032, 640), (40, 30016, 384), (1100, 9472, 1152), (230, 9600, 896), (20, 38016, 128)])
@pytest.mark.parametrize("gated", [False, True])
def test_linear_waves(tg, m, n, k, gated):
    """Several tiles a CTA, each begun at another K; stages that are no multiple of four."""
    g = H.generator(m + n)
    x, w = activations(tg, m, k, g), H.make_weights((n, k), "fp6_e2m3", g)
    a = run(tg, x, w, dtype=torch.float32, gated=gated)
    assert torch.equal(a, tg.scaled_linear(x, w, dtype=torch.float32, gated=gated))
    run(tg, x, w, dtype=E4M3, gated=gated, activation="silu")


def test_chain_of_dependent_launches(tg):
    """Norms and products that start as the ones before them end give what they give one by one."""
    g = H.generator(17)
    up, down = H.make_weights((1024, 512), "fp4_e2m1", g), H.make_weights((512, 1024), "fp4_e2m1", g)
    h0 = rows((30, 512), g, torch.bfloat16)

    def layers(wait):
        h = h0
        for _ in range(25):
            x = tg.rms_norm(h, dtype=E4M3)
            wait()
            m = tg.scaled_linear(x, up, activation="gelu", dtype=E4M3)
            wait()
            h = tg.scaled_linear(m, down, residual=h)
            wait()
        return h

    want = layers(torch.cuda.synchronize)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        a = layers(lambda: None)
        with torch.cuda.stream(side):
            b = layers(lambda: None)
        torch.cuda.synchronize()
        assert torch.equal(a, want) and torch.equal(b, want)


@pytest.mark.parametrize("general", [False, True])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("activation", [None, "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, E4M3])
def test_epilogue(tg, activation, gated, dtype, general):
    g = H.generator(7)
    m, n, k = 37, 576, 256
    x, w = activations(tg, m, k, g), H.make_weights((n, k), "fp6_e2m3", g)
    cols = n // 2 if gated else n
    for bias in (None, rows((n,), g, torch.bfloat16)):
        for residual in (None, rows((m, cols), g, torch.float16, 4.0)):
            run(tg, x, w, general, activation=activation, gated=gated, dtype=dtype, bias=bias, residual=residual)


@pytest.mark.parametrize("k", [32, 64, 96, 160, 1056])
def test_linear_ragged_blocks(tg, k):
    """Columns that are no whole stages: the general kernel."""
    g = H.generator(k)
    x = activations(tg, 5, k, g)
    for fmt in H.BITS:
        run(tg, x, H.make_weights((70, k), fmt, g), dtype=torch.float32)


def test_linear_operands_of_any_layout(tg):
    g = H.generator(11)
    w = H.make_weights((192, 256), "fp4_e2m1", g)
    x = tg.quantize(rows((2, 3, 256), g))
    y = tg.scaled_linear(x, w, dtype=torch.float32)
    assert y.shape == (2, 3, 192)
    flat = run(tg, tg.BlockScaled(x.codes.flatten(0, 1), x.scales.flatten(0, 1)), w, dtype=torch.float32)
    assert torch.equal(y.flatten(0, 1), flat)
    wide = tg.quantize(rows((6, 512), g))
    part = tg.BlockScaled(wide.codes[:, 256:], wide.scales[:, 8:])
    run(tg, part, w, dtype=torch.bfloat16)
    # residual rows with a stride of their own; weights off a 32-byte boundary
    res = rows((6, 400), g)
    run(tg, part, w, dtype=torch.float32, residual=res[:, 100:292])
    moved = torch.empty(w.data.numel() + 16, dtype=torch.uint8, device="cuda")[16:]
    moved.copy_(w.data)
    run(tg, part, tg.PackedTensor(moved, w.format, w.shape, w.scales, 32), dtype=torch.float32)
    assert tg.scaled_linear(tg.quantize(rows((0, 256), g)), w).shape == (0, 192)


@pytest.mark.parametrize("k", [1 << 24, (1 << 24) + 128])
def test_linear_of_very_long_rows(tg, k):
    """The last width of the tensor cores' kernel, and the first behind it."""
    g = H.generator(17)
    run(tg, activations(tg, 2, k, g), H.make_weights((3, k), "fp4_e2m1", g), dtype=torch.float32)


def test_nan_stays_in_its_row(tg):
    """A NaN scale of a token or of a weight row reaches that row or column alone."""
    g = H.generator(12)
    x, w = activations(tg, 20, 256, g), H.make_weights((200, 256), "fp4_e2m1", g)
    clean = tg.scaled_linear(x, w, dtype=torch.float32)
    x.scales.view(torch.uint8)[3, 1] = 255
    w.scales.view(torch.uint8)[150, 7] = 255
    for general in (False, True):
        y = tg.scaled.scaled_linear(x, w, dtype=torch.float32, _general=general)
        want = torch.zeros_like(y, dtype=torch.bool)
        want[3], want[:, 150] = True, True
        assert torch.equal(y.isnan(), want)
        if not general:
            assert torch.equal(y[~want], clean[~want])


def test_extreme_scales(tg):
    """The smallest and largest scale bytes: results as fp32 holds them."""
    g = H.generator(13)
    x, w = activations(tg, 4, 128, g), H.make_weights((128, 128), "fp4_e2m1", g)
    x.scales.view(torch.uint8).fill_(127 + 60)
    w.scales.view(torch.uint8).fill_(127 - 100)
    run(tg, x, w, dtype=torch.float32)
    x.scales.view(torch.uint8).fill_(127 - 100)
    w.scales.view(torch.uint8).fill_(127 + 110)
    run(tg, x, w, dtype=torch.float32)


def test_streams_graphs_and_devices(tg):
    """Recorded and replayed beside an eager call on another stream; new inputs at replay."""
    g = H.generator(14)
    w = H.make_weights((640, 1024), "fp4_e2m1", g)
    xs = [rows((24, 1024), g, torch.bfloat16) for _ in range(3)]
    weight = 1 + 0.1 * rows((1024,), g)

    def step(x):
        return tg.scaled_linear(tg.rms_norm(x, weight, dtype=E4M3), w, activation="silu", dtype=torch.float32)

    want = [step(x) for x in xs]
    steps = [tg.GraphStep(step, xs[0]) for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        a = steps[0](xs[1])
        with torch.cuda.stream(side):
            b = steps[1](xs[2])
            c = step(xs[0])
    torch.cuda.synchronize()
    assert torch.equal(a, want[1]) and torch.equal(b, want[2]) and torch.equal(c, want[0])


def test_device_status_is_clean(tg):
    from tinygrad_dx12_b200 import _lib

    torch.cuda.synchronize()
    flags = ctypes.c_uint32(9)
    _lib.call("b200_device_status", 0, ctypes.byref(flags), 0)
    assert flags.value & 1 == 0
