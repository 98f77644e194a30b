"""The epilogue's activations alone: rows of zeros, so that a bias in fp32 is what is activated, to the bit. Every value of
the result is held to its own size, the tails among them."""

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


def grid():
    """4096 values: the middle, both tails until they vanish, the neighbourhood of zero."""
    ends = torch.cat((torch.linspace(-12, 12, 2400), torch.linspace(-110, -12, 800), torch.linspace(12, 110, 200)))
    small = torch.logspace(-37, 0, 348)
    return torch.cat((ends, small, -small)).float().cuda()


def relative(v, name):
    """How far fp32 may take an activation of v from its value, relative to it, and absolutely where it vanishes.

    A sigmoid by t = e^-|z| <= 1 as a power of two: the power 2 ulp and its correction half of one, 1 + t another half, the
    division 2, two products one: 6 ulp, at most 2^-23 each; 8 are allowed. log2(e) as a number of fp32 is off by 1.4e-8 of
    itself, which moves the power by |z| times that, |z| / 8 ulp; a power below 2^-126 is zero, and v multiplies it. tanh's
    form: its argument has 5 roundings of half an ulp, each of which moves the power by |z| of it.
    gelu by 2^(-v^2 log2(e) / 2) times a polynomial in 1 / (1 + p|v|): its eight steps and its fit 3.3 (its terms add up to 2.3
    times its value), the power 2 and its correction half of one, the division 2, products and the subtraction 2: 10, and 12 are
    allowed; log2(e) / 2 moves the power by v^2 / 18 ulp; below 2^-126 it is zero, and half of v multiplies it."""
    ulp, a = 2.0 ** -23, v.abs()
    z = {"silu": a, "gelu_tanh": 2 * math.sqrt(2 / math.pi) * (a + 0.044715 * a ** 3)}.get(name, torch.zeros_like(a))
    rel = ((12 if name == "gelu" else 8) + z / 8) * ulp
    least = (2 * a.clamp(max=200) + 2) * 2.0 ** -149
    if name == "gelu":
        return rel + ulp * a.square() / 18, least + a.clamp(max=15) * 2.0 ** -127
    if name == "gelu_tanh":
        rel = rel + 2.5 * ulp * z
    return rel, least + a.clamp(max=128) * 2.0 ** -126


def exactly(v, name):
    """The activation in 64 bits; gelu's tail by erfc's scaled form, which keeps its precision."""
    if name != "gelu":
        return H.activate(v, name)
    z = v.abs().clamp(max=40) * math.sqrt(0.5)  # the tail of 40 is no number of 64 bits
    tail = 0.5 * torch.special.erfcx(z) * torch.exp(-z * z)
    return v * torch.where(v < 0, tail, 1 - tail)


def subnormal(dtype):
    """Half the distance between the type's subnormals (fp16's: ``half_step``)."""
    return {torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}.get(dtype, 0.0)


def activated(tg, bias, general, rows=17, **kw):
    from tinygrad_dx12_b200 import scaled

    g = H.generator(1)
    x, w = tg.quantize(torch.zeros((rows, 128), device="cuda")), H.make_weights((bias.numel(), 128), "fp4_e2m1", g)
    return scaled.scaled_linear(x, w, bias=bias, _general=general, **kw)


@pytest.mark.parametrize("general", [True, False])
@pytest.mark.parametrize("name", ["relu", "silu", "gelu", "gelu_tanh"])
def test_activation_by_its_own_size(tg, name, general):
    v = grid()
    want = exactly(v.double(), name)
    rel, least = relative(v.double(), name)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        y = activated(tg, v, general, activation=name, dtype=dtype)
        H.check(y, want.expand(17, -1), (rel * want.abs() + least + subnormal(dtype)).expand(17, -1))


@pytest.mark.parametrize("general", [True, False])
@pytest.mark.parametrize("name", ["relu", "silu", "gelu", "gelu_tanh"])
def test_gate_by_its_own_size(tg, name, general):
    """A tail times a large number is no tail."""
    v = grid()
    up = torch.exp2(torch.linspace(-20, 20, v.numel(), device="cuda")) * torch.where(torch.arange(v.numel(), device="cuda") % 3 == 0, -1.0, 1.0)
    want = exactly(v.double(), name) * up.double()
    rel, least = relative(v.double(), name)
    tol = (rel + 2.0 ** -24) * want.abs() + least * up.abs() + 2.0 ** -149
    bias = torch.cat((v, up))
    for dtype in (torch.float32, torch.bfloat16):
        y = activated(tg, bias, general, activation=name, gated=True, dtype=dtype)
        H.check(y, want.expand(17, -1), (tol + subnormal(dtype)).expand(17, -1))
    H.check8(activated(tg, bias, general, activation=name, gated=True, dtype=E4M3), want.expand(17, -1), tol.expand(17, -1))


@pytest.mark.parametrize("general", [True, False])
@pytest.mark.parametrize("name", [None, "relu", "silu", "gelu", "gelu_tanh"])
def test_infinities_nan_and_large_values(tg, name, general):
    """What the formula gives for them in 64 bits, as fp32 holds it."""
    v = torch.tensor([-math.inf, -3e38, -1.5, -0.0, 0.0, 2.0, 3e38, math.inf, math.nan], device="cuda")
    v = torch.cat((v, v[:7].flip(0)))  # a block's half

    def same(y, want):
        want32 = want.float()
        assert torch.equal(y.isnan(), want32.isnan().expand_as(y)) and torch.equal(y.isinf(), want32.isinf().expand_as(y))
        inf = want32.isinf()
        assert torch.equal(y[:, inf], want32[inf].expand(y.shape[0], -1))
        fin = want32.isfinite()
        assert bool(((y[:, fin].double() - want[fin]).abs() <= 16 * 2.0 ** -23 * want[fin].abs()).all())

    same(activated(tg, v, general, activation=name, dtype=torch.float32), exactly(v.double(), name))
    gate, up = v.repeat_interleave(v.numel()), v.repeat(v.numel())
    y = activated(tg, torch.cat((gate, up)), general, activation=name, gated=True, dtype=torch.float32)
    # the activated half is a number of fp32 before the gate's product
    a = exactly(gate.double(), name).float().double()
    same(y, a * up.double())
