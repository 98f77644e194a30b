"""Derivatives of rotary() beside the plain backward pass: forward mode, torch.func's transforms, and either
over the other. The map is linear, so every answer is the map or its transpose of something known, in
rotary()'s own bits; an answer that mixes in torch's arithmetic gets a tolerance."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import tinygrad_dx12_b200 as tg

pytestmark = pytest.mark.gpu


def operands(dtype=torch.float32):
    table = tg.RotaryTable.build(32, 50, layout="interleaved")
    g = torch.Generator().manual_seed(500)
    x, t = (torch.randn((6, 3, 64), generator=g).to(dtype).cuda() for _ in "xt")
    return x, t, table, torch.arange(6).cuda() * 7


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("transpose", [False, True])
def test_forward_mode(dtype, transpose):
    x, t, table, pos = operands(dtype)
    y, dy = tg.rotary(x, table, pos, transpose), tg.rotary(t, table, pos, transpose)
    with forward_ad.dual_level():
        out = forward_ad.unpack_dual(tg.rotary(forward_ad.make_dual(x, t), table, pos, transpose))
        assert torch.equal(out.primal, y) and torch.equal(out.tangent, dy)
        assert forward_ad.unpack_dual(tg.rotary(x, table, pos, transpose)).tangent is None
        with pytest.raises(ValueError, match="cannot write into out"):
            tg.rotary(forward_ad.make_dual(x, t), table, pos, out=torch.empty_like(x))
        with torch.no_grad():  # a tangent is no gradient
            assert torch.equal(forward_ad.unpack_dual(tg.rotary(forward_ad.make_dual(x, t), table, pos, transpose)).tangent, dy)
    with forward_ad.dual_level():  # a dual tensor that needs a gradient, too
        z = x.clone().requires_grad_()
        out = tg.rotary(forward_ad.make_dual(z, t), table, pos, transpose)
        assert torch.equal(forward_ad.unpack_dual(out).tangent, dy)
        (gz,) = torch.autograd.grad(forward_ad.unpack_dual(out).primal, z, t)
        assert torch.equal(gz, tg.rotary(t, table, pos, not transpose))


def test_transforms():
    x, t, table, pos = operands()
    f = lambda a: tg.rotary(a, table, pos)  # noqa: E731
    y, dy = torch.func.jvp(f, (x,), (t,))
    assert torch.equal(y, f(x)) and torch.equal(dy, f(t))
    assert torch.equal(torch.func.grad(lambda a: (f(a) * t).sum())(x), tg.rotary(t, table, pos, transpose=True))
    y, pull = torch.func.vjp(f, x)
    assert torch.equal(pull(t)[0], tg.rotary(t, table, pos, transpose=True))


def test_one_over_the_other():
    """Of sum(rotary(x)^3) / 3: the gradient is R^T y^2, its derivative along t is 2 R^T (y * R t)."""
    x, t, table, pos = operands()
    f = lambda a: (tg.rotary(a, table, pos) ** 3).sum() / 3  # noqa: E731
    y, dy = tg.rotary(x, table, pos), tg.rotary(t, table, pos)
    want = tg.rotary(2 * y * dy, table, pos, transpose=True)
    close = lambda a: torch.allclose(a, want, rtol=2.0 ** -18, atol=2.0 ** -18 * want.abs().max().item())  # noqa: E731
    assert close(torch.func.jvp(torch.func.grad(f), (x,), (t,))[1])
    assert close(torch.func.grad(lambda a: (torch.func.grad(f)(a) * t).sum())(x))
    assert close(torch.func.grad(lambda a: torch.func.jvp(f, (a,), (t,))[1])(x))
    z = x.clone().requires_grad_()
    (g,) = torch.autograd.grad(f(z), z, create_graph=True)
    assert close(torch.autograd.grad(g, z, t)[0])
    assert torch.allclose(g, tg.rotary(y * y, table, pos, transpose=True), rtol=2.0 ** -18, atol=2.0 ** -18)


def test_positions_changed_before_the_gradient():
    x, t, table, pos = operands()
    z = x.clone().requires_grad_()
    y = tg.rotary(z, table, pos)
    pos += 1
    with pytest.raises(RuntimeError, match="changed in place"):
        torch.autograd.grad(y, z, t)


def test_no_rule_for_vmap():
    """A transform without a rule refuses; nothing runs on a batched tensor's storage."""
    x, _, table, pos = operands()
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda a: tg.rotary(a, table, pos))(x[None].expand(2, 6, 3, 64))
