"""TPStack with 8-bit activations between its projections (``ScaledOps``): every step against its formula in 64 bits,
with attention over a cache, recorded, and its shards."""

import pytest
import torch

import scaled_helpers as H
from tests.stack_helpers import CONFIGS, initial_h
from tinygrad_dx12_b200 import stack as S

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


class Checked(S.ScaledOps):
    """Each step's result against the formula over its own inputs, so that no rounding is carried along."""

    def linear(self, w, x, out_dtype):
        import tinygrad_dx12_b200 as tg

        y = super().linear(w, x, out_dtype)
        x8 = x.value if isinstance(x, S._Rows) else x if isinstance(x, tg.BlockScaled) else tg.quantize(x)
        if isinstance(x, torch.Tensor):
            codes, scales = H.quantise(x)
            assert torch.equal(x8.codes.view(torch.uint8), codes.view(torch.uint8)) and torch.equal(x8.scales.view(torch.uint8), scales)
        H.check(y, *H.product(H.values(x8.codes, x8.scales), H.weights(w)))
        return y

    def gated(self, w, x, out, act):
        y = super().gated(w, x, out, act)
        H.check8(y, *H.product(H.values(x.value.codes, x.value.scales), H.weights(w), gated=True))
        return y

    def add_rmsnorm(self, h, partial, x):
        before = h.clone()
        super().add_rmsnorm(h, partial, x)
        t = before if partial is None else (before.float() + partial).to(h.dtype)
        assert torch.equal(h, t)
        want = t.double() / (t.double().square().mean(-1, keepdim=True) + S.EPS).sqrt()
        H.check8(x.value, want, want.abs() * ((h.shape[1] / 1024 + 40) / 2 + 4) * 2.0 ** -24)


def stack(ops, **kw):
    return S.TPStack(CONFIGS["fp4"], device="cuda", ops=ops, **kw)


@pytest.mark.parametrize("m", [1, 5, 130])
def test_every_step(m):
    cfg = CONFIGS["fp4"]
    h = initial_h(cfg, m).cuda()
    y = stack(Checked()).forward(h.clone())
    assert torch.equal(y, stack(S.ScaledOps()).forward(h.clone()))
    # 8-bit rows: each value's rounding is at most 2^-4 of it, 0.026 of it in the mean square; three products a layer
    # read them one behind another, two layers
    r = stack(S.CudaOps()).forward(h.clone())
    assert float((y.float() - r.float()).norm() / r.float().norm()) < 0.026 * 6


def test_recorded_with_attention():
    import tinygrad_dx12_b200 as tg

    cfg = S.StackConfig(hidden=256, q_dim=256, kv_dim=128, inter=512, layers=2, fmt="fp4_e2m1", block=32, scale="e8m0", act=torch.bfloat16)
    st = S.TPStack(cfg, device="cuda", ops=S.ScaledOps())
    table = tg.RotaryTable.build(64, 64, device="cuda")
    cache = S.StackCache(cfg, table, 8, page_size=16, head_dim=64)
    where = S.StackStep(torch.tensor([0, 16], device="cuda"), torch.tensor([0, 0], device="cuda"),
                        torch.tensor([[0], [1]], dtype=torch.int32, device="cuda"), torch.tensor([1, 1], dtype=torch.int32, device="cuda"))
    hs = [initial_h(cfg, 2).cuda() * (i + 1) for i in range(3)]
    want = [st.forward(h.clone(), cache, where) for h in hs]
    step = tg.GraphStep(lambda h: st.forward(h.clone(), cache, where), hs[0])
    for h, w in zip(hs, want):
        assert torch.equal(step(h), w)


def test_int4_stacks_are_refused():
    with pytest.raises(ValueError, match="FP4 or FP6"):
        S.TPStack(CONFIGS["int4"], device="cuda", ops=S.ScaledOps()).forward(initial_h(CONFIGS["int4"], 1).cuda())
