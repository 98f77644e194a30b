"""Products on either side of the token counts where their tiles change form, dense and by experts' shares."""

import pytest
import torch

import scaled_helpers as H
from test_gpu_experts import pairs64
from test_gpu_scaled import activations, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tg():
    import tinygrad_dx12_b200 as tg

    return tg


@pytest.mark.parametrize("m", [1024, 1025, 2303, 2304, 2305, 2400, 5000])
@pytest.mark.parametrize("n,k", [(700, 256), (4096, 384)])
def test_dense(tg, m, n, k):
    g = H.generator(m)
    x = activations(tg, m, k, g)
    run(tg, x, H.make_weights((n, k), "fp4_e2m1", g), dtype=torch.float32)
    run(tg, x, H.make_weights((n, k), "fp6_e2m3", g), dtype=torch.bfloat16, activation="gelu", bias=torch.randn(n, device="cuda", generator=g))


@pytest.mark.parametrize("share", [100, 112, 113, 224, 225, 600, 1100])
@pytest.mark.parametrize("n,k", [(640, 256), (2304, 384)])
def test_experts(tg, share, n, k):
    g = H.generator(share)
    tokens = share * 3 // 2
    at = torch.rand((tokens, 3), device="cuda", generator=g).argsort(-1)[:, :2].to(torch.int32)
    r = tg.plan_experts(at, torch.rand((tokens, 2), device="cuda", generator=g), 3)
    x, w = tg.quantize(torch.randn((tokens, k), device="cuda", generator=g)), H.make_weights((3, n, k), "fp6_e3m2", g)
    bias = torch.randn((3, n), device="cuda", generator=g)
    for kw in (dict(bias=None), dict(bias=bias, activation="silu")):
        v, tol = pairs64(H.values(x.codes, x.scales), w, r, **kw)
        y = tg.expert_linear(x, w, r, dtype=torch.float32, **kw)
        H.check(y, v, tol)
        assert torch.equal(y, tg.expert_linear(x, w, r, dtype=torch.float32, **kw))
