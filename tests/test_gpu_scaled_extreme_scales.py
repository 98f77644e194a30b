"""Scale bytes of activations and weights far apart, whose product alone fp32 has to hold: every kernel, dense and through
experts."""

import pytest
import torch

import scaled_helpers as H

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tg():
    import tinygrad_dx12_b200 as tg

    return tg


@pytest.mark.parametrize("general", [True, False])
@pytest.mark.parametrize("ws,xs", [(127 + 124, 27), (254, 27), (0, 227), (1, 200), (20, 190), (240, 40), (0, 254), (254, 0)])
def test_far_scales(tg, ws, xs, general):
    """Sums of 100 to 10^5 times 2^(ws + xs - 254): normal numbers, though neither factor's product with a sum need be."""
    from tinygrad_dx12_b200 import experts, scaled

    g = H.generator(ws)
    for fmt in sorted(H.BITS):
        x = tg.quantize(torch.randn((5, 128), device="cuda", generator=g))
        w = H.make_weights((2, 64, 128), fmt, g)
        x.scales.view(torch.uint8).fill_(xs)
        w.scales.view(torch.uint8).fill_(ws)
        one = tg.PackedTensor(w.data, fmt, (128, 128), w.scales.view(torch.uint8).view(128, 4).view(torch.float8_e8m0fnu), 32)
        v, tol = H.product(H.values(x.codes, x.scales), H.weights(one))
        assert v.abs().max() < 1e38 and v.abs().median() > 1e-37
        y = scaled.scaled_linear(x, one, dtype=torch.float32, _general=general)
        H.check(y, v, tol)
        r = tg.plan_experts(torch.tensor([[0], [1], [1], [0], [1]], dtype=torch.int32, device="cuda"), torch.ones((5, 1), device="cuda"), 2)
        y = experts.expert_linear(x, w, r, dtype=torch.float32, _general=general)
        at = torch.tensor([0, 1, 1, 0, 1], device="cuda")[:, None] * 64 + torch.arange(64, device="cuda")
        H.check(y, v.gather(1, at), tol.gather(1, at))


def test_a_nan_scale_meets_any_other(tg):
    """Byte 255 is a NaN beside the smallest and the largest scale."""
    from tinygrad_dx12_b200 import scaled

    g = H.generator(3)
    x, w = tg.quantize(torch.randn((3, 128), device="cuda", generator=g)), H.make_weights((64, 128), "fp6_e2m3", g)
    for ws, xs in ((0, 227), (127, 127), (254, 27)):
        for general in (True, False):
            x.scales.view(torch.uint8).fill_(xs)
            w.scales.view(torch.uint8).fill_(ws)
            x.scales.view(torch.uint8)[1, 2] = 255
            y = scaled.scaled_linear(x, w, dtype=torch.float32, _general=general)
            assert y[1].isnan().all() and not y[0].isnan().any() and not y[2].isnan().any()
