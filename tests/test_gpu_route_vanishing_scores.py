"""Routing where scores that decide vanish in 32 bits, or lie closer than their error there: the order is that of 64 bits."""

import math

import pytest
import torch

import scaled_helpers as H
from test_gpu_experts import check_route

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tg():
    import tinygrad_dx12_b200 as tg

    return tg


def far_rows(count, groups, size, low, high, g):
    """Group 0 holds the two largest logits, the others lie ``low`` to ``high`` below."""
    x = -low - (high - low) * torch.rand((count, groups * size), device="cuda", generator=g)
    x[:, 0], x[:, 1] = 0.0, -1.0
    return x


@pytest.mark.parametrize("low,high", [(60, 90), (84, 92), (88, 102), (99, 103), (100, 110), (60, 110)])
@pytest.mark.parametrize("experts,groups", [(8, 4), (64, 16), (96, 8), (256, 32)])
def test_groups_by_vanishing_sums(tg, experts, groups, low, high):
    """Subnormal scores are off by steps of 2^-149, whatever their size."""
    g = H.generator(experts + low)
    x = far_rows(4000, groups, experts // groups, low, high, g)
    for k in (2, 4):
        check_route(tg, x, k, groups=groups, top_groups=2, group_best=2)
    check_route(tg, x[:50], 4, groups=groups, top_groups=2, group_best=2)  # few rows: routing and plan in one launch
    check_route(tg, x, 3, groups=groups, top_groups=2, group_best=2, renormalize=False)


def test_a_row_whose_sums_round_the_other_way(tg):
    x = torch.tensor([[0.0, -1.0, -102.15482, -101.485115, -101.961075, -101.73406, -102.237724, -101.74245]], device="cuda")
    r = check_route(tg, x, 4, groups=4, top_groups=2, group_best=2)
    assert set(r.indices[0].tolist()) == {0, 1, 2, 3}


@pytest.mark.parametrize("low,high", [(60, 90), (88, 103), (100, 110)])
def test_experts_by_vanishing_scores(tg, low, high):
    """A bias of zeros: the scores alone decide."""
    g = H.generator(low)
    x = far_rows(4000, 1, 40, low, high, g)
    zeros = torch.zeros(40, device="cuda")
    check_route(tg, x, 6, bias=zeros)
    check_route(tg, x - 4, 6, bias=zeros, scores="sigmoid")
    check_route(tg, x - 4, 6, groups=8, top_groups=3, group_best=2, scores="sigmoid")


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_scores_within_their_error(tg, scores):
    """Differences of 2^-20 to 2^-15 of scores whose logits lie up to 80 apart, with biases up to the scores' size."""
    g = H.generator(31)
    base = -80 * torch.rand((3000, 1), device="cuda", generator=g).repeat(1, 64)
    x = base + torch.randn((3000, 64), device="cuda", generator=g) * 2.0 ** -16
    x[:, :2] = 0.0  # the largest
    zeros = torch.zeros(64, device="cuda")
    check_route(tg, x, 8, bias=zeros, scores=scores)
    check_route(tg, x, 8, bias=torch.linspace(0, 1e-6, 64, device="cuda"), scores=scores)
    for top_groups in (1, 3, 7):
        check_route(tg, x, 4, groups=8, top_groups=top_groups, group_best=2, scores=scores)
        check_route(tg, x, 4, groups=8, top_groups=top_groups, group_best=2, scores=scores, bias=zeros)


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_groups_by_sums_beyond_32_bits(tg, scores):
    """Two large biases add to infinity in 32 bits; their sums are ordered all the same."""
    g = H.generator(32)
    x = torch.randn((500, 32), device="cuda", generator=g)
    big = torch.finfo(torch.float32).max
    for pairs in ([(math.inf, 1e38), (math.inf, 3e38), (math.inf, math.inf), (big, 2e38)],
                  [(-big, -big), (-big, -3e38), (-2e38, -3e38), (-big, -1e38)]):
        bias = torch.full((32,), -big, device="cuda")
        for i, (a, b) in enumerate(pairs):
            bias[8 * i + 3], bias[8 * i + 6] = a, b
        for top_groups in (1, 2, 3):
            check_route(tg, x, 4, groups=4, top_groups=top_groups, group_best=2, bias=bias, scores=scores)


@pytest.mark.parametrize("pairs", [[(1e38, 3.3e38), (2e38, 3.3e38), (3e38, 3.2e38), (1.5e38, 3e38)],
                                   [(-3e38, -3.1e38), (-1e38, -2.9e38), (-2e38, -2.8e38), (-2.5e38, -1.9e38)]])
def test_one_expert_of_such_groups(tg, pairs):
    """The choice within the group is plain; which group it is, is not."""
    g = H.generator(33)
    x = torch.randn((500, 32), device="cuda", generator=g)
    bias = torch.full((32,), -torch.finfo(torch.float32).max, device="cuda")
    for i, (a, b) in enumerate(pairs):
        bias[8 * i + 3], bias[8 * i + 6] = a, b
    for top_groups in (1, 2, 3):
        check_route(tg, x, 1, groups=4, top_groups=top_groups, group_best=2, bias=bias, scores="sigmoid")
