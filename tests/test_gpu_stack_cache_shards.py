"""The stack's caches over several ranks: each rank keeps its own key heads. Ranks' shares of one layer's
projected tokens, one after the other on one GPU, against the layer that is not split."""

from __future__ import annotations

import dataclasses

import pytest
import torch

import tinygrad_dx12_b200 as tg
from tests.stack_helpers import SMALL_INT4
from tests.test_gpu_stack_attention import layout, step_of
from tinygrad_dx12_b200 import stack as S

pytestmark = pytest.mark.gpu
CFG = dataclasses.replace(SMALL_INT4, q_dim=512, kv_dim=256)  # 8 heads of 64 over 4


def caches(world):
    return S.StackCache(CFG, tg.RotaryTable.build(64, 256), pages=40, page_size=16, head_dim=64, format="int8", world=world,
                        layers=1)


@pytest.mark.parametrize("world", [2, 4])
@pytest.mark.parametrize("tokens,prefix", [(1, 0), (40, 0), (1, 30)])
def test_shares_of_ranks(world, tokens, prefix):
    whole, ranks = caches(1), [caches(world) for _ in range(world)]
    front, tables = layout(2, 8, first=2)
    g = torch.Generator().manual_seed(510)
    q, kv = CFG.q_dim // world, CFG.kv_dim // world

    def attend(step, n):
        """The layer's whole result, and the ranks' side by side."""
        x = torch.randn((n, CFG.q_dim + 2 * CFG.kv_dim), generator=g).half().cuda()
        qs, ks, vs = x.split([CFG.q_dim, CFG.kv_dim, CFG.kv_dim], 1)
        parts = [c.attend(0, torch.cat([qs[:, r * q:(r + 1) * q], ks[:, r * kv:(r + 1) * kv], vs[:, r * kv:(r + 1) * kv]], 1), q, step)
                 for r, c in enumerate(ranks)]
        return whole.attend(0, x, CFG.q_dim, step), torch.cat(parts, 1)

    if prefix:
        attend(step_of(front[None], 0, prefix), prefix)
    shared = (front, prefix) if prefix else ()
    for start in range(3):
        a, b = attend(step_of(tables, start * tokens, tokens, *shared), 2 * tokens)
        # the runs are cut differently over the SMs: two roundings of the result and of its weights
        assert ((a - b).abs() <= 2.0 ** -10 * a.abs() + 2.0 ** -9 * a.abs().max()).all()
    for name in ("k", "v", "k_scales", "v_scales"):  # each rank's cache holds its heads of the whole one
        every = torch.cat([getattr(c.layers[0], name) for c in ranks], 1)
        assert torch.equal(every.view(torch.uint8), getattr(whole.layers[0], name).view(torch.uint8))
