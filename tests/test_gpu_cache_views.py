"""Caches whose tensors are views with gaps: rows of codes and of scales apart, pages and heads apart, scale rows
that no vector load fits. Written, read back and attended to like a dense cache, to the bit, and nothing in the
gaps is touched."""

from __future__ import annotations

import pytest
import torch

import tinygrad_dx12_b200 as tg
from tests.test_gpu_cache import randn, status

pytestmark = pytest.mark.gpu
BF, E8 = torch.bfloat16, torch.float8_e8m0fnu


def gapped(dense):
    """A cache like ``dense`` (zeros) in larger tensors of 0x55 bytes."""
    def wide(t, row):
        pages, heads, size, n = t.shape
        raw = torch.uint8 if t.dtype == E8 else t.dtype
        big = torch.empty((pages + 1, heads + 2, size + 3, row), dtype=raw, device="cuda")
        big.view(torch.uint8).fill_(0x55)
        view = big[:pages, :heads, :size, :n]
        view.zero_()
        return big, view.view(t.dtype) if t.dtype == E8 else view

    parts = [wide(t, t.shape[3] + 16) for t in (dense.k, dense.v)] + [wide(t, t.shape[3] + 1) for t in (dense.k_scales, dense.v_scales)]
    return [big for big, _ in parts], tg.PackedCache(*(v for _, v in parts), dense.format, dense.head_dim, dense.block_size)


@pytest.mark.parametrize("fmt", ["int8", "fp8e4m3", "int4", "fp4_e2m1"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("blocked,e8", [(False, False), (False, True), (True, False), (True, True)])
def test_views_with_gaps(fmt, dim, blocked, e8):
    dense = tg.PackedCache.empty(9, 32, 3, dim, fmt, block_size=32 if blocked else dim, scale_dtype=E8 if e8 else BF)
    big, cache = gapped(dense)
    before = [t.clone() for t in big]
    n = 9 * 32 - 40
    slots = torch.randperm(9 * 32, generator=torch.Generator().manual_seed(600))[:n].cuda()
    k, v = randn((n, 3, dim), 601, BF).cuda(), randn((n, 3, dim), 602, BF).cuda()
    table, pos = tg.RotaryTable.build(dim, 400), torch.arange(n).cuda()
    for c in (dense, cache):
        tg.cache_write(c, k, v, slots, table, pos)
    for a, b in zip(tg.cache_read(dense, slots), tg.cache_read(cache, slots)):
        assert torch.equal(a, b)
    tables = torch.tensor([[4, 0, 8, 2], [1, 5, 3, 7]], dtype=torch.int32).cuda()
    for queries in (1, 40):  # 4 and 160 query rows of a key head
        q = randn((2, queries, 12, dim), 603, BF).cuda()
        lengths = torch.tensor([120, 45], dtype=torch.int32).cuda()
        for prefix in (None, torch.tensor([6], dtype=torch.int32).cuda()):
            shared = dict(prefix=prefix, prefix_length=30) if prefix is not None else {}
            a = tg.cache_attention(q, dense, tables, lengths, return_lse=True, **shared)
            b = tg.cache_attention(q, cache, tables, lengths, return_lse=True, **shared)
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    for t, old, view in zip(big, before, (cache.k, cache.v, cache.k_scales, cache.v_scales)):
        view = view.view(torch.uint8) if view.dtype == E8 else view
        view.zero_()
        assert torch.equal(t.view(torch.uint8), old.view(torch.uint8))
    assert status() == 0
