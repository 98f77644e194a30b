"""The projection stack with attention over its packed caches: against the same layers with plain
attention over what the caches hold, token by token and in one chunk, with a shared prefix, and as a
recorded step."""

from __future__ import annotations

import dataclasses
import math

import pytest
import torch

import tinygrad_dx12_b200 as tg
from tests import cache_helpers as ref
from tests.stack_helpers import SMALL_FP4, SMALL_INT4, initial_h
from tinygrad_dx12_b200 import stack as S

pytestmark = pytest.mark.gpu

PAGE = 16


def layout(batch, per, first=0):
    """Page tables of ``batch`` requests, in an order of their own, behind ``first`` shared pages."""
    order = torch.randperm(first + batch * per, generator=torch.Generator().manual_seed(5))
    return order[:first], order[first:].view(batch, per)


def step_of(tables, start, count, prefix=None, prefix_length=0):
    """``count`` new tokens of each request after ``start`` cached ones."""
    at = torch.arange(start, start + count)
    slots = tables[:, at // PAGE] * PAGE + at % PAGE
    positions = (prefix_length + at).expand(tables.shape[0], -1)
    lengths = torch.full((tables.shape[0],), start + count, dtype=torch.int32)
    i32 = lambda t: t.to(torch.int32).cuda()  # noqa: E731
    return S.StackStep(slots.reshape(-1).cuda(), positions.reshape(-1).cuda(), i32(tables), lengths.cuda(),
                       None if prefix is None else i32(prefix), prefix_length)


class PlainCache(S.StackCache):
    """attend() by the formulas: turned and quantised by the package's write, attended to in float64."""

    def attend(self, layer, qkv, q_rows, step):
        cache, d = self.layers[layer], self.head_dim
        rows = qkv.view(qkv.shape[0], -1, d)
        heads, kv = q_rows // d, cache.kv_heads
        q = tg.cache_write(cache, rows[:, heads:heads + kv], rows[:, heads + kv:], step.slots, self.table, step.positions,
                           q=rows[:, :heads])
        every = torch.arange(cache.pages * PAGE, device="cuda")
        k, v = (x.cpu().double() for x in tg.cache_read(cache, every, dtype=torch.float32))
        batch = step.lengths.shape[0]
        n = q.shape[0] // batch
        q = q.view(batch, n, heads, d).cpu()
        front = torch.zeros(0, dtype=torch.int64)
        if step.prefix is not None:
            i = torch.arange(step.prefix_length)
            front = step.prefix.cpu().long()[i // PAGE] * PAGE + i % PAGE
        out = torch.empty_like(q)
        for b in range(batch):
            length = int(step.lengths[b])
            i = torch.arange(length)
            at = torch.cat([front, step.tables[b].cpu().long()[i // PAGE] * PAGE + i % PAGE])
            ends = [len(front) + length - n + j + 1 for j in range(n)]
            r, _, _ = ref.attend(q[b].double(), k[at], v[at], 1 / math.sqrt(d), ends)
            out[b] = r.to(out.dtype)
        return out.view(qkv.shape[0], q_rows).cuda()


def caches(cfg, cls, **kw):
    table = tg.RotaryTable.build(64, 256)
    return cls(cfg, table, pages=40, page_size=PAGE, head_dim=64, **kw)


def close(a, b, act):
    """Two forward passes whose attention outputs agree to a rounding of the activations: h differs by
    roundings that the layers pass on, 2^-8 (bf16) or 2^-11 (fp16) each, six of them a layer and two layers."""
    unit = 2.0 ** -8 if act == torch.bfloat16 else 2.0 ** -11
    a, b = a.double(), b.double()
    return (a - b).norm() <= 12 * unit * b.norm()


@pytest.mark.parametrize("base,fmt,block,scale", [(SMALL_INT4, "int8", None, torch.bfloat16),
                                                  (SMALL_FP4, "fp4_e2m1", 32, torch.float8_e8m0fnu),
                                                  (SMALL_FP4, "fp8e4m3", None, torch.bfloat16)])
def test_decode_and_chunk(base, fmt, block, scale):
    cfg = dataclasses.replace(base, kv_dim=128)
    st = S.TPStack(cfg, device="cuda")
    kw = dict(format=fmt, block_size=block, scale_dtype=scale)
    real, plain, chunk = caches(cfg, S.StackCache, **kw), caches(cfg, PlainCache, **kw), caches(cfg, S.StackCache, **kw)
    _, tables = layout(2, 4)
    n = 21
    h0 = torch.stack([initial_h(cfg, n, 7), initial_h(cfg, n, 8)]).cuda()  # (batch, tokens, hidden)
    last = None
    for t in range(n):
        step = step_of(tables, t, 1)
        a = st.forward(h0[:, t].clone(), real, step)
        b = st.forward(h0[:, t].clone(), plain, step)
        assert close(a, b, cfg.act), t
        last = a
    whole = st.forward(h0.reshape(2 * n, -1).clone(), chunk, step_of(tables, 0, n)).view(2, n, -1)
    assert close(whole[:, -1], last, cfg.act)
    with pytest.raises(ValueError, match="go together"):
        st.forward(h0[:, 0].clone(), real)


def test_shared_prefix_and_recorded_step():
    cfg = dataclasses.replace(SMALL_INT4, kv_dim=128)
    st = S.TPStack(cfg, device="cuda")
    real, plain = caches(cfg, S.StackCache), caches(cfg, PlainCache)
    front, tables = layout(3, 4, first=3)
    n_front = 37
    prompt = initial_h(cfg, n_front, 9).cuda()
    for c in (real, plain):  # the prompt is one request whose pages the batch then shares
        st.forward(prompt.clone(), c, step_of(front[None], 0, n_front))
    h0 = initial_h(cfg, 3, 10).cuda()
    step = step_of(tables, 0, 1, front, n_front)
    a = st.forward(h0.clone(), real, step)
    assert close(a, st.forward(h0.clone(), plain, step), cfg.act)
    # the step as a graph over its own inputs, replayed for the next token
    record = tg.GraphStep(lambda h, slots, pos, lengths: st.forward(h.clone(), real, S.StackStep(
        slots, pos, step.tables, lengths, step.prefix, n_front)), h0, step.slots, step.positions, step.lengths)
    assert torch.equal(record(), a)
    h1, after = initial_h(cfg, 3, 11).cuda(), step_of(tables, 1, 1, front, n_front)
    out = record(h1, after.slots, after.positions, after.lengths).clone()
    assert close(out, st.forward(h1.clone(), plain, after), cfg.act)
