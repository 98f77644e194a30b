"""Recorded steps own the memory that their kernels leave partial results in: two recordings of one stream,
replayed on two streams at once beside eager calls on the stream that recorded them, give each the bits of an
eager call; steps that are gone give their memory back to later ones; a capture needs no call before it."""

from __future__ import annotations

import gc
import threading

import numpy as np
import pytest
import torch

import tinygrad_dx12_b200 as tg
from oracle import packed_ref
from tests.helpers import to_device
from tests.test_gpu_cache import Case
from tinygrad_dx12_b200.linalg import _packed_linear

pytestmark = pytest.mark.gpu

# lengths, queries, prefix: few rows cut over many CTAs, many rows, a prefix of few and of many rows
KINDS = {"few": ([20000, 1, 333], 1, 0), "many": ([3000, 90], 75, 0), "one tile": ([6000], 20, 0),
         "prefix": ([400, 70, 900], 1, 5000), "prefix of many": ([300] * 40, 1, 3000)}


# packed products whose tiles several CTAs share: rows, columns, tokens, path
PRODUCTS = {"split K": (4096, 4096, 8, "gemv"), "shared tiles": (9600, 1024, 1, "mx"), "shared tiles, 16 tokens": (8192, 2048, 16, "mx")}


def call(kind, seed):
    """A step over its own operands, and the eager result."""
    if kind in PRODUCTS:
        rows, cols, m, path = PRODUCTS[kind]
        w = to_device(packed_ref.make_packed(np.random.default_rng(seed), "fp4_e2m1", rows, cols, 32, "e8m0"), "cuda:0", "e8m0")
        x = torch.randn((m, cols), generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).cuda()

        def product():
            y = _packed_linear(w, x, torch.float32, path)
            for _ in range(3):
                y = torch.maximum(y, _packed_linear(w, x, torch.float32, path))
            return y

        return product, product()
    lengths, queries, prefix = KINDS[kind]
    c = Case(lengths, queries=queries, heads=8, kv=2, fmt="int8", page=64, prefix=prefix, seed=seed)
    q, tables = c.q.cuda(), c.tables.to(torch.int32).cuda()
    n = torch.tensor(lengths, dtype=torch.int32).cuda()
    shared = dict(prefix=c.prefix.to(torch.int32).cuda(), prefix_length=prefix) if prefix else {}

    def step():
        return tg.cache_attention(q, c.cache, tables, n, **shared)

    return step, step()


def record(step, stream):
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        out = step()
    return graph, out


@pytest.mark.parametrize("kind", [*KINDS, *PRODUCTS])
def test_recordings_of_one_stream_replayed_at_once(kind):
    (a, want_a), (b, want_b), (c, want_c) = call(kind, 400), call(kind, 410), call(kind, 420)
    side, one, two = (torch.cuda.Stream() for _ in range(3))
    assert len({side.cuda_stream, one.cuda_stream, two.cuda_stream}) == 3
    (ga, out_a), (gb, out_b) = record(a, side), record(b, side)
    torch.cuda.synchronize()
    for _ in range(20):
        out_a.zero_(), out_b.zero_()
        torch.cuda.synchronize()
        eager = []
        for _ in range(5):
            with torch.cuda.stream(one):
                ga.replay()
            with torch.cuda.stream(two):
                gb.replay()
            with torch.cuda.stream(side):
                eager.append(c())
        torch.cuda.synchronize()
        assert torch.equal(out_a, want_a) and torch.equal(out_b, want_b)
        assert all(torch.equal(e, want_c) for e in eager)


def test_steps_give_their_memory_back():
    run, want = call("many", 430)  # 38 MiB a recording
    x = torch.zeros(1, device="cuda")

    def step():
        return tg.GraphStep(lambda _: run(), x)

    def free():
        gc.collect()
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        return torch.cuda.mem_get_info()[0]

    for _ in range(40):  # every stream of torch's pool has its workspace for direct calls
        step()
    kept = step()
    before = free()
    for _ in range(30):
        other = step()
        assert torch.equal(other(), want)
        del other
    assert before - free() < 200 << 20  # 30 blocks would be 1.1 GiB
    kept.outputs.zero_()
    assert torch.equal(kept(), want)
    with pytest.raises(RuntimeError, match="on purpose"):  # a recording that fails gives its memory back, too
        tg.GraphStep(lambda _: failing(run), x)
    assert torch.equal(step()(), want) and torch.equal(kept(), want)


def failing(run):
    run()
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("on purpose")


@pytest.mark.parametrize("kind", list(PRODUCTS))
def test_first_products_captured(kind):
    """The kernel and the bits of a direct call."""
    step, want = call(kind, 450)
    graph, out = record(step, torch.cuda.Stream())
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


@pytest.mark.parametrize("queries,heads", [(1, 8), (13, 10), (26, 10), (60, 10)])  # 4, 65, 130 and 300 rows of a key head
@pytest.mark.parametrize("prefix", [0, 500])
def test_first_calls_captured(queries, heads, prefix):
    c = Case([2000, queries, 0, 130], queries=queries, heads=heads, kv=2, fmt="fp8e4m3", page=64, prefix=prefix, seed=440)
    good, lse = c.run()
    q, t, n = c.q.cuda(), c.tables.to(torch.int32).cuda(), torch.tensor(c.lengths, dtype=torch.int32).cuda()
    shared = dict(prefix=c.prefix.to(torch.int32).cuda(), prefix_length=prefix) if prefix else {}
    graph, (out, out_lse) = record(lambda: tg.cache_attention(q, c.cache, t, n, return_lse=True, **shared), torch.cuda.Stream())
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, good) and torch.equal(out_lse, lse)
    c.check(out, out_lse)


@pytest.mark.parametrize("order", ["row", "column"])  # the lean decode call, and the general one
def test_recorded_host_operands(order):
    """Recorded steps with pinned host tokens own the buffers these are staged in: later calls on the recording's
    stream, larger ones too, leave them alone, and two recordings of one stream can be replayed at once."""
    w = to_device(packed_ref.make_packed(np.random.default_rng(460), "fp4_e2m1", 1024, 4096, 32, "e8m0"), "cuda:0", "e8m0")
    side, one, two = (torch.cuda.Stream() for _ in range(3))

    def token(seed, m=2):
        x = torch.randn((m, 4096), generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16)
        return x.pin_memory().t() if order == "row" else x.t().contiguous().pin_memory()

    def product(x):
        return tg.matmul(w, x, dtype=torch.bfloat16)

    a, b = token(461), token(462)
    want_a, want_b = product(a).clone(), product(b).clone()
    (ga, out_a), (gb, out_b) = record(lambda: product(a), side), record(lambda: product(b), side)
    with torch.cuda.stream(side):
        big = token(463, 40)
        want_big = product(big).clone()
        others = [torch.full((1 << 14,), 7.0, device="cuda", dtype=torch.bfloat16) for _ in range(64)]
    torch.cuda.synchronize()
    for _ in range(20):
        out_a.zero_(), out_b.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(one):
            ga.replay()
        with torch.cuda.stream(two):
            gb.replay()
        with torch.cuda.stream(side):
            got = product(big)
        torch.cuda.synchronize()
        assert torch.equal(out_a, want_a) and torch.equal(out_b, want_b) and torch.equal(got, want_big)
    assert all((t == 7).all() for t in others)


def test_streams_of_threads(monkeypatch):
    """The handle that stands for a stream of each thread's own: two threads at once, each with its workspace."""
    from tinygrad_dx12_b200 import attention

    per_thread = 2  # cudaStreamPerThread
    steps = [call("few", 470), call("few", 480)]
    monkeypatch.setattr(attention, "stream_ptr", lambda device: per_thread)
    torch.cuda.synchronize()
    start = threading.Barrier(2)
    got = [[], []]

    def work(i):
        torch.cuda.set_device(0)
        start.wait()
        got[i] += [steps[i][0]() for _ in range(40)]

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for outs, (_, want) in zip(got, steps):
        assert len(outs) == 40 and all(torch.equal(o, want) for o in outs)
