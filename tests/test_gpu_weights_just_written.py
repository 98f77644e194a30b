"""Weights that the kernel in front writes, one that lets its followers start before it has ended: products read what it
wrote, eager and recorded."""

import pytest
import torch

import scaled_helpers as H

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tg():
    import tinygrad_dx12_b200 as tg

    return tg


def words(n, g):
    """Bytes that are finite, nonzero numbers of float16 two by two, which adding zero leaves as they are."""
    b = torch.randint(0, 256, (n // 2, 2), dtype=torch.uint8, device="cuda", generator=g)
    b[:, 0] |= 1
    b[:, 1] &= 0xEF
    return b.view(-1)


@pytest.mark.parametrize("rows,n,k", [(1, 20480, 4096), (40, 8192, 2048), (1, 512, 8192)])
@pytest.mark.parametrize("what", ["codes", "scales"])
def test_written_by_the_norm_before(tg, rows, n, k, what):
    g = H.generator(n + rows)
    x = tg.quantize(torch.randn((rows, k), device="cuda", generator=g))
    size = n * k // 2
    codes, scales = torch.empty(size, dtype=torch.uint8, device="cuda"), torch.full((n, k // 32), 122, dtype=torch.uint8, device="cuda")
    w = tg.PackedTensor(codes, "fp4_e2m1", (n, k), scales.view(torch.float8_e8m0fnu), 32)
    target = codes if what == "codes" else scales.view(-1)
    codes.copy_(words(size, g))
    into = target.view(torch.float16).view(-1, 512)
    zeros = torch.zeros_like(into)
    if what == "codes":
        sets = [words(size, g) for _ in range(2)]
    else:  # 118 to 123: exponents of float16 below its infinities
        sets = [torch.randint(118, 124, (n * k // 32,), dtype=torch.uint8, device="cuda", generator=g) for _ in range(2)]
    sources = [s.view(torch.float16).view(-1, 512) for s in sets]

    def step(source):
        tg.rms_norm(zeros, residual=source, total=into)  # the sum is what it writes
        return tg.scaled_linear(x, w, dtype=torch.float32)

    want = []
    for s in sets:
        target.copy_(s)
        torch.cuda.synchronize()
        want.append(tg.scaled_linear(x, w, dtype=torch.float32))
        torch.cuda.synchronize()
    assert not torch.equal(want[0], want[1])
    for i in range(10):
        got = step(sources[i % 2])
        assert torch.equal(got, want[i % 2])
    graph, out = torch.cuda.CUDAGraph(), []
    with torch.cuda.graph(graph):
        out = [step(sources[i % 2]) for i in range(4)]
    for _ in range(5):
        graph.replay()
    torch.cuda.synchronize()
    for i, got in enumerate(out):
        assert torch.equal(got, want[i % 2])
