"""A kernel that may start while the one in front still runs reads nothing of it before that one has ended: any
tensor may be what that one writes, weights among them. Read from the sources: a read too early shows only by chance."""

import pathlib
import re

import pytest

CSRC = pathlib.Path(__file__).resolve().parent.parent / "tinygrad_dx12_b200" / "csrc"
WAIT = re.compile(r'^  (asm volatile\("griddepcontrol\.wait;"|follow\(\);)')  # at the kernel's own level: unconditional
MEMORY = re.compile(r"tma_load|\b(p|rp\.a|ep)\.(x|xs|ws|ys|y|offsets|order|part|tickets|bias|residual|weight|total|indices|weights|logits|counts)\b"
                    r"|reinterpret_cast<const uint4 \*>\((x|src)|\b(offsets|order|codes|scales_|indices)\[")


def kernels(name):
    """(name, lines) of each kernel's body."""
    lines = (CSRC / name).read_text().splitlines()
    for i, line in enumerate(lines):
        if line.startswith("__global__"):
            first = next(j for j in range(i, i + 6) if lines[j].endswith("{"))
            end = next(j for j in range(first, len(lines)) if lines[j] == "}")
            head = " ".join(lines[i:first + 1])
            yield re.search(r"(\w+)\((?:const|int|float|uint|void)", head.split("__launch_bounds__", 1)[-1].split(")", 1)[-1]).group(1), lines[first + 1:end]


@pytest.mark.parametrize("name", ["scaled_mma.cu", "scaled_rows.cu", "experts_route.cu"])
def test_nothing_is_read_before_the_wait(name):
    found = dict(kernels(name))
    assert found
    for kernel, body in found.items():
        waits = [i for i, line in enumerate(body) if WAIT.match(line)]
        assert len(waits) == 1, f"{kernel}: one wait that every thread comes to"
        early = [line.strip() for line in body[:waits[0]] if MEMORY.search(line.split("//")[0])]
        assert not early, f"{kernel}: {early}"
        assert not [line for line in body[waits[0] + 1:] if "griddepcontrol.wait" in line], kernel


def test_sources_are_read():
    names = [k for n in ("scaled_mma.cu", "scaled_rows.cu", "experts_route.cu") for k, _ in kernels(n)]
    for k in ("scaled_kernel", "gather_kernel", "norm_kernel", "values_kernel", "route_kernel", "plan_place_kernel", "combine_kernel"):
        assert k in names
