"""Waits that run out must end their kernel. Each bounded wait gives every thread its own answer, and threads
of one group may get different ones (one sees the abort flag, another the barrier's phase). So no thread may
leave a loop by its own answer where others go on to a barrier or to a warp-wide instruction that counts on
it. Read from the sources: a stalled wait cannot be staged on a GPU."""

import pathlib
import re

import pytest

CSRC = pathlib.Path(__file__).resolve().parent.parent / "tinygrad_dx12_b200" / "csrc"
SOURCES = sorted(CSRC.glob("*.cu"))
WAIT = re.compile(r"\bmbar_wait\w*\(")
GROUP_BARRIER = re.compile(r"\b(meet<|epi_sync\(|tmem_sync\(|consumer_sync<)")
LEAVES = re.compile(r"\b(break|return)\b")


def indent(line):
    return len(line) - len(line.lstrip())


def blocks_around(lines, i):
    """The lines that open the blocks around line i, the innermost first."""
    level, found = indent(lines[i]), []
    for j in range(i - 1, -1, -1):
        if lines[j].strip() and indent(lines[j]) < level:
            level = indent(lines[j])
            found.append(j)
    return found


def body(lines, i):
    """The lines of the block that line i opens."""
    out = []
    for line in lines[i + 1:]:
        if line.strip() and indent(line) <= indent(lines[i]):
            break
        out.append(line)
    return out


def own_answer(lines, i):
    """Whether line i leaves a loop on a wait's answer that is a thread's own."""
    line = lines[i].split("//")[0]
    if not LEAVES.search(line):
        return False
    if WAIT.search(line):
        return "__all_sync" not in line
    m = re.search(r"if \(!(\w+)\) (?:break|return)", line)
    if not m:
        return False
    for j in range(i - 1, max(0, i - 60), -1):  # how the flag came about, the last time before this line
        if re.search(rf"\b{m.group(1)} = ", lines[j]):
            text = " ".join(lines[j:j + 2])
            local = re.search(r"\bwait\(", text)  # a kernel's own wait(), the nearest before
            helper = [k for k in range(j) if "auto wait = " in lines[k]][-1:] if local else []
            agreed = "__all_sync" in text or any("__all_sync" in " ".join(lines[k:k + 3]) for k in helper)
            return bool(WAIT.search(text) or local) and not agreed
    return False


def offences(path):
    lines = path.read_text().splitlines()
    for i, line in enumerate(lines):
        if not own_answer(lines, i):
            continue
        around = blocks_around(lines, i)
        if any("lane == 0" in lines[j] or "threadIdx.x == 0" in lines[j] for j in around):
            continue  # one thread's loop
        if any(re.search(r"\bbool mbar_wait|\bauto wait = ", lines[j]) for j in around):
            continue  # the wait itself
        yield f"{path.name}:{i + 1}: {line.strip()}"


@pytest.mark.parametrize("path", SOURCES, ids=lambda p: p.name)
def test_no_thread_leaves_alone(path):
    assert not list(offences(path))


def test_what_is_in_flight_is_waited_for():
    """A CTA that gave up waits for its copies and products by time alone: a wait that also ends on the abort
    flag, which is up by then, would let it exit under them."""
    found, drains = [], 0
    for path in SOURCES:
        lines = path.read_text().splitlines()
        for i, line in enumerate(lines):
            if re.search(r"if \(\*abort_flag\) \{", line):
                found += [f"{path.name}: {x.strip()}" for x in body(lines, i) if WAIT.search(x)]
            if re.search(r"mbar_wait\w*\(&?(drain|done)\b(?!\[.*parts)", line):
                found.append(f"{path.name}:{i + 1}: {line.strip()}")
            drains += "mbar_drain(" in line
    assert not found and drains >= 11


def test_warps_agree_before_group_barriers():
    """In a loop with a barrier of several warps, nobody leaves on a warp's answer either: only on the barrier's."""
    found = []
    for path in SOURCES:
        lines = path.read_text().splitlines()
        for i, line in enumerate(lines):
            code = line.split("//")[0]
            if not re.match(r"\s*for \(.*\{$", code) or not GROUP_BARRIER.search(" ".join(body(lines, i))):
                continue
            if re.search(r"&& ok\b|&& alive\b", code):
                found.append(f"{path.name}:{i + 1}: {code.strip()}")
            for j, inner in enumerate(lines[i + 1:i + 1 + len(body(lines, i))], i + 1):
                if LEAVES.search(inner) and "meet<" not in inner and (WAIT.search(inner) or re.search(r"if \(!(ok|alive|got)\)", inner)):
                    found.append(f"{path.name}:{j + 1}: {inner.strip()}")
    assert not found
