"""``ScaledOps`` over ranks: the shards of a stack of 8-bit activations, every rank in a thread of its own on one GPU (no kernel
waits for another rank's; the partial sums meet on the host). Each step of each rank against its formula."""

import dataclasses
import threading

import pytest
import torch

from tests.stack_helpers import CONFIGS, initial_h
from test_gpu_stack_scaled import Checked
from tinygrad_dx12_b200 import stack as S

pytestmark = pytest.mark.gpu
FP4 = CONFIGS["fp4"]
FP6 = dataclasses.replace(FP4, fmt="fp6_e3m2")


class Meeting:
    """Adds the ranks' partial sums in the order of the ranks."""

    def __init__(self, world):
        self.barrier, self.parts = threading.Barrier(world, timeout=120), [None] * world

    def all_reduce(self, rank, t):
        self.parts[rank] = t.clone()
        self.barrier.wait()
        total = torch.stack(self.parts).sum(0)
        self.barrier.wait()
        t.copy_(total)


class Shared(Checked):
    def __init__(self, rank, meeting):
        super().__init__()
        self.rank, self.meeting = rank, meeting

    def all_reduce(self, t):
        assert t.dtype == torch.float32
        self.meeting.all_reduce(self.rank, t)


def over_ranks(cfg, world, h):
    meeting, out, failed = Meeting(world), [None] * world, []

    def run(rank):
        try:
            out[rank] = S.TPStack(cfg, rank, world, device="cuda", ops=Shared(rank, meeting)).forward(h.clone())
        except BaseException as e:  # noqa: BLE001
            failed.append(e)
            meeting.barrier.abort()

    threads = [threading.Thread(target=run, args=(r,)) for r in range(world)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for e in failed:
        if not isinstance(e, threading.BrokenBarrierError):
            raise e
    assert not failed
    return out


# K of a rank's o / down shard: 128 / 256 (tensor cores), 64 / 128 and 128 / 352 (the general kernel for one of them)
@pytest.mark.parametrize("cfg,world", [(FP4, 2), (FP4, 4), (FP6, 2), (dataclasses.replace(FP4, inter=704), 2)])
@pytest.mark.parametrize("m", [1, 33])
def test_every_step_of_every_rank(cfg, world, m):
    h = initial_h(cfg, m).cuda()
    ys = over_ranks(cfg, world, h)
    for y in ys[1:]:
        assert torch.equal(y, ys[0])
    # against the stack that is not split: the same blocks are quantised, from sums in another order, so codes on a border
    # turn; no more than the roundings themselves, 0.026 of a value in the mean square, three products a layer, two layers
    whole = S.TPStack(cfg, device="cuda", ops=S.ScaledOps()).forward(h.clone())
    assert float((ys[0].float() - whole.float()).norm() / whole.float().norm()) < 0.026 * 6


def test_shards_off_the_blocks_are_refused():
    with pytest.raises(ValueError, match="scale block"):
        S.TPStack(dataclasses.replace(FP4, inter=96), 0, 2, device="cuda", ops=S.ScaledOps())
