"""bench.timed_steps: when a cooperative timeout is measured again, when it ends the run, and what is reported (no GPU: the runtime, the
process group and the checks are stand-ins)."""
import os
import sys
from types import SimpleNamespace as S

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
import bench  # noqa: E402


class Timeout(Exception):
    pass


def _run(world, shared, late, other=0):
    """`late`: outcomes of the checks, one per attempt; `other`: the attempts in which the other rank is late."""
    seen = S(steps=0, falls=0, checks=0, polls=[], reduced=0)

    def check(device):
        seen.checks += 1
        if late[seen.checks - 1]:
            raise Timeout()

    def step():
        seen.steps += 1
        seen.polls.append(ops.COOP_POLL_RAISES)
        return 0.5

    def all_reduce(t, op):
        seen.reduced += 1
        if t.dtype == torch.int32 and seen.checks <= other:
            t.fill_(1)
    ops = S(COOP_POLL_RAISES=True, CoopTimeout=Timeout, _COOP_MSG="late", coop_check=check,
            coop_fall_back=lambda device: setattr(seen, "falls", seen.falls + 1))
    dist = S(get_backend=lambda: "gloo", barrier=lambda: None, all_reduce=all_reduce, ReduceOp=S(MAX=0))
    fake = S(tensor=torch.tensor, float64=torch.float64, int32=torch.int32, cuda=S(synchronize=lambda: None))
    timer = S(reset=lambda steps, warmup: None)
    try:
        got = bench.timed_steps(fake, dist, ops, timer, step, 3, 2, world, shared, "cpu")
    except Timeout:
        got = None
    assert ops.COOP_POLL_RAISES is True                 # as it was found, whatever happened
    return got, seen


@pytest.mark.parametrize("world", [1, 8])
def test_a_rank_with_a_gpu_of_its_own_is_measured_once(world):
    got, seen = _run(world, False, [0])
    assert got[1:] == (0.5, 0) and got[0] > 0 and seen.steps == 5 and all(seen.polls)
    got, seen = _run(world, False, [1, 0])
    assert got is None and seen.falls == 0 and seen.steps == 5


def test_ranks_that_share_a_gpu_fall_back_together():
    assert _run(2, True, [0])[0][2] == 0
    for late, other in (([1, 0], 0), ([0, 0], 1)):      # this rank, or the other one
        got, seen = _run(2, True, late, other)
        assert got[2] == 1 and seen.falls == 1 and seen.steps == 10 and not any(seen.polls)
    got, seen = _run(2, True, [1, 1, 0])
    assert got[2] == 2 and seen.falls == 2
    got, seen = _run(2, True, [1, 1, 1])
    assert got is None and seen.falls == 2
