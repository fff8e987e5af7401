"""How the copying warps of the tensor-core prefill kernel share their barriers: every order of their steps, on the CPU.

A barrier has a number of completed phases, arrivals missing in the running one and bytes outstanding; a wait with a parity
passes while the number of completed phases has the other parity.  The walk below takes every order of the warps' steps and of
the copies' arrivals, and finds the states in which somebody still waits and nothing can happen any more."""

import os
import re

import pytest

from conftest import REPO

WARPS, STAGES = 3, 2


def source():
    with open(os.path.join(REPO, "smaq_b200", "csrc", "prefill_tc.cu")) as f:
        return f.read()


def arrivals_of_v_part():
    loaders = int(re.search(r"PT_LOADERS = (\d+);", source()).group(1))
    assert loaders == 32 * WARPS
    count = re.search(r"mbar_init\(&bars\.v_part, ([^)]+)\)", source()).group(1)
    return {"1": 1, "PT_LOADERS / 32": loaders // 32}[count]


def stuck_states(arrivals, blocks):
    """States without a way on.  ``blocks``: for each neighbouring block whose rows are cleared, the boxes of each warp.

    A warp's steps for a block: wait until the block's stage is free (``v_empty``: all warps are through with the block
    STAGES before), arrive at ``v_part`` (the first warp announces all boxes; the others arrive only where the barrier counts
    them) and issue its boxes, wait for the block's phase."""
    start = ((0, 0),) * WARPS, (0, arrivals, 0), 0     # (block, step) of each warp; (phases, missing, bytes); copies in flight
    seen, todo, stuck = {start}, [start], []
    while todo:
        warps, (phases, missing, owed), flying = todo.pop()
        ways = []

        def settle(w, phases, missing, owed, flying):
            if missing == 0 and owed == 0:
                phases, missing = phases + 1, arrivals
            ways.append((w, (phases, missing, owed), flying))

        if flying:
            settle(warps, phases, missing, owed - 1, flying - 1)
        for i, (b, step) in enumerate(warps):
            def to(x):
                return warps[:i] + (x,) + warps[i + 1:]
            if b == len(blocks):
                continue
            if step == 0:
                if b < STAGES or all(x[0] > b - STAGES for x in warps):
                    ways.append((to((b, 1)), (phases, missing, owed), flying))
            elif step == 1:
                mine = blocks[b][i]
                if i == 0:
                    settle(to((b, 2)), phases, missing - 1, owed + sum(blocks[b]), flying + mine)
                else:
                    settle(to((b, 2)), phases, missing - (arrivals > 1), owed, flying + mine)
            elif phases % 2 != b % 2:
                ways.append((to((b + 1, 0)), (phases, missing, owed), flying))
        if not ways and any(b < len(blocks) for b, _ in warps):
            stuck.append(warps)
        for s in ways:
            if s not in seen:
                seen.add(s)
                todo.append(s)
    return stuck


PATTERNS = [[(1, 0, 0)] * 4, [(1, 1, 1), (1, 0, 0), (1, 1, 0)], [(0, 1, 0), (1, 0, 0), (0, 0, 1), (1, 0, 0)], [(0, 0, 0), (1, 0, 0), (0, 0, 0)], [(2, 1, 1)] * 3]


@pytest.mark.parametrize("blocks", PATTERNS)
def test_no_order_of_steps_leaves_a_warp_waiting(blocks):
    assert not stuck_states(arrivals_of_v_part(), blocks)


def test_one_arrival_a_phase_is_not_enough():
    """The walk finds what it looks for: with the first warp's arrival alone a late warp's phase comes round again."""
    assert stuck_states(1, [(1, 0, 0)] * 4)
