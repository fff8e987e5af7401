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


def scans_first():
    """Whether a block's rows are looked through before their warp lets the products have them."""
    text = source()
    copies = text[text.index("if (pt.tma) {"):]
    copies = copies[:copies.index("return;")]
    return copies.rindex("look_for_special(s)") < copies.index("mbar_arrive(bar)")


def overwritten_scans(scan_first, blocks):
    """Orders in which a warp copies into a stage whose rows another warp still looks through.  A warp's steps for a block:
    copy when the products are through with the stage's last block, then scan and arrive, or arrive and scan."""
    start, found = ((0, 0),) * WARPS + (0,), []        # (block, step) of each warp; blocks that the products are through with
    seen, todo = {start}, [start]
    while todo:
        state = todo.pop()
        warps, through = state[:WARPS], state[WARPS]
        arrived = [b + (step == 2 and not scan_first) for b, step in warps]     # blocks that each warp has arrived for
        ways = [warps + (through + 1,)] if through < min(arrived) else []
        for i, (b, step) in enumerate(warps):
            if b == blocks or (step == 0 and b >= STAGES and through <= b - STAGES):
                continue
            if step == 0:
                if any(x[0] <= b - STAGES for x in warps):
                    found.append(state)
                new = (b, 1)
            elif step == 1 and not scan_first:
                new = (b, 2)
            else:
                new = (b + 1, 0)
            ways.append(warps[:i] + (new,) + warps[i + 1:] + (through,))
        for s in ways:
            if s not in seen:
                seen.add(s)
                todo.append(s)
    return found


def test_no_stage_is_filled_while_it_is_looked_through():
    assert not overwritten_scans(scans_first(), 4)


def test_arriving_before_the_scan_is_not_enough():
    assert overwritten_scans(False, 4)
