"""Every unit of a paged attention call is merged by someone: the host launches the merge kernel
wherever the device may leave a unit to it (no GPU needed)."""
import random

import pytest

import paged_plan as plans
from paged_plan import AT_THE_BOUND, Call


@pytest.fixture(scope="module")
def lib():
    return plans.probe()


@pytest.mark.parametrize("call", AT_THE_BOUND, ids=str)
def test_units_at_the_bound_are_merged(lib, call):
    plan, _ = call.plan(lib)
    assert plan["split"] and not plan["chunk"]
    pieces = call.cuts(plan)
    left = call.left(plan, pieces)
    assert left  # what the case is for
    assert plan["combine"], f"nobody merges units {left}"


def test_no_unit_is_left_unmerged(lib):
    r = random.Random(5)
    planned = at_once = cut = 0
    for _ in range(6000):
        call = plans.draw(r)
        plan, _ = call.plan(lib)
        if plan["chunk"] or not plan["split"]:
            continue
        pieces = call.cuts(plan)
        assert len(pieces) == len(call.unit_rows(plan["rows"]))
        left = call.left(plan, pieces)
        assert plan["combine"] or not left, f"{call}: nobody merges units {left}"
        planned += plan["combine"]
        at_once += not plan["combine"]
        cut += bool(left)
    assert planned > 300 and at_once > 300 and cut > 100  # both sides are drawn


def test_the_merge_kernel_is_not_launched_needlessly(lib):
    """Far from the bound the launch is one kernel (the second costs about 2.5 us)."""
    for call in (Call(2, 7, 64, 16, [4097], [1], cu=False), Call(8, 4, 128, 64, [8192] * 32, [1] * 32, cu=False),
                 Call(8, 4, 128, 16, [7600, 20], [4, 4])):
        plan, _ = call.plan(lib)
        assert plan["split"] and not plan["combine"]
        assert not call.left(plan, call.cuts(plan))
