"""How the cache attention kernel waits, on the CPU: phases of its ring by the model of test_barrier_phases, and waits of whole warps by the rule of
test_kernel_waits."""
import os
import re

import pytest

from test_barrier_phases import Role, out_of_order, phases_early, phases_missed
from test_kernel_waits import lone_waits

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dark-forest_b200", "csrc", "cache_attention.cu")


def ring(parts, stages, pass_over=False):
    """k_cache_attention over parts of (row warps, number of stages): a loading warp and four computing ones. pass_over: a warp leaves out the stages
    that it takes no token of, and the others arrive for it."""
    load, compute = Role(), [Role() for _ in range(4)]
    at = 0
    for n, (weight, count) in enumerate(parts):
        for tile in range(count):
            slot, use = at % stages, at // stages
            if use:
                load.wait("EMPTY%d" % slot, use - 1)
            load.mark("scales written", at)
            load.arrive("FULL%d" % slot)
            for w, role in enumerate(compute):
                idle = weight == 1 and tile & 1 != w >> 1
                if idle and pass_over:
                    role.arrive("EMPTY%d" % slot)  # stands for the second arrival of a warp that has the stage
                    continue
                role.wait("FULL%d" % slot, use)
                if not idle:
                    role.mark("scales read", at)
                role.arrive("EMPTY%d" % slot)
            at += 1
        for role in compute:  # the barrier of the computing warps at the end of a part
            role.arrive("PART")
            role.wait("PART", n)
    return {"load": load, **{"compute %d" % w: role for w, role in enumerate(compute)}}


PARTS = [[(1, 1)], [(1, 9)], [(4, 7)], [(2, 3), (1, 8), (4, 5), (1, 0), (1, 2)], [(1, 5), (1, 6), (2, 4)]]


def stage_counts():
    with open(SOURCE) as f:
        text = f.read()
    return sorted({int(n) for n in re.findall(r"[?:] (\d+)\b(?! \?)", re.search(r"kStagesOf = (.*?);", text).group(1).replace("(", "").replace("kRows<MODE> == 8", "few"))})


@pytest.mark.parametrize("parts", PARTS)
def test_every_wait_sees_its_phase(parts):
    assert stage_counts() and min(stage_counts()) >= 2
    for stages in stage_counts():
        roles = ring(parts, stages)
        assert phases_missed(roles) == [] and phases_early(roles) == set()
        assert out_of_order(roles, "scales written", "scales read") == set()
        assert out_of_order(roles, "scales read", "scales written", stages) == set()


def test_a_warp_that_passes_over_stages_comes_early():
    roles = ring([(1, 9)], 3, pass_over=True)
    assert phases_early(roles) != set()


def test_whole_warps_wait_as_warps():
    with open(SOURCE) as f:
        src = f.read()
    assert "mbar_wait_warp" in src and lone_waits(src) == []
