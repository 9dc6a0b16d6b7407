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


def many(parts, ring):
    """k_cache_attention_many over parts of n stages, `ring` stages of codes. Four widening warps do the same: two stand for them; a row role for the even stages and one for
    the odd ones."""
    load, mma, widen, rows = Role(), Role(), [Role(), Role()], [Role(), Role()]
    at = 0
    for n_part, n in enumerate(parts):
        for role in rows:
            role.mark("q written", n_part)
            role.arrive("Q_FULL")
        mma.wait("Q_FULL", n_part)

        def scores(j):
            mma.wait("K_FULL%d" % (j % 2), j // 2)
            if j >= 2:
                mma.wait("S_FREE%d" % (j % 2), j // 2 - 1)
            mma.mark("scores", j)
            mma.arrive("S_FULL%d" % (j % 2))
            mma.arrive("K_FREE%d" % (j % 2))

        for j in range(at, at + min(n, 2)):
            scores(j)
        for i in range(n):
            j = at + i
            if i + 2 < n:
                scores(j + 2)
            mma.wait("V_FULL%d" % (j % 2), j // 2)
            mma.wait("P_FULL%d" % (j % 2), j // 2)
            if i == 0 and n_part:
                mma.wait("O_FREE", n_part - 1)
            mma.mark("product", j)
            if i == 0:
                mma.mark("output begun", n_part)
            mma.arrive("PV_DONE%d" % (j % 2))

        def keys(role, j):
            role.wait("FULL%d" % (j % ring), j // ring)
            if j >= 2:
                role.wait("K_FREE%d" % (j % 2), j // 2 - 1)
            role.mark("scale written", j)
            role.arrive("K_FULL%d" % (j % 2))

        for role in widen:
            for j in range(at, at + min(n, 2)):
                keys(role, j)
            for j in range(at, at + n):
                if j + 2 < at + n:
                    keys(role, j + 2)
                if j >= 2:
                    role.wait("PV_DONE%d" % (j % 2), j // 2 - 1)
                role.mark("codes read", j)
                role.arrive("V_FULL%d" % (j % 2))
                role.arrive("EMPTY%d" % (j % ring))
        for j in range(at, at + n):
            b, use, slot = j % 2, j // 2, j % ring
            if j >= ring:
                load.wait("EMPTY%d" % slot, j // ring - 1)
            load.mark("codes", j)
            load.arrive("FULL%d" % slot)
            role = rows[b]  # even stages, odd stages
            role.wait("S_FULL%d" % b, use)
            role.mark("scale read", j)
            role.arrive("S_FREE%d" % b)
            if use:
                role.wait("PV_DONE%d" % b, use - 1)
            role.mark("weights written", j)
            role.arrive("P_FULL%d" % b)
        at += n
        for b, role in enumerate(rows):
            last = at - 1 - (at - 1 - b) % 2
            if last >= at - n:
                role.wait("PV_DONE%d" % b, last // 2)
            role.arrive("ROWS")
            role.wait("ROWS", n_part)
            role.mark("output read", n_part)
            role.arrive("O_FREE")
    return {"load": load, "mma": mma, **{"widen %d" % i: r for i, r in enumerate(widen)}, **{"rows %d" % i: r for i, r in enumerate(rows)}}


@pytest.mark.parametrize("parts", [[1], [2], [7], [1, 1, 1], [3, 1, 4, 2], [10, 9]])
@pytest.mark.parametrize("stages", [4, 8])
def test_every_wait_of_the_many_row_kernel_sees_its_phase(parts, stages):
    roles = many(parts, stages)
    assert phases_missed(roles) == [] and phases_early(roles) == set()
    assert out_of_order(roles, "scale written", "scale read") == set()
    assert out_of_order(roles, "scale read", "scale written", 4) == set()          # four places
    assert out_of_order(roles, "codes read", "codes", stages) == set()
    assert out_of_order(roles, "product", "weights written", 2) == set()           # two buffers of weights
    assert out_of_order(roles, "weights written", "product") == set()
    assert out_of_order(roles, "output read", "output begun", 1) == set()


@pytest.mark.parametrize("source", [SOURCE, SOURCE.replace(".cu", "_many.cu")])
def test_whole_warps_wait_as_warps(source):
    with open(source) as f:
        src = f.read()
    assert "mbar_wait_warp" in src and lone_waits(src) == []
