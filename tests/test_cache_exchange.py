"""What the two halves of the many-row attention kernel's row warps tell each other through shared memory, on the CPU: the maximum of each half of a query
row, then each half's state. Marks and roles by the model of test_barrier_phases."""
import os
import re

import pytest

from test_barrier_phases import Role, out_of_order, phases_early, phases_missed

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dark-forest_b200", "csrc", "cache_attention_many.cu")


def halves(parts):
    """Parts of n stages: half b of the row warps has the stages j with j % 2 == b, which come when both halves have written q."""
    mma, rows = Role(), [Role(), Role()]
    at = uses = 0
    for n_part, n in enumerate(parts):
        for b, role in enumerate(rows):
            if n:
                role.mark("maximum written", n_part)
                role.arrive("ROWS")
                role.wait("ROWS", uses)
                role.mark("maximum read", n_part)
                role.arrive("Q_FULL")
            for j in range(at, at + n):
                if j % 2 == b:
                    role.wait("S_FULL%d" % b, j // 2)
                    role.arrive("S_FREE%d" % b)
            role.mark("state written", n_part)
            role.arrive("ROWS")
            role.wait("ROWS", uses + (1 if n else 0))
            role.mark("state read", n_part)
            role.arrive("ROWS")
            role.wait("ROWS", uses + (2 if n else 1))
        if n:
            mma.wait("Q_FULL", sum(1 for m in parts[:n_part] if m))
            for j in range(at, at + n):
                if j >= 2:
                    mma.wait("S_FREE%d" % (j % 2), j // 2 - 1)
                mma.arrive("S_FULL%d" % (j % 2))
        at += n
        uses += 3 if n else 2
    return {"mma": mma, "rows 0": rows[0], "rows 1": rows[1]}


def kernel_text():
    with open(SOURCE) as f:
        return f.read()


@pytest.mark.parametrize("parts", [[1], [2], [1, 1, 1], [0, 1, 0, 3], [5, 1, 4]])
def test_what_a_half_reads_is_still_there(parts):
    roles = halves(parts)
    assert phases_missed(roles) == [] and phases_early(roles) == set()
    assert out_of_order(roles, "maximum written", "maximum read") == set()
    assert out_of_order(roles, "state written", "state read") == set()
    assert out_of_order(roles, "state read", "state written", 1) == set()
    assert out_of_order(roles, "maximum read", "maximum written", 1) == set()


def test_a_part_of_one_stage_needs_a_place_of_its_own_for_the_maximum():
    """The half without a stage goes on to its state while the other may still be ahead of reading its maximum, so the two must not share a place."""
    assert out_of_order(halves([1]), "maximum read", "state written") != set()
    assert out_of_order(halves([2]), "maximum read", "state written") == set()
    text = kernel_text()
    place, = re.findall(r"top = fmaxf\(top, (\w+)\[1 - b\]\S*\[row\]\)", text)
    stores = re.findall(r"\b%s\[b\]\S*\[row\] = (\w+);" % place, text)
    assert stores == ["top"], stores  # nothing else is ever written there
