"""Plan and release of every size as a process's first calls: nothing of an earlier, larger call helps a later one."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CODE = """
import sys
sys.path.insert(0, {root!r})
from __graft_entry__ import load_package
import torch
p = load_package()
ints = lambda n, x: torch.full((n,), x, dtype=torch.int32, device="cuda")
for n in {sizes}:
    table = torch.arange(n, dtype=torch.int32, device="cuda")[:, None].contiguous()
    if {plan}:
        lens, starts, slots, positions, state = p.cache_plan(ints(n, 3), ints(n, 1), table, ints(n, 0), ints(1, n), 16, n)
        assert torch.equal(slots, table[:, 0] * 16 + 3) and state.tolist() == [n, 0] and lens.eq(4).all()
    else:
        free = ints(n, -1)
        lens, count = p.cache_release(ints(n, 5), ints(n, 1), table, free, ints(1, 0), 16)
        assert torch.equal(free, table[:, 0]) and count.item() == n and lens.eq(0).all()
    assert p.sync_status() == 0
print("done")
"""


@pytest.mark.parametrize("plan,sizes", [(True, [6079, 6080, 6144, 6145, 16384, 6144, 1025]), (False, [12160, 12161, 12288, 12289, 16384, 12288, 1025])])
def test_sizes_in_a_fresh_process(plan, sizes):
    import torch
    assert torch.cuda.is_available()
    got = subprocess.run([sys.executable, "-c", CODE.format(root=ROOT, sizes=sizes, plan=plan)], capture_output=True, text=True, timeout=300)
    assert got.returncode == 0 and got.stdout.strip() == "done", got.stderr[-2000:]
