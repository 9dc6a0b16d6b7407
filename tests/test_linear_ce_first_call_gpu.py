"""The loss from hidden states, its gradient and the optimiser step as a process's first calls of the library, inside a stream capture: nothing of theirs is left to a call before."""
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
p.lib()
torch.manual_seed(0)
dtype = torch.bfloat16 if {bf16} else torch.float32
x, w = torch.randn({rows}, 96, device="cuda").to(dtype), torch.randn(700, 96, device="cuda").to(dtype)
t = torch.randint(0, 700, ({rows},), device="cuda", dtype=torch.int32)
ps, ms, gs = ([torch.randn(*{shape}, device="cuda") for _ in range(2)] for _ in range(3))
ones = torch.ones({rows}, device="cuda")
torch.cuda.synchronize()
def step():
    loss, lse = p.linear_cross_entropy(x, w, t)
    d = p.linear_cross_entropy_backward(x, w, t, lse, ones)
    p.muon_update(ps, ms, gs, 0.1)
    return (loss, lse, *d)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = step()
held = [q.clone() for q in ps + ms]
graph.replay()
torch.cuda.synchronize()
assert p.sync_status() == 0
after = [q.clone() for q in ps + ms]
for q, h in zip(ps + ms, held):
    q.copy_(h)
want = step()
torch.cuda.synchronize()
assert p.sync_status() == 0
assert all(torch.equal(a, b) for a, b in zip(got, want)) and all(torch.equal(a, b) for a, b in zip(after, ps + ms))
assert not torch.equal(ps[0], held[0])
print("done")
"""


@pytest.mark.parametrize("rows,bf16,shape", [(200, False, (130, 200)), (200, True, (64, 96)), (5, False, (300, 60)), (3, True, (384, 384))])
def test_captured_in_a_fresh_process(rows, bf16, shape):
    import torch
    assert torch.cuda.is_available()
    got = subprocess.run([sys.executable, "-c", CODE.format(root=ROOT, rows=rows, bf16=bf16, shape=shape)], capture_output=True, text=True, timeout=300)
    assert got.returncode == 0 and got.stdout.strip() == "done", got.stderr[-2000:]
