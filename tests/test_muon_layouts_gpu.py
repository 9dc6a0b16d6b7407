"""Matrices to orthogonalise that lie row by row of all of them, as the heads' parts of a projection do: in, out and in place. Counts of steps."""
import pytest

from helpers import pkg

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("n,rows,cols", [(3, 40, 70), (4, 130, 64), (2, 300, 150), (5, 1, 33), (70, 20, 8)])
def test_row_by_row_of_all_matrices(torch, dtype, n, rows, cols):
    p = pkg()
    torch.manual_seed(n)
    u = torch.randn(n, rows, cols, device="cuda").to(torch.bfloat16 if dtype == "bf16" else torch.float32)
    want = p.orthogonalize(u)
    held = torch.full((rows + 1, n, cols + 4), 7.0, dtype=u.dtype, device="cuda")
    out = held[:rows, :, :cols].transpose(0, 1)
    assert p.orthogonalize(u, out=out) is out and torch.equal(out, want)
    out.copy_(u)
    assert torch.equal(p.orthogonalize(out, out=out), want)
    assert p.sync_status() == 0
    held[:rows, :, :cols] = 7.0
    assert bool((held == 7.0).all())


def test_results_that_would_overlap(torch):
    p = pkg()
    u = torch.randn(3, 6, 8, device="cuda")
    held = torch.zeros(1000, device="cuda")
    for strides in ((7, 24, 1), (8, 23, 1), (0, 24, 1), (40, 8, 1), (8, 8, 1)):
        with pytest.raises(p.AttentionError):
            p.orthogonalize(u, out=held.as_strided((3, 6, 8), strides))
    assert not held.any()


def test_steps_are_whole_numbers(torch):
    """Not what 32 bits leave of them, nor what lies in front of a decimal point."""
    p = pkg()
    u = torch.randn(6, 8, device="cuda")
    three = [[torch.randn(6, 8, device="cuda")] for _ in range(3)]
    kept = three[0][0].clone()
    for steps in (2 ** 32 + 5, 2 ** 64 + 5, -2 ** 64 + 5, -1, 0, 65, 2.5, float("inf"), float("nan")):
        with pytest.raises((p.AttentionError, TypeError, OverflowError)):
            p.orthogonalize(u, steps)
        with pytest.raises((p.AttentionError, TypeError, OverflowError)):
            p.muon_update(*three, 0.1, steps=steps)
    assert torch.equal(three[0][0], kept) and torch.equal(p.orthogonalize(u, torch.tensor(5)), p.orthogonalize(u, 5.0))
