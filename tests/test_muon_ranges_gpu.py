"""Orthogonalised updates at the ends of what they accept: norms near the smallest that fp32 has."""
import pytest

from helpers import pkg

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch


def polynomial(u, steps, a, b, c):
    for _ in range(steps):
        g = u @ u.transpose(-1, -2)
        u = a * u + (b * g + c * (g @ g)) @ u
    return u


@pytest.mark.parametrize("rows,cols", [(60, 90), (90, 60), (100, 700), (150, 260), (260, 150)])
@pytest.mark.parametrize("size", [1e-36, 1e-38, 1e-41, 3e37])
def test_norms_at_the_ends_of_fp32(torch, rows, cols, size):
    """eps = 0: the result does not depend on the update's size. The same update times a power of two has the same bits; and the bound of tests/test_muon_gpu.py, of what the
    update is after it has been rounded (values near 1e-41 are multiples of 2^-149)."""
    p = pkg()
    torch.manual_seed(rows)
    u = (torch.randn(2, rows, cols, device="cuda") + 2 * torch.randn(2, rows, 3, device="cuda") @ torch.randn(2, 3, cols, device="cuda")).clamp(-8, 8) * size
    assert bool(u.isfinite().all())
    o = p.orthogonalize(u, 5, eps=0.0)
    assert p.sync_status() == 0
    power = 2.0 ** 126 if size < 1 else 2.0 ** -100
    assert torch.equal(o, p.orthogonalize(u * power, 5, eps=0.0))
    x = u.double() / torch.linalg.matrix_norm(u.double(), keepdim=True)
    tall = rows > cols
    want = polynomial(x.transpose(1, 2) if tall else x, 5, 3.4445, -4.7750, 2.0315)
    want = want.transpose(1, 2) if tall else want
    side = min(rows, cols)
    bound = 37 * 2.0 ** -19 * side ** 0.5 * sum(3.4445 ** i for i in range(5)) / 4 + 3.4445 ** 5 * 2.0 ** -22 + 2.0 ** -24 * torch.linalg.matrix_norm(want)
    assert bool((torch.linalg.matrix_norm(o.double() - want) <= bound).all())
