"""Orthogonalised updates at the ends of what they accept: norms near the smallest that fp32 has, and polynomials that take singular values above 2."""
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


def with_singular_values(torch, rows, cols, values):
    torch.manual_seed(rows + cols)
    k = len(values)
    q, r = (torch.linalg.qr(torch.randn(n, k, dtype=torch.float64, device="cuda"))[0] for n in (rows, cols))
    return (q * torch.tensor(values, dtype=torch.float64, device="cuda")) @ r.t()


@pytest.mark.parametrize("rows,cols", [(50, 70), (100, 700), (200, 300), (300, 200)])
def test_singular_values_above_2(torch, rows, cols):
    """3.2 s - 0.2 s^3 takes 0.8 to 2.46 and 0.1 to 0.32: s^2 is 6.0 and |b s^2| 1.2 in the second step, both below 15. Errors as in tests/test_muon_gpu.py: a step's products are off
    by 3 (|a| + |b| + |c|) 2^-19 |X|, here of norms up to 2.9, and what was off before grows by |f'| <= 3.2."""
    p = pkg()
    u = with_singular_values(torch, rows, cols, (0.8, 0.5, 0.3, 0.1)).float()
    x = u.double() / u.double().norm()
    want = polynomial(x if rows <= cols else x.t(), 2, 3.2, -0.2, 0.0)
    want = want if rows <= cols else want.t()
    o = p.orthogonalize(u, 2, (3.2, -0.2, 0.0), 0.0)
    assert p.sync_status() == 0
    assert float((o.double() - want).norm()) <= 3 * 3.4 * 2.0 ** -19 * (3.2 * 1.0 + 2.9 * 6.0) + 3.2 ** 2 * 2.0 ** -22 + 2.0 ** -24 * float(want.norm())


@pytest.mark.parametrize("rows,cols", [(50, 70), (100, 700), (200, 300), (300, 200)])
def test_factors_that_leave_their_range(torch, rows, cols):
    """7.9 s - 7 s^3 takes 0.5 to 3.08, of which |b s^2| is 66: more than the factors hold, although s is not above 3.8. With these values on the diagonal they are elements of the factors: the
    matrix comes out infinite or NaN there, not as some finite number, and no other is touched."""
    p = pkg()
    u = torch.zeros(2, rows, cols, device="cuda")
    for i in range(4):
        u[0, i, i] = 0.5
    u[1] = with_singular_values(torch, rows, cols, (1.0,)).float()  # 0.9, 2.0
    o = p.orthogonalize(u, 2, (7.9, -7.0, 0.0), 0.0)
    assert p.sync_status() == 0
    assert not bool(o[0].diagonal()[:4].isfinite().any())
    assert torch.equal(o[1], p.orthogonalize(u[1], 2, (7.9, -7.0, 0.0), 0.0)) and bool(o[1].isfinite().all())
