"""Gradient of the loss from hidden states where an operand is near the smallest numbers of fp32: what undoes its scale must not lose bits on the way.

Tolerance. All logits are about 0, so |t| = |z - lse| is ln 600 = 6.4: a probability is off by (6.4 + 4) 2^-22 = 2.5e-6 of itself, operands and G by 3 * 2^-22, a contraction of up to 600 by
(16 + 5) 2^-23 = 2.5e-6: less than 2^-17 = 7.6e-6 of the magnitudes' sum in all. Results, and in few rows' calls x times grad and each of a sum's steps as well, may lie below 2^-126, where a
rounding is off by up to 2^-150: 2 rows + 2 of them."""
import pytest

from helpers import pkg
from test_linear_ce_gpu import case, check_loss

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch


@pytest.mark.parametrize("rows", [8, 130])
@pytest.mark.parametrize("small", ["x", "w"])
@pytest.mark.parametrize("scale", [0.7, 3e-3])
def test_operands_near_the_smallest_numbers(torch, rows, small, scale):
    p = pkg()
    x, w, targets = case(torch, 31, rows, 600, 200, "fp32")
    (x if small == "x" else w).mul_(2.0 ** -116)
    loss, lse = p.linear_cross_entropy(x, w, targets, scale)
    check_loss(torch, x, w, targets, scale, loss, lse)
    grad = torch.rand(rows, device="cuda") + 0.5
    d_x, d_w = p.linear_cross_entropy_backward(x, w, targets, lse, grad, scale)
    assert p.sync_status() == 0
    g = torch.exp(scale * (x.double() @ w.double().t()) - lse.double()[:, None])
    g[torch.arange(rows, device="cuda"), targets.long()] -= 1.0
    g *= scale * grad.double()[:, None]
    least = (2 * rows + 2) * 2.0 ** -150
    for got, a, b in ((d_x, g, w.double()), (d_w, g.t(), x.double())):
        assert bool(((got.double() - a @ b).abs() <= 2.0 ** -17 * (a.abs() @ b.abs()) + least).all())
