"""The gradient of rows that nothing can come of (every logit -inf): no part of anything, so that a padded row does not poison what is added up over rows."""
import pytest

from helpers import pkg

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("cols", [1, 37, 5001])
@pytest.mark.parametrize("phase", [0, 1])
def test_gradient_of_rows_without_columns(dtype, cols, phase):
    import torch
    p = pkg()
    gen = torch.Generator(device="cuda")
    gen.manual_seed(cols)
    wide = torch.randn((5, cols + phase), generator=gen, device="cuda").to(getattr(torch, dtype))
    x = wide[:, phase:]
    x[1:4] = float("-inf")
    targets = torch.tensor([0, cols - 1, -1, cols, 0], dtype=torch.int32, device="cuda")
    g, h = torch.tensor([1.0, 2.0, 3.0, 0.0, 1.0], device="cuda"), torch.tensor([0.5, 1.0, -1.0, 0.0, 0.0], device="cuda")
    logp, entropy, lse, _, _ = p.token_logprobs(x, targets, 0.8)
    assert torch.isneginf(lse[1:4]).all() and (entropy[1:4] == 0).all() and torch.isneginf(logp[1]) and (logp[2:4] == 0).all()
    for gg, hh in ((g, h), (g, None), (None, h)):
        d = p.token_logprobs_backward(x, targets, lse, entropy, gg, hh, 0.8)
        assert p.sync_status() == 0
        assert (d[1:4] == 0).all()
        z = x[[0, 4]].double() * 0.8
        logs = z.log_softmax(1)
        prob, one = logs.exp(), torch.zeros_like(z)
        one[:, 0] = 1
        want = 0.8 * ((gg[[0, 4]].double()[:, None] if gg is not None else 0.0) * (one - prob)
                      - (hh[[0, 4]].double()[:, None] if hh is not None else 0.0) * prob * (logs - (prob * logs).sum(1, keepdim=True)))
        # as for other rows: p within (|z| + |lse| + 4) 2^-22 of itself, below 2^-17 here; bf16 results have 8 bits
        assert ((d[[0, 4]].double() - want).abs() <= want.abs() * (2.0 ** -8 if dtype == "bfloat16" else 0.0) + 2.0 ** -17 * 4 * (want.abs() + prob * 16)).all()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("cols", [1, 37, 5001])
def test_gradient_of_rows_of_the_lowest_value(dtype, cols):
    """Rows masked with the type's lowest value instead of -inf, all of them or all columns but one, at scales where the product with the scale is rounded:
    the logsumexp's own rounding is then larger than any exponent, but a probability is at most 1, so that a gradient is at most scale * (|g| + |h| * (log p +
    entropy)), and the row with one column left has a gradient of 0."""
    import torch
    p = pkg()
    kind = getattr(torch, dtype)
    x = torch.full((4, cols), torch.finfo(kind).min, dtype=kind, device="cuda")
    x[1, cols // 2] = 2.0
    x[2] *= 0.7
    x[3] = 1e30
    targets = torch.tensor([0, cols // 2, -1, cols - 1], dtype=torch.int32, device="cuda")
    g, h = torch.tensor([1.0, 2.0, 3.0, -1.0], device="cuda"), torch.tensor([0.5, 1.0, -1.0, 0.25], device="cuda")
    for scale in (1.0, 0.9, 0.7, 0.3):
        _, entropy, lse, _, _ = p.token_logprobs(x, targets, scale)
        d = p.token_logprobs_backward(x, targets, lse, entropy, g, h, scale).float()
        assert p.sync_status() == 0
        most = scale * (2 * g.abs() + h.abs() * (entropy.abs() + 1)) * (1 + 2.0 ** -7)
        assert (d.abs().amax(1) <= most).all(), (scale, d.abs().amax(1), most)
        assert d[1].abs().max() <= 2.0 ** -20 * scale * 3
