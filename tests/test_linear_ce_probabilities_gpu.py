"""Gradient of the loss from hidden states where probabilities are far from 1: columns that are unlikely in every row, and targets that are nearly certain.

Tolerances. G = p - onehot is held times 2^15, where fp16 has 11 bits down to 2^-14 and steps of 2^-24 below: one part (bf16 calls) is off by at most 2^-11 of G or 2^-40,
two parts (fp32), of which the second is held another 2^11 higher, by 2^-22 or 2^-51. fp32 operands likewise, with 2^-51 of the largest (2^14 times a scale at least). The rest as in
tests/test_linear_ce_gpu.py: logits (width / 16 + 2) 2^-23 (bf16) or (16 + width / 128) 2^-23 of the sum of their terms' magnitudes, an exponential of y (|y| + 4) 2^-22, contractions of n
(n / 16 + 2) 2^-23 or (16 + n / 128) 2^-23, results half a step of their type."""
import pytest

from helpers import pkg

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch


def products_cut(bf16, n):
    return (n / 16 + 2) * 2.0 ** -23 if bf16 else (16 + n / 128) * 2.0 ** -23


def unlikely_columns(torch, seed, rows, vocab, width, depths, dtype, alike=False):
    """Rows share a direction that the columns behind the first `vocab` have in reverse: their logits are about -depth; the others' are those of noise. alike: every row has as
    much of that direction, so that a column's probabilities are nearly the same in all rows and its row of the gradient consists of small ones only."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    u = r(width)
    u /= u.norm()
    x = r(rows, width)
    if alike:
        x -= (x @ u)[:, None] * u
    x = (x + 4.0 * u).to(dtype)
    w = r(vocab, width) * width ** -0.5
    far = 0.3 * r(len(depths), width) * width ** -0.5 - torch.tensor(depths, device="cuda")[:, None] / 4.0 * u
    targets = torch.randint(0, vocab, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    return x, torch.cat([w, far]).to(dtype), targets


@pytest.mark.parametrize("alike", [False, True])
@pytest.mark.parametrize("dtype,rows,vocab,width,depths", [
    ("fp32", 8, 700, 128, (12, 14, 16, 18)), ("fp32", 9, 700, 128, (12, 14, 16, 18)), ("fp32", 40, 700, 128, (12, 14, 16, 18)), ("fp32", 300, 1500, 200, (11, 13, 15, 17, 18)),
    ("bf16", 9, 700, 128, (4, 6, 9, 11)), ("bf16", 300, 1500, 200, (4, 6, 9, 11))])
def test_columns_that_are_unlikely_in_every_row(torch, dtype, rows, vocab, width, depths, alike):
    """Their rows of the weight's gradient, each against its own size: probabilities of about 1e-8 to 1e-11 (fp32), down to 1e-8 (bf16); where rows are not alike, of some
    powers of ten on either side."""
    p = pkg()
    bf16 = dtype == "bf16"
    x, w, targets = unlikely_columns(torch, rows, rows, vocab, width, depths, torch.bfloat16 if bf16 else torch.float32, alike)
    xd, wd = x.double(), w.double()
    z = xd @ wd.t()
    lse = torch.logsumexp(z, 1).float()
    grad = torch.rand(rows, device="cuda") + 0.5
    _, d_w = p.linear_cross_entropy_backward(x, w, targets, lse, grad, want_x=False)
    assert p.sync_status() == 0
    z, t = z[:, vocab:], (z - lse.double()[:, None])[:, vocab:]
    g = torch.exp(t)
    lowest, highest = float(g.min()), float(g.max())
    assert lowest < (1e-7 if bf16 else 2e-11) and highest > 2e-9
    fx = grad.double()[:, None] * xd
    want = g.t() @ fx
    e = products_cut(bf16, width) * (xd.abs() @ wd[vocab:].abs().t()) + (0.0 if bf16 else width * 2.0 ** -49 * float(xd.abs().max() * wd.abs().max()))
    dg = torch.expm1(e + (t.abs() + 4) * 2.0 ** -22) * g + torch.maximum(g * (2.0 ** -11 if bf16 else 2.0 ** -22), torch.full_like(g, 2.0 ** -40 if bf16 else 2.0 ** -51))
    more = (2.0 ** -11 if bf16 else 2.0 ** -22) + products_cut(bf16, rows) + 2.0 ** -22
    half = torch.finfo(x.dtype).eps / 2
    least = 2.0 ** -39 if bf16 else 2.0 ** -50  # of x times grad, relative to its largest
    tol = ((dg + more * (g + dg)).t() @ fx.abs() + (g + dg).sum(0)[:, None] * least * float(fx.abs().max())) * (1 + half) + 1.01 * half * want.abs()
    off = (d_w[vocab:].double() - want).abs()
    assert bool((off <= tol).all()), float((off / tol).max())
    # the tolerance itself is a small part of every row
    assert float((tol.norm(dim=1) / want.norm(dim=1)).max()) < (2.0 ** -4 if bf16 else 2.0 ** -8)


@pytest.mark.parametrize("rows,vocab,width,pull", [(75, 364, 256, 14.0), (600, 533, 768, 18.0), (40, 300, 1000, 16.0), (20, 9000, 2048, 20.0)])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("both", [True, False])
def test_targets_that_are_nearly_certain(torch, dtype, rows, vocab, width, pull, both):
    """1 - p of about 1e-4 and less: e^log p - 1 from a logit of terms of one sign. Its products are exact or rounded to 24 bits and added in double, log p is rounded once, and lse is the
    caller's: (2^-24) of log p, 2^-22 for expm1, and G's rounding. One of 16 rows has lse equal to the target's logit: a loss of 0, and no gradient at the target."""
    p = pkg()
    bf16 = dtype == "bf16"
    gen = torch.Generator(device="cuda")
    gen.manual_seed(rows)
    td = torch.bfloat16 if bf16 else torch.float32
    x, w = (torch.randn((n, width), generator=gen, device="cuda") for n in (rows, vocab))
    w = (w * width ** -0.5).to(td)
    targets = torch.randint(0, vocab, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    x = (x + pull * w[targets.long()].float()).to(td)
    xd, wd, at, row = x.double(), w.double(), targets.long(), torch.arange(rows, device="cuda")
    z = xd @ wd.t()
    lse = torch.logsumexp(z, 1).float()
    lse[::16] = z[row, at][::16].float()
    t = z - lse.double()[:, None]
    d_x, d_w = p.linear_cross_entropy_backward(x, w, targets, lse, torch.ones(rows, device="cuda"), want_weight=both)
    assert p.sync_status() == 0
    log_p = t[row, at].clamp(max=0.0)
    g = torch.exp(t.clamp(max=0.0))
    g[row, at] = torch.expm1(log_p)
    part, least = (2.0 ** -11, 2.0 ** -40) if bf16 else (2.0 ** -22, 2.0 ** -51)
    e = products_cut(bf16, width) * (xd.abs() @ wd.abs().t()) + (0.0 if bf16 else width * 2.0 ** -49 * float(xd.abs().max() * wd.abs().max()))
    dg = torch.expm1(e + (t.abs() + 4) * 2.0 ** -22) * g.abs()
    dg[row, at] = 2.0 ** -24 * t[row, at].abs() + 2.0 ** -50 * (xd * wd[at]).abs().sum(1) + 2.0 ** -22 * g[row, at].abs()
    dg += torch.maximum(g.abs() * part, torch.full_like(g, least))
    half = torch.finfo(td).eps / 2
    want = g @ wd
    tol = (dg + (products_cut(bf16, vocab) + part) * (g.abs() + dg)) @ wd.abs() + (g.abs() + dg).sum(1)[:, None] * 2.0 ** -38 * float(wd.abs().max())
    off = (d_x.double() - want).abs()
    assert bool((off <= tol * (1 + half) + 1.01 * half * want.abs()).all()), float((off / tol).max())
    if both:
        want = g.t() @ xd
        tol = (dg + (products_cut(bf16, rows) + part) * (g.abs() + dg)).t() @ xd.abs() + (g.abs() + dg).sum(0)[:, None] * 2.0 ** -38 * float(xd.abs().max())
        off = (d_w.double() - want).abs()
        assert bool((off <= tol * (1 + half) + 1.01 * half * want.abs()).all()), float((off / tol).max())
