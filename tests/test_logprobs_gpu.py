"""Log probabilities of given tokens on the GPU against 64 bits, their gradient against the formula and against differences."""
import numpy as np
import pytest

import cache_reference as ref
from helpers import pkg

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch


def ints(torch, x):
    return torch.from_numpy(np.asarray(x, np.int32)).cuda()


def logits_of(torch, rng, rows, cols, dtype, size=3.0, stride=0, offset=0):
    """A tensor with rows `stride` elements apart (0: together) and the float64 values that it holds."""
    td = torch.bfloat16 if dtype == "bf16" else torch.float32
    wide = torch.zeros((rows, max(stride, cols + offset)), dtype=td, device="cuda")
    x = wide[:, offset:offset + cols]
    x.copy_(torch.from_numpy((rng.standard_normal((rows, cols)) * size).astype(np.float32)))
    return x, x.to(torch.float64).cpu().numpy()


def check(torch, x, values, targets, scale, top):
    """An exponential of y = z - max has a relative error of about |y| 2^-23 (its argument's rounding) and 2^-22; in the sums these
    weigh as the probabilities do. logp adds the rounding of its two numbers."""
    p = pkg()
    logp, entropy, lse, ids, best = p.token_logprobs(x, ints(torch, targets), scale, top)
    assert p.sync_status() == 0
    w_logp, w_entropy, w_lse, w_ids, w_best = ref.logprobs(values, targets, scale, top)
    unit = 2.0 ** -20
    spread = 4 + np.log(values.shape[1])

    def near(got, want, tol):
        got = got.cpu().numpy().astype(np.float64)
        assert np.array_equal(np.isneginf(got), np.isneginf(want))
        fine = np.isfinite(want)
        assert (np.abs(got - want)[fine] <= np.broadcast_to(tol, want.shape)[fine]).all(), np.abs(got - want)[fine].max()

    at = np.abs(np.where(np.isfinite(w_lse), w_lse, 0.0))
    near(lse, w_lse, unit * (spread + at))
    near(logp, w_logp, unit * (spread + 2 * at + np.abs(np.where(np.isfinite(w_logp), w_logp, 0.0))))
    near(entropy, w_entropy, 4 * unit * spread)
    assert np.array_equal(ids.cpu().numpy(), w_ids)
    near(best, w_best, (unit * (spread + 2 * at))[:, None] + unit * np.abs(np.where(np.isfinite(w_best), w_best, 0.0)))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("rows,cols,top,stride,offset", [(1, 1, 1, 0, 0), (3, 2, 2, 0, 0), (2, 31, 31, 0, 0), (5, 33, 32, 0, 1), (7, 300, 20, 0, 0), (4, 1023, 5, 1032, 3),
                                                         (3, 8191, 32, 0, 0), (6, 50257, 20, 50304, 0), (2, 50257, 1, 0, 0), (700, 2053, 5, 0, 0),
                                                         (200, 50257, 20, 0, 0), (2, 106001, 7, 0, 2), (2, 151936, 20, 0, 0), (1, 460001, 32, 0, 1), (2, 999999, 3, 0, 0)])
def test_against_64_bits(torch, dtype, rows, cols, top, stride, offset):
    rng = np.random.RandomState(cols % 1000)
    x, values = logits_of(torch, rng, rows, cols, dtype, stride=stride, offset=offset)
    check(torch, x, values, rng.randint(0, cols, rows), 1.0, top)
    check(torch, x, values, rng.randint(0, cols, rows), 1 / 0.7, 0)


def test_equal_logits_come_in_the_order_of_their_index(torch):
    rng = np.random.RandomState(2)
    for cols in (40, 5000, 50257, 470003):
        for dtype in ("fp32", "bf16"):
            x, values = logits_of(torch, rng, 4, cols, dtype)
            x[0] = 1.5                                    # all equal
            x[1] = x[1].round()                           # many equal
            x[2, :] = -0.0
            x[2, ::3] = 0.0                               # equal too
            x[3] = -7.0
            x[3, cols // 2:cols // 2 + 20] = 4.0
            check(torch, x, x.to(torch.float64).cpu().numpy(), np.array([0, 1, 2, 3]), 0.5, 32)


def test_columns_that_cannot_come(torch):
    rng = np.random.RandomState(3)
    for cols in (35, 3001, 50257):
        x, _ = logits_of(torch, rng, 6, cols, "fp32")
        x[0] = float("-inf")                              # nothing can come
        x[1] = float("-inf")
        x[1, 17] = -2.0                                   # one can
        x[2, 1:] = float("-inf")
        x[3, cols // 3:] = float("-inf")                  # fewer than are asked for, in the small case
        x[4] = torch.finfo(torch.float32).min             # the type's lowest value everywhere: all alike
        x[5] = torch.finfo(torch.float32).min
        x[5, 5] = 3.0
        check(torch, x, x.to(torch.float64).cpu().numpy(), np.array([3, 17, 30, cols - 1, 7, 8]), 1.0, 20)


def test_rows_without_a_distribution_and_without_a_target(torch):
    p = pkg()
    rng = np.random.RandomState(4)
    for cols in (50, 50257):
        x, values = logits_of(torch, rng, 5, cols, "fp32")
        x[1, 20] = float("nan")
        x[2, 21] = float("inf")
        x[1, 10] = float("inf")
        logp, entropy, lse, ids, best = p.token_logprobs(x, ints(torch, [-1, 3, 4, cols, 2 ** 31 - 1]), 1.0, 3)
        assert p.sync_status() == 0
        assert logp[0] == 0 and logp[3] == 0 and logp[4] == 0
        for v in (logp, entropy, lse):
            assert torch.isnan(v[1:3]).all()
        assert torch.isnan(best[1:3]).all()
        assert ids[1, :2].tolist() == [20, 10] and ids[2, 0] == 21
        w = ref.logprobs(values[[0, 3, 4]], np.array([0, 0, 0]), 1.0, 3)
        assert np.abs(lse[[0, 3, 4]].cpu().numpy() - w[2]).max() < 1e-4 and np.array_equal(ids[[0, 3, 4]].cpu().numpy(), w[3])


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("rows,cols,stride,offset", [(1, 1, 0, 0), (3, 33, 0, 0), (4, 1023, 1032, 3), (5, 50257, 0, 0), (700, 515, 0, 0), (2, 200003, 0, 1), (40, 8192, 0, 0)])
def test_gradient_against_the_formula(torch, dtype, rows, cols, stride, offset):
    """p = exp(z - lse) has a relative error of (|z| + |lse| + 4) 2^-22; the gradient follows it; bf16 results are rounded to 8 bits."""
    p = pkg()
    rng = np.random.RandomState(cols % 997)
    x, values = logits_of(torch, rng, rows, cols, dtype, stride=stride, offset=offset)
    targets = rng.randint(0, cols, rows)
    if rows > 2:
        targets[1] = -1
    g, h = rng.standard_normal(rows), rng.standard_normal(rows)
    tg, th = (torch.from_numpy(v).to("cuda", torch.float32) for v in (g, h))
    g, h = tg.cpu().numpy().astype(np.float64), th.cpu().numpy().astype(np.float64)
    scale = 1 / 0.75
    logp, entropy, lse, _, _ = p.token_logprobs(x, ints(torch, targets), scale)
    wide = torch.full((rows, cols + 9), 5.0, dtype=x.dtype, device="cuda")
    for gg, hh, out in ((tg, th, None), (tg, None, wide[:, 4:4 + cols]), (None, th, None)):
        d = p.token_logprobs_backward(x, ints(torch, targets), lse, entropy, gg, hh, scale, d_logits=out)
        assert p.sync_status() == 0
        ng, nh = (g if gg is not None else 0 * g), (h if hh is not None else 0 * h)
        want = ref.logprobs_backward(values, targets, scale, ng, nh)
        w_lse = lse.cpu().numpy().astype(np.float64)[:, None]
        prob = np.exp(values * scale - w_lse)
        size = scale * prob * (np.abs(ng)[:, None] + np.abs(nh)[:, None] * (np.abs(values * scale - w_lse) + np.log(cols) + 4))
        tol = 2.0 ** -21 * (np.abs(values * scale) + np.abs(w_lse) + 4) * size + 2.0 ** -21 * np.abs(want) + 1e-30
        if dtype == "bf16":
            tol = tol + 2.0 ** -8 * np.abs(want)
        assert (np.abs(d.to(torch.float64).cpu().numpy() - want) <= tol).all()
    assert (wide[:, :4] == 5).all() and (wide[:, 4 + cols:] == 5).all()
    kept = x.clone()  # in place: d_logits may be the logits
    same = p.token_logprobs_backward(kept, ints(torch, targets), lse, entropy, tg, th, scale, d_logits=kept)
    assert same is kept and torch.equal(kept, p.token_logprobs_backward(x, ints(torch, targets), lse, entropy, tg, th, scale))


def test_gradient_against_differences(torch):
    """Central differences of the 64-bit function, step 1e-4: their error is of the order of 1e-8, the kernel's within 1e-6 of the gradient's size."""
    p = pkg()
    rng = np.random.RandomState(8)
    x, values = logits_of(torch, rng, 2, 23, "fp32", size=1.5)
    targets, g, h, scale = np.array([4, 19]), np.array([1.0, -0.5]), np.array([0.25, 2.0]), 1.25
    _, entropy, lse, _, _ = p.token_logprobs(x, ints(torch, targets), scale)
    got = p.token_logprobs_backward(x, ints(torch, targets), lse, entropy, torch.tensor(g, dtype=torch.float32, device="cuda"),
                                    torch.tensor(h, dtype=torch.float32, device="cuda"), scale).cpu().numpy()

    def objective(v):
        logp, entropy, _, _, _ = ref.logprobs(v, targets, scale, 0)
        return (g * logp + h * entropy).sum()

    for r in range(2):
        for c in range(23):
            up, down = values.copy(), values.copy()
            up[r, c] += 1e-4
            down[r, c] -= 1e-4
            assert abs((objective(up) - objective(down)) / 2e-4 - got[r, c]) < 2e-6


def test_gradient_where_columns_cannot_come(torch):
    p = pkg()
    rng = np.random.RandomState(9)
    x, _ = logits_of(torch, rng, 3, 5001, "fp32")
    x[0, 100:] = float("-inf")
    x[1] = float("-inf")
    targets = ints(torch, [5, 6, 7])
    one = torch.ones(3, device="cuda")
    logp, entropy, lse, _, _ = p.token_logprobs(x, targets)
    d = p.token_logprobs_backward(x, targets, lse, entropy, one, one)
    assert p.sync_status() == 0
    assert (d[0, 100:] == 0).all() and torch.isfinite(d[0]).all() and torch.isfinite(d[2]).all()
    want = ref.logprobs_backward(x[:1, :100].to(torch.float64).cpu().numpy(), np.array([5]), 1.0, np.ones(1), np.ones(1))
    assert np.abs(d[0, :100].cpu().numpy() - want[0]).max() < 1e-5


def test_the_same_bits_every_time_and_on_another_stream(torch):
    p = pkg()
    rng = np.random.RandomState(10)
    x, _ = logits_of(torch, rng, 9, 50257, "fp32")
    targets = ints(torch, rng.randint(0, 50257, 9))
    first = p.token_logprobs(x, targets, 1.0, 20)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = p.token_logprobs(x, targets, 1.0, 20)
    side.synchronize()
    assert p.sync_status() == 0
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_refusals(torch):
    p = pkg()
    x, t = torch.zeros((3, 40), device="cuda"), ints(torch, [0, 1, 2])
    f = torch.zeros(3, device="cuda")
    p.token_logprobs(x, t, 1.0, 32)
    p.token_logprobs(x[:0], t[:0], 1.0, 4)
    for a in ((x.double(), t), (x.cpu(), t), (x[0], t), (x, t.long()), (x, t[:2]), (x.t(), t), (x, t, 0.0), (x, t, -1.0), (x, t, float("nan")), (x, t, float("inf")),
              (x, t, 1.0, 33), (x, t, 1.0, -1), (x[:, :10], t, 1.0, 11), (x[:, :0], t)):
        with pytest.raises(p.AttentionError):
            p.token_logprobs(*a)
    with pytest.raises(p.AttentionError):
        p.token_logprobs(x, t, logp=f[:2])
    with pytest.raises(p.AttentionError):
        p.token_logprobs(x, t, 1.0, 2, top_ids=t)
    for a, kw in (((x, t, f[:1], f, f), {}), ((x, t, f, f, f.double()), {}), ((x, t, f, f, f), {"d_logits": x.bfloat16()}),
                  ((x, t, f, f, f), {"d_logits": x[:, :20]}), ((x, t, f, f, f), {"scale": 0.0})):
        with pytest.raises(p.AttentionError):
            p.token_logprobs_backward(*a, **kw)
    assert p.lib().df_attn_last_status() != p.DF_OK and p.sync_status() == 0
