"""Softmax cross entropy from hidden states on the GPU against 64 bits, and its gradient against the formula and against differences.

Tolerances. fp16 has 11 significant bits: the step at 1 is 2^-10, so a rounding to it is off by at most 2^-11 of the value; of a value held in two parts the first
leaves at most 2^-11 of it and the second 2^-11 of that, 2^-22. A logit is a sum of `width` products; s is the largest sum of their magnitudes. bf16 products are
exact; the tensor cores cut a sum off at each 16 of the contraction, by at most 2^-23 of what it has come to: (width / 16 + 2) 2^-23 s. fp32 operands are held in two
parts (or to 2^-39 of the largest of their row, or of the weight), the product of their low parts, 2^-22, is left out, sums are cut off 8 times and rounded every
128: (6 + 8 + 2 + width / 128) 2^-23 s.
An exponential of y adds (|y| + 4) 2^-22, a sum of 2^-22, logarithm and sum of two numbers 2^-22 of each.
G = p - onehot: a relative error of p as above, 2^-11 by its rounding to fp16 (bf16 calls) or 2^-22 (two parts), 2^-38 at least. A contraction of n adds, of the
magnitudes' sum, (n / 16 + 2) 2^-23 (bf16 calls) or (16 + n / 128) 2^-23; the result half a step of its type."""
import numpy as np
import pytest

from helpers import pkg

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch


def case(torch, seed, rows, vocab, width, dtype, padded=0.0, stride=0, offset=0, size=1.0):
    """x [rows, width], weight [vocab, width] (parts of wider tensors from `offset` on where stride is given), targets, all on the GPU."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    td = torch.bfloat16 if dtype == "bf16" else torch.float32

    def held(n):
        wide = torch.full((n, max(stride, width + offset)), float("nan"), dtype=td, device="cuda")
        x = wide[:, offset:offset + width]
        x.copy_(torch.randn((n, width), generator=gen, device="cuda") * size)
        return x

    x, w = held(rows), held(vocab)
    w *= width ** -0.5
    targets = torch.randint(0, vocab, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    if padded:
        targets[torch.rand((rows,), generator=gen, device="cuda") < padded] = -1
    return x, w, targets


def exact(torch, x, w, targets, scale):
    """z, lse, loss in 64 bits, and the error that the logits may have; rows without a target are 0."""
    xd, wd = x.double(), w.double()
    width = x.shape[1]
    there = (targets >= 0) & (targets < w.shape[0])
    xd = torch.where(there[:, None], xd, 0.0)
    z = scale * (xd @ wd.t())
    s = scale * float((xd.abs() @ wd.abs().t()).max())
    if x.dtype == torch.bfloat16:
        e = (width / 16 + 2) * 2.0 ** -23 * s
    else:
        e = (16 + width / 128) * 2.0 ** -23 * s + scale * width * 2.0 ** -38 * float(xd.abs().max() * wd.abs().max())
    lse = torch.logsumexp(z, 1)
    picked = z.gather(1, targets.long().clamp(0, w.shape[0] - 1)[:, None]).squeeze(1)
    zero = torch.zeros_like(lse)
    return z, torch.where(there, lse, zero), torch.where(there, lse - picked, zero), there, e


def check_loss(torch, x, w, targets, scale, loss, lse):
    z, w_lse, w_loss, there, e = exact(torch, x, w, targets, scale)
    tol = 2 * e + 2.0 ** -19 * 2 + 2.0 ** -22 * (z.abs().amax(1) + w_lse.abs() + np.log(w.shape[0]) + 4)
    assert bool(((lse.double() - w_lse).abs() <= tol).all()) and bool(((loss.double() - w_loss).abs() <= 2 * tol).all())
    assert bool((loss[~there] == 0).all()) and bool((lse[~there] == 0).all())


def check_gradient(torch, x, w, targets, lse, grad, scale, d_x, d_w):
    """Everything from the lse that was given."""
    z, _, _, there, e = exact(torch, x, w, targets, scale)
    bf16 = x.dtype == torch.bfloat16
    t = torch.where(there[:, None], z - lse.double()[:, None], float("-inf"))
    p = torch.exp(t).clamp(max=1.0)
    one = torch.zeros_like(p)
    at = torch.nonzero(there).squeeze(1)
    one[at, targets[at].long()] = 1.0
    g = p - one
    # p is e^t, at most 1, and what is computed e^t' with |t' - t| <= d: it lies between e^(t - d) and e^min(t + d, 0). Where d is small, either end is p d from p;
    # where logits are so large that their own rounding is above 1, the ends are 0 and 1.
    d = e + (t.abs().nan_to_num(posinf=0.0) + 4) * 2.0 ** -22
    ends = torch.maximum(torch.exp((t + d).clamp(max=0.0)) - p, p - torch.exp((t - d).clamp(max=0.0)))
    # What is off by a part of the product is so of the G that is computed, at most |g| + dg: |g' y' - g y| <= |g' - g| |y| + |g'| |y' - y|.
    dg = torch.where(there[:, None], ends, 0.0) + g.abs() * (2.0 ** -11 if bf16 else 2.0 ** -22) + 2.0 ** -38
    most = g.abs() + dg
    f = torch.where(there, scale * grad.double(), 0.0)
    xd, wd = torch.where(there[:, None], x.double(), 0.0), w.double()

    def cut(n):
        return (n / 16 + 2) * 2.0 ** -23 if bf16 else (16 + n / 128) * 2.0 ** -23

    half = torch.finfo(x.dtype).eps / 2
    vocab, rows = w.shape[0], x.shape[0]
    if d_x is not None:
        want = f[:, None] * (g @ wd)
        tol = f.abs()[:, None] * ((dg + (cut(vocab) + 2.0 ** -22) * most) @ wd.abs() + vocab * 2.0 ** -38 * float(wd.abs().max())) * (1 + half) + 1.01 * half * want.abs()
        off = (d_x.double() - want).abs()
        assert bool((off <= tol).all()), float((off - tol).max())
        assert bool((d_x[~there] == 0).all())
    if d_w is not None:
        fx = f[:, None] * xd
        want = g.t() @ fx
        # x times grad enters in fp16: 2^-11 of itself in bf16 calls, two parts in fp32 ones
        more = (2.0 ** -11 if bf16 else 2.0 ** -22) + cut(rows) + 2.0 ** -22
        tol = ((dg + more * most).t() @ fx.abs() + rows * 2.0 ** -38 * float(fx.abs().max() if rows else 0.0)) * (1 + half) + 1.01 * half * want.abs()
        off = (d_w.double() - want).abs()
        assert bool((off <= tol).all()), float((off - tol).max())


SHAPES = [(1, 1, 1), (1, 2, 7), (2, 31, 8), (3, 32, 63), (5, 33, 64), (127, 255, 65), (128, 256, 128), (129, 257, 129), (300, 1000, 330), (257, 129, 768), (40, 3001, 777), (64, 513, 1600),
          (9, 50257, 96), (700, 2053, 72), (4, 301, 515), (8, 9001, 130), (16, 777, 200), (17, 777, 200), (3, 12000, 770), (12, 400, 3300), (6, 300, 3300)]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("rows,vocab,width", SHAPES)
def test_against_64_bits(torch, dtype, rows, vocab, width):
    p = pkg()
    x, w, targets = case(torch, rows + vocab, rows, vocab, width, dtype, padded=0.2 if rows > 4 else 0.0)
    scale = 0.7 if rows % 2 else 1.0
    loss, lse = p.linear_cross_entropy(x, w, targets, scale)
    assert p.sync_status() == 0
    check_loss(torch, x, w, targets, scale, loss, lse)
    grad = torch.randn(rows, device="cuda") + 0.5
    d_x, d_w = p.linear_cross_entropy_backward(x, w, targets, lse, grad, scale)
    assert p.sync_status() == 0
    assert d_x.dtype == x.dtype and d_w.dtype == w.dtype
    check_gradient(torch, x, w, targets, lse, grad, scale, d_x, d_w)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("width,stride,offset", [(64, 72, 0), (64, 72, 8), (64, 70, 0), (63, 65, 1), (100, 104, 3), (8, 0, 1)])
def test_strides_and_alignment(torch, dtype, width, stride, offset):
    """Rows that lie apart, and that begin at any element; what lies between the rows of the results stays."""
    p = pkg()
    rows, vocab = 70, 500
    x, w, targets = case(torch, 7, rows, vocab, width, dtype, 0.1, stride, offset)
    loss, lse = p.linear_cross_entropy(x, w, targets)
    check_loss(torch, x, w, targets, 1.0, loss, lse)
    grad = torch.rand(rows, device="cuda")
    outs = [torch.full((n, max(stride, width + offset)), 7.0, dtype=x.dtype, device="cuda") for n in (rows, vocab)]
    views = [o[:, offset:offset + width] for o in outs]
    d_x, d_w = p.linear_cross_entropy_backward(x, w, targets, lse, grad, d_x=views[0], d_weight=views[1])
    assert p.sync_status() == 0 and d_x is views[0] and d_w is views[1]
    check_gradient(torch, x, w, targets, lse, grad, 1.0, d_x, d_w)
    for o in outs:
        o[:, offset:offset + width] = 7.0
        assert bool((o == 7.0).all())


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_rows_that_are_left_out(torch, dtype):
    """Targets outside the vocabulary, whatever their rows hold, and a batch of nothing else."""
    p = pkg()
    x, w, targets = case(torch, 3, 200, 400, 48, dtype)
    out = torch.tensor([0, 3, 64, 131, 199], device="cuda")
    targets[out] = torch.tensor([-1, 400, -2 ** 31, 2 ** 31 - 1, 1000], dtype=torch.int32, device="cuda")
    x[out] = torch.tensor([float("nan"), float("inf"), float("-inf"), 3e38, -3e38], device="cuda")[:, None].to(x.dtype)
    grad = torch.rand(200, device="cuda")
    grad[out] = torch.tensor([float("nan"), float("inf"), 1e30, -1.0, 0.0], device="cuda")
    loss, lse = p.linear_cross_entropy(x, w, targets)
    check_loss(torch, x, w, targets, 1.0, loss, lse)
    d_x, d_w = p.linear_cross_entropy_backward(x, w, targets, lse, grad)
    check_gradient(torch, x, w, targets, lse, grad, 1.0, d_x, d_w)
    targets.fill_(-1)
    loss, lse = p.linear_cross_entropy(x, w, targets)
    assert not loss.any() and not lse.any()
    d_x, d_w = p.linear_cross_entropy_backward(x, w, targets, lse, grad)
    assert p.sync_status() == 0 and not d_x.any() and not d_w.any()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_values_that_are_not_finite(torch, dtype):
    """A NaN or an infinity in a row makes that row's loss NaN and no other's; one in the weight every row's."""
    p = pkg()
    x, w, targets = case(torch, 4, 150, 300, 64, dtype)
    x[5, 3], x[130, 63] = float("nan"), float("inf")
    loss, lse = p.linear_cross_entropy(x, w, targets)
    bad = torch.zeros(150, dtype=torch.bool, device="cuda")
    bad[5] = bad[130] = True
    assert bool((loss.isnan() == bad).all()) and bool((lse[bad].isnan()).all())
    good = torch.nonzero(~bad).squeeze(1)
    check_loss(torch, x[good], w, targets[good], 1.0, loss[good], lse[good])
    d_x, d_w = p.linear_cross_entropy_backward(x, w, targets, lse, torch.ones(150, device="cuda"))
    assert bool((d_x.isnan().any(1) == bad).all()) and bool(d_w.isnan().all())
    x, w, targets = case(torch, 4, 150, 300, 64, dtype)
    w[7, 0] = float("nan")
    loss, lse = p.linear_cross_entropy(x, w, targets)
    assert bool(loss.isnan().all())
    assert p.sync_status() == 0


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("size", [30.0, 1e-4, 1e-20, 1e18])
def test_large_and_small(torch, dtype, size):
    """Logits of a few hundred (one column has all), nearly none, and operands whose scales leave fp16 far behind."""
    p = pkg()
    x, w, targets = case(torch, 5, 130, 700, 96, dtype, size=size)
    w *= min(1.0, 1e18 / size) if size > 1 else 1.0
    if size == 1e18:
        w *= 1e-18
    loss, lse = p.linear_cross_entropy(x, w, targets)
    assert p.sync_status() == 0
    check_loss(torch, x, w, targets, 1.0, loss, lse)
    grad = torch.rand(130, device="cuda") + 0.1
    d_x, d_w = p.linear_cross_entropy_backward(x, w, targets, lse, grad)
    check_gradient(torch, x, w, targets, lse, grad, 1.0, d_x, d_w)


def test_gradient_against_differences(torch):
    """The loss in 64 bits moved along random directions by h, against the gradient along them: the second difference bounds what h costs."""
    p = pkg()
    x, w, targets = case(torch, 6, 40, 90, 24, "fp32")
    grad = torch.rand(40, device="cuda") + 0.5
    _, lse = p.linear_cross_entropy(x, w, targets, 0.8)
    d_x, d_w = p.linear_cross_entropy_backward(x, w, targets, lse, grad, 0.8)

    def total(xd, wd):
        z = 0.8 * (xd @ wd.t())
        return float((grad.double() * (torch.logsumexp(z, 1) - z.gather(1, targets.long()[:, None]).squeeze(1))).sum())

    h = 1e-4
    for seed in range(4):
        torch.manual_seed(seed)
        a, b = torch.randn_like(x).double(), torch.randn_like(w).double()
        for u, v in ((a, 0 * b), (0 * a, b), (a, b)):
            up, mid, down = (total(x.double() + k * h * u, w.double() + k * h * v) for k in (1, 0, -1))
            along = float((d_x.double() * u).sum() + (d_w.double() * v).sum())
            # third differences are h^2 times the third derivative, here below 1e4; gradients below 1e-5 of their size off
            assert abs((up - down) / (2 * h) - along) <= 1e4 * h * h + 2e-5 * float((d_x.double() * u).abs().sum() + (d_w.double() * v).abs().sum()) + 1e-9 * abs(up + mid + down) / h


@pytest.mark.parametrize("dtype,rows,vocab,width", [("fp32", 4100, 20011, 40), ("bf16", 8200, 20011, 40), ("fp32", 33, 130001, 520)])
def test_several_pieces(torch, dtype, rows, vocab, width):
    """More than a piece of the vocabulary at a time is held, in both directions where the weight is cut into parts."""
    p = pkg()
    x, w, targets = case(torch, 8, rows, vocab, width, dtype, 0.1)
    targets[:4] = torch.tensor([0, vocab - 1, vocab // 2, 255], dtype=torch.int32)
    loss, lse = p.linear_cross_entropy(x, w, targets)
    check_loss(torch, x, w, targets, 1.0, loss, lse)
    grad = torch.rand(rows, device="cuda")
    d_x, d_w = p.linear_cross_entropy_backward(x, w, targets, lse, grad)
    assert p.sync_status() == 0
    check_gradient(torch, x, w, targets, lse, grad, 1.0, d_x, d_w)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_one_gradient_alone_and_the_same_bits(torch, dtype):
    p = pkg()
    x, w, targets = case(torch, 9, 600, 3000, 136, dtype, 0.1)
    loss, lse = p.linear_cross_entropy(x, w, targets)
    grad = torch.rand(600, device="cuda")
    both = p.linear_cross_entropy_backward(x, w, targets, lse, grad)
    size = p.linear_cross_entropy_workspace_bytes(600, 3000, 136, dtype == "bf16", True)
    for _ in range(3):
        dirty = torch.randint(0, 256, (size,), dtype=torch.uint8, device="cuda")  # a workspace may hold anything
        again = p.linear_cross_entropy(x, w, targets, workspace=dirty)
        assert torch.equal(again[0], loss) and torch.equal(again[1], lse)
        a = p.linear_cross_entropy_backward(x, w, targets, lse, grad, want_weight=False, workspace=dirty)
        b = p.linear_cross_entropy_backward(x, w, targets, lse, grad, want_x=False, workspace=dirty)
        assert a[1] is None and b[0] is None and torch.equal(a[0], both[0]) and torch.equal(b[1], both[1])
    assert p.linear_cross_entropy_backward(x, w, targets, lse, grad, want_x=False, want_weight=False) == (None, None)


def test_no_rows(torch):
    p = pkg()
    x, w, targets = case(torch, 1, 3, 20, 8, "fp32")
    loss, lse = p.linear_cross_entropy(x[:0], w, targets[:0])
    assert loss.shape == (0,) and lse.shape == (0,)
    d_x, d_w = p.linear_cross_entropy_backward(x[:0], w, targets[:0], lse, loss)
    assert d_x.shape == (0, 8) and not d_w.any()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_captured_and_replayed_with_other_inputs(torch, dtype):
    p = pkg()
    x, w, targets = case(torch, 10, 260, 900, 72, dtype, 0.2)
    grad = torch.rand(260, device="cuda")
    loss, lse = (torch.empty(260, device="cuda") for _ in range(2))
    d_x, d_w = torch.empty_like(x), torch.empty_like(w)
    ws = torch.empty(p.linear_cross_entropy_workspace_bytes(260, 900, 72, dtype == "bf16", True), dtype=torch.uint8, device="cuda")

    def step():
        p.linear_cross_entropy(x, w, targets, 1.0, loss, lse, ws)
        p.linear_cross_entropy_backward(x, w, targets, lse, grad, 1.0, d_x, d_w, workspace=ws)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in (11, 12):
        for a, b in zip((x, w, targets), case(torch, seed, 260, 900, 72, dtype, 0.3)):
            a.copy_(b)
        graph.replay()
        assert p.sync_status() == 0
        check_loss(torch, x, w, targets, 1.0, loss, lse)
        check_gradient(torch, x, w, targets, lse, grad, 1.0, d_x, d_w)


def test_two_streams(torch):
    """Calls that run at the same time, each with its own workspace; and a stream that is given by name, its workspace from the allocator."""
    p = pkg()
    streams = [torch.cuda.Stream() for _ in range(2)]
    cases = [case(torch, s, 512, 4000, 128, d) for s, d in ((20, "fp32"), (21, "bf16"))]
    want = [p.linear_cross_entropy(*c) for c in cases]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for s, c in zip(streams, cases):
            with torch.cuda.stream(s):
                loss, lse = p.linear_cross_entropy(*c)
                got.append((loss, lse, *p.linear_cross_entropy_backward(*c, lse, torch.ones_like(lse))))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert torch.equal(g[0], want[i % 2][0]) and torch.equal(g[1], want[i % 2][1])
        assert torch.equal(g[2], got[i % 2][2]) and torch.equal(g[3], got[i % 2][3])
    named = [p.linear_cross_entropy(*cases[0], stream=streams[0]) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(n[0], want[0][0]) for n in named) and p.sync_status() == 0


def test_refusals(torch):
    p = pkg()
    x, w, targets = case(torch, 2, 6, 20, 16, "fp32")
    loss, lse = p.linear_cross_entropy(x, w, targets)
    for call in (lambda: p.linear_cross_entropy(x.cpu(), w, targets), lambda: p.linear_cross_entropy(x, w.cpu(), targets), lambda: p.linear_cross_entropy(x, w, targets.long()),
                 lambda: p.linear_cross_entropy(x, w[:, :15], targets), lambda: p.linear_cross_entropy(x, w.bfloat16(), targets), lambda: p.linear_cross_entropy(x.half(), w.half(), targets),
                 lambda: p.linear_cross_entropy(x, w, targets[:5]), lambda: p.linear_cross_entropy(x.t(), w, targets), lambda: p.linear_cross_entropy(x[0], w, targets),
                 lambda: p.linear_cross_entropy(x, w, targets, 0.0), lambda: p.linear_cross_entropy(x, w, targets, loss=loss[:5]),
                 lambda: p.linear_cross_entropy(x, w, targets, loss=loss, lse=loss), lambda: p.linear_cross_entropy(x, w, targets, workspace=torch.empty(100, dtype=torch.uint8, device="cuda")),
                 lambda: p.linear_cross_entropy_backward(x, w, targets, lse[:5], lse), lambda: p.linear_cross_entropy_backward(x, w, targets, lse, lse.double()),
                 lambda: p.linear_cross_entropy_backward(x, w, targets, lse, lse, d_x=x), lambda: p.linear_cross_entropy_backward(x, w, targets, lse, lse, d_x=torch.empty_like(w))):
        with pytest.raises((p.AttentionError, ValueError, TypeError)):
            call()
    again = p.linear_cross_entropy(x, w, targets)
    assert torch.equal(again[0], loss) and p.sync_status() == 0


def test_pieces_of_a_weight_that_is_copied(torch):
    p = pkg()
    x, w, targets = case(torch, 77, 40, 70001, 2047, "bf16", padded=0.2, stride=2049, offset=1)  # 16-byte loads cannot start at its rows: 287 MB of copies
    assert p.linear_cross_entropy_workspace_bytes(40, 70001, 2047, True, False) < 280 << 20
    targets[:2] = torch.tensor([0, 70000], dtype=torch.int32, device="cuda")
    loss, lse = p.linear_cross_entropy(x, w, targets)
    check_loss(torch, x, w, targets, 1.0, loss, lse)


@pytest.mark.parametrize("rows,vocab,width", [(75, 364, 256), (600, 533, 768), (40, 300, 1000)])
def test_gradient_of_targets_of_high_probability(torch, rows, vocab, width):
    """p - 1 at the target. Its logit is a sum of terms of one sign, about 11 here: a product rounded to 24 bits and lanes' sums of width / 32 terms, then five more, are
    off by (width / 32 + 6) 2^-24 of it at most, scale and lse's difference by 2^-24 of their own size, and expm1 by 2^-22 of its result."""
    p = pkg()
    x, w, targets = case(torch, 5, rows, vocab, width, "fp32")
    x += 9.0 * w[targets.long()]
    z = x.double() @ w.double().t()
    lse = torch.logsumexp(z, 1).float()
    d_x, _ = p.linear_cross_entropy_backward(x, w, targets, lse, torch.ones(rows, device="cuda"), want_weight=False)
    picked = z.gather(1, targets.long()[:, None]).squeeze(1)
    g = torch.exp(z - lse.double()[:, None])
    g[torch.arange(rows, device="cuda"), targets.long()] = torch.expm1(picked - lse.double())
    want = g @ w.double()
    at_target = ((width / 32 + 6) * 2.0 ** -24 * (x.double() * w[targets.long()].double()).abs().sum(1) + 2.0 ** -24 * (picked.abs() + lse.double().abs())) \
        * torch.exp(picked - lse.double()) + 2.0 ** -22 * g.abs().max(1).values
    # the other logits, p each: sums cut off as in exact(), 22-bit operands
    e = (16 + width / 128) * 2.0 ** -23 * (x.double().abs() @ w.double().abs().t()) + width * 2.0 ** -38 * float(x.abs().max() * w.abs().max())
    others = torch.exp(z - lse.double()[:, None]) * (e + (z.abs() + lse.double().abs()[:, None] + 4) * 2.0 ** -22)
    others[torch.arange(rows, device="cuda"), targets.long()] = 0.0
    wide = w.double().abs()
    tol = at_target[:, None] * wide[targets.long()] + others @ wide + (16 + vocab / 128) * 2.0 ** -23 * (g.abs() @ wide) + vocab * 2.0 ** -38 * float(wide.max()) + want.abs() * 2.0 ** -23
    assert bool(((d_x.double() - want).abs() <= tol).all())
