"""Matrices orthogonalised by Newton-Schulz products, and the optimiser step that applies them, on the GPU against 64 bits.

Tolerance. A step takes a singular value s to f(s) = a s + b s^3 + c s^5; |f'| and the quotients (f(s) +- f(t)) / (s +- t) are at most a on the values that occur, so an error
of X grows by a at most. Each of a step's three products is off by at most e = 2^-19 of the norms of its factors (two parts of each of two values: 2^-22 each; what is left out:
2^-22; sums cut off four times and rounded: 6 * 2^-23; G's and B's own rounding 2^-22: 7 * 2^-22 in all), which makes 3 (|a| + |b| + |c|) e |X| a step in all; |X| is at most 1.21 sqrt(side) after a step. With
k steps: |O - exact| <= 37 e sqrt(side) (1 + a + .. + a^(k-1)), and a k-fold part for the first X, rounded to 2^-22. The type's rounding comes on top."""
import pytest

from helpers import pkg

pytestmark = pytest.mark.gpu
A, B, C = 3.4445, -4.7750, 2.0315


@pytest.fixture(scope="module")
def torch():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch


def exact(torch, u, steps, eps=1e-7):
    x = u.double() / (torch.linalg.matrix_norm(u.double(), keepdim=True) + eps)
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.transpose(-1, -2)
    for _ in range(steps):
        g = x @ x.transpose(-1, -2)
        x = A * x + (B * g + C * (g @ g)) @ x
    return x.transpose(-1, -2) if tall else x


def bound(torch, want, steps):
    """Of the 2-norm of a matrix's error."""
    side = min(want.shape[-2:])
    grown = sum(A ** i for i in range(steps))
    half = torch.finfo(torch.float32).eps / 2
    return 37 * 2.0 ** -19 * side ** 0.5 * grown / 4 + A ** steps * 2.0 ** -22 + half * torch.linalg.matrix_norm(want)


def check(torch, got, want, steps):
    off = torch.linalg.matrix_norm(got.double() - want)
    tol = bound(torch, want, steps)
    if got.dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * torch.linalg.matrix_norm(want)
    assert bool((off <= tol).all()), (float(off.max()), float(tol.min()))


def updates(torch, seed, n, rows, cols, dtype="fp32", size=1e-3):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    u = size * (r(n, rows, cols) + 2 * r(n, rows, 3) @ r(n, 3, cols))
    return u.to(torch.bfloat16 if dtype == "bf16" else torch.float32)


SMALL = [(1, 1, 1), (2, 1, 40), (1, 40, 1), (3, 16, 16), (2, 31, 65), (1, 64, 128), (2, 128, 129), (1, 127, 256), (2, 256, 128), (1, 255, 3), (1, 128, 257), (3, 100, 700), (2, 513, 65), (1, 2048, 128), (70, 5, 300), (1, 1, 2048), (1, 77, 2049)]
LARGE = [(1, 129, 129), (2, 130, 257), (1, 257, 130), (1, 3, 257), (1, 1000, 5), (3, 131, 515), (1, 515, 131), (1, 384, 384), (2, 300, 701), (1, 128, 2000), (1, 640, 129), (70, 130, 130)]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("n,rows,cols", SMALL + LARGE)
def test_against_64_bits(torch, dtype, n, rows, cols):
    p = pkg()
    u = updates(torch, rows + cols, n, rows, cols, dtype)
    for steps in (1, 2, 5):
        o = p.orthogonalize(u, steps)
        assert p.sync_status() == 0 and o.shape == u.shape and o.dtype == u.dtype
        check(torch, o, exact(torch, u, steps), steps)


@pytest.mark.parametrize("rows,cols", [(768, 768), (1024, 700), (700, 1500), (1200, 2400)])
def test_larger(torch, rows, cols):
    """Sizes whose contractions are cut among CTAs, and whose products are launches of their own; a factor of 4 of what sums in 32 bits give."""
    p = pkg()
    u = updates(torch, 1, 1, rows, cols)
    o = p.orthogonalize(u)
    assert p.sync_status() == 0
    want = exact(torch, u, 5)
    check(torch, o, want, 5)
    x = u / (torch.linalg.matrix_norm(u, keepdim=True) + 1e-7)
    tall = rows > cols
    x = x.transpose(1, 2) if tall else x
    for _ in range(5):
        g = x @ x.transpose(1, 2)
        x = A * x + (B * g + C * (g @ g)) @ x
    x = x.transpose(1, 2) if tall else x
    assert float((o.double() - want).norm()) <= 4 * float((x.double() - want).norm())


@pytest.mark.parametrize("rows,cols", [(40, 70), (140, 300)])
def test_strides(torch, rows, cols):
    """Rows and matrices that lie apart and begin anywhere, in and out; what lies between stays. Two-dimensional, and in place."""
    p = pkg()
    u = updates(torch, 5, 3, rows, cols)
    want = p.orthogonalize(u)
    wide = torch.full((3, rows + 2, cols + 5), float("nan"), device="cuda")
    wide[:, 1:rows + 1, 3:cols + 3] = u
    out = torch.full((3, rows + 1, cols + 3), 7.0, device="cuda")
    got = p.orthogonalize(wide[:, 1:rows + 1, 3:cols + 3], out=out[:, :rows, 1:cols + 1])
    assert torch.equal(got, want)
    out[:, :rows, 1:cols + 1] = 7.0
    assert bool((out == 7.0).all())
    assert torch.equal(p.orthogonalize(u[1]), want[1])
    assert torch.equal(p.orthogonalize(u[:1].expand(3, rows, cols)), want[:1].expand(3, rows, cols))
    assert p.orthogonalize(u, out=u) is u and torch.equal(u, want)
    assert p.sync_status() == 0


@pytest.mark.parametrize("rows,cols", [(60, 90), (150, 260)])
@pytest.mark.parametrize("size", [1e-30, 1e-12, 1e30])
def test_any_size(torch, rows, cols, size):
    """The norm is taken in double: gradients whose squares leave fp32. eps = 0 leaves the scale out of it."""
    p = pkg()
    u = updates(torch, 6, 1, rows, cols, size=1.0) * size
    check(torch, p.orthogonalize(u, 5, eps=0.0), exact(torch, u, 5, 0.0), 5)
    o = p.orthogonalize(u)
    assert p.sync_status() == 0
    check(torch, o, exact(torch, u, 5), 5)


@pytest.mark.parametrize("rows,cols", [(60, 90), (150, 260), (260, 150)])
def test_zeros_and_values_that_are_not_finite(torch, rows, cols):
    """A zero matrix gives 0; a NaN or infinity makes its matrix NaN and touches no other."""
    p = pkg()
    u = updates(torch, 7, 5, rows, cols)
    want = p.orthogonalize(u)
    v = u.clone()
    v[0] = 0.0
    v[2, 3, 5] = float("nan")
    v[4, rows - 1, cols - 1] = float("inf")
    o = p.orthogonalize(v)
    assert p.sync_status() == 0
    assert not o[0].any() and bool(o[2].isnan().all()) and bool(o[4].isnan().all())
    assert torch.equal(o[1], want[1]) and torch.equal(o[3], want[3])


def test_other_polynomials(torch):
    p = pkg()
    for coefficients in ((1.5, -0.5, 0.0), (1.875, -1.25, 0.375)):
        a, b, c = coefficients
        for rows, cols in ((50, 50), (200, 300)):
            u = updates(torch, 8, 1, rows, cols)
            x = u.double()[0] / (torch.linalg.matrix_norm(u.double()[0]) + 1e-7)
            for _ in range(8):
                g = x @ x.t()
                x = a * x + (b * g + c * (g @ g)) @ x
            o = p.orthogonalize(u, 8, coefficients)
            # an error grows by a at most, 1.875^8 = 153, as above
            assert float((o[0].double() - x).norm()) <= 37 * 2.0 ** -19 * rows ** 0.5 * sum(a ** i for i in range(8)) / 4 + a ** 8 * 2.0 ** -22


def tensors(torch, seed, n, rows, cols):
    torch.manual_seed(seed)
    return [[torch.randn(rows, cols, device="cuda") * s for _ in range(n)] for s in (0.02, 5e-3, 1e-3)]


@pytest.mark.parametrize("n,rows,cols", [(1, 5, 7), (3, 64, 128), (2, 130, 65), (5, 200, 333), (2, 333, 200), (70, 24, 32), (66, 136, 129)])
@pytest.mark.parametrize("nesterov", [True, False])
def test_step(torch, n, rows, cols, nesterov):
    """Momentum: one rounding of a multiply and add. Parameters: the bound of the update times the step, and two roundings. Two steps, one after the other."""
    p = pkg()
    parameters, momenta, gradients = tensors(torch, n + rows, n, rows, cols)
    kw = dict(momentum=0.9, weight_decay=0.1, nesterov=nesterov, update_scale=1.5)
    for lr in (0.02, 0.5):
        before = [[t.double() for t in ts] for ts in (parameters, momenta)]
        p.muon_update(parameters, momenta, gradients, lr, **kw)
        assert p.sync_status() == 0
        for q, m, g, q0, m0 in zip(parameters, momenta, gradients, *before):
            want = 0.9 * m0 + g.double()
            assert bool(((m.double() - want).abs() <= 2.0 ** -23 * (m0.abs() + g.double().abs())).all())
            u = (g.double() + 0.9 * m.double() if nesterov else m.double())
            o = exact(torch, u, 5)
            off = q.double() - (q0 * (1 - lr * 0.1) - lr * 1.5 * o)
            assert float(off.norm()) <= 1.5 * lr * float(bound(torch, o, 5)) * 1.01 + 2.0 ** -22 * float(q0.norm() + 1.5 * lr * o.norm())


def test_step_of_views(torch):
    """Parameters that are parts of one buffer, at any element."""
    p = pkg()
    for rows, cols in ((10, 11), (140, 131)):
        held = torch.zeros(3 * rows * cols + 5, device="cuda")
        parts = [held[1 + i * rows * cols:1 + (i + 1) * rows * cols].view(rows, cols) for i in range(3)]
        parameters, momenta, gradients = tensors(torch, 4, 3, rows, cols)
        for a, b in zip(parts, parameters):
            a.copy_(b)
        m2 = [m.clone() for m in momenta]
        p.muon_update(parameters, momenta, gradients, 0.1)
        p.muon_update(parts, m2, gradients, 0.1)
        assert all(torch.equal(a, b) for a, b in zip(parts, parameters)) and all(torch.equal(a, b) for a, b in zip(m2, momenta))
        assert not held[:1].any() and not held[-4:].any()


@pytest.mark.parametrize("rows,cols", [(48, 80), (150, 200), (768, 768)])
def test_captured_replayed_and_on_two_streams(torch, rows, cols):
    p = pkg()
    u = updates(torch, 9, 2, rows, cols)
    out = torch.empty_like(u)
    ws = torch.randint(0, 256, (max(256, p.orthogonalize_workspace_bytes(2, rows, cols)),), dtype=torch.uint8, device="cuda")
    p.orthogonalize(u, out=out, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p.orthogonalize(u, out=out, workspace=ws)
    for seed in (10, 11, 10):
        u.copy_(updates(torch, seed, 2, rows, cols))
        graph.replay()
        assert p.sync_status() == 0
        check(torch, out, exact(torch, u, 5), 5)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for _ in range(6):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(p.orthogonalize(u))
    torch.cuda.synchronize()
    assert p.sync_status() == 0 and all(torch.equal(g, out) for g in got)
    named = p.orthogonalize(u, stream=streams[1])
    torch.cuda.synchronize()
    assert torch.equal(named, out)


def test_refusals(torch):
    p = pkg()
    u = updates(torch, 3, 2, 8, 12)
    ps, ms, gs = tensors(torch, 1, 2, 8, 12)
    for call in (lambda: p.orthogonalize(u.cpu()), lambda: p.orthogonalize(u.half()), lambda: p.orthogonalize(u[0, 0]), lambda: p.orthogonalize(u.transpose(1, 2)), lambda: p.orthogonalize(u, 0),
                 lambda: p.orthogonalize(u, 65), lambda: p.orthogonalize(u, 5, (1.0, 2.0)), lambda: p.orthogonalize(u, 5, (20.0, 0.0, 0.0)), lambda: p.orthogonalize(u, 5, eps=-1.0),
                 lambda: p.orthogonalize(u, out=u[:1]), lambda: p.orthogonalize(u, out=u.bfloat16()), lambda: p.orthogonalize(u, workspace=torch.empty(8, dtype=torch.uint8, device="cuda")),
                 lambda: p.orthogonalize(u[:, :0]), lambda: p.muon_update(ps, ms[:1], gs, 0.1), lambda: p.muon_update(ps, ms, [g.bfloat16() for g in gs], 0.1),
                 lambda: p.muon_update(ps, ms, [gs[0], gs[1].t()], 0.1), lambda: p.muon_update(ps, ps, gs, 0.1), lambda: p.muon_update([ps[0], ps[0]], ms, gs, 0.1),
                 lambda: p.muon_update(ps, ms, gs, float("nan")), lambda: p.muon_update([q[:, 1:] for q in ps], [m[:, 1:] for m in ms], [g[:, 1:] for g in gs], 0.1)):
        with pytest.raises((p.AttentionError, ValueError, TypeError)):
            call()
    p.muon_update([], [], [], 0.1)
    assert p.sync_status() == 0
