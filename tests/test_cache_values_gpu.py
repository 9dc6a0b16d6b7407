"""Attention over the 8-bit cache where V's scales lie far apart and where weights must not lose bits: each row against 64 bits, relative to what that
row adds up, and rows that do not see a page bit for bit whatever its scale is."""
import numpy as np
import pytest

from helpers import pkg
from test_cache_gpu import Problem, dev, torch  # noqa: F401 (torch: the fixture)

pytestmark = pytest.mark.gpu


def reference(pr, r):
    """Request r in 64 bits: out [rows, heads, d], size [rows, heads] = the largest dim's sum of weight * |v|, magnitude [rows, heads] = the largest sum of
    magnitudes of a visible score."""
    n, group = pr.lens[r], pr.heads // pr.k.shape[1]
    pages = pr.table[r, :-(-n // pr.page)]
    rows = np.arange(pr.starts[r], pr.starts[r + 1])
    sees = np.arange(n)[None] <= (n - len(rows) + np.arange(len(rows)))[:, None]
    out = np.zeros((len(rows), pr.heads, pr.d))
    size, magnitude = np.zeros((len(rows), pr.heads)), np.zeros((len(rows), pr.heads))
    for h in range(pr.heads):
        k, v = (x[pages, h // group].reshape(-1, pr.d)[:n] for x in (pr.k, pr.v))
        q = pr.q[rows, h]
        s = np.where(sees, q @ k.T * pr.scale, -np.inf)
        w = np.exp(s - s.max(1, keepdims=True))
        w /= w.sum(1, keepdims=True)
        out[:, h] = w @ v
        size[:, h] = (w @ np.abs(v)).max(1)
        magnitude[:, h] = np.where(sees, np.abs(q) @ np.abs(k).T, 0.0).max(1) * pr.scale
    return out, size, magnitude


def check_rows(pr, out):
    """A score (fp32 sums of d products, q in 22 bits) is within 2^-19 of its sum of magnitudes, so a weight and the sum that it is divided by are within
    twice that of themselves; exponentials, the weights' 22 bits and fp32 sums add 2^-18, tensor-core sums cut off at each of len / 16 steps of one or
    two parts 2^-23 each. Weights are held relative to the largest weight * scale of their row, so all of it is relative to the row's own sum. bf16
    results are that, rounded once: half a unit in the last of 8 bits."""
    out = out.to(pr.torch.float64).cpu().numpy().reshape(-1, pr.heads, pr.d)
    for r, n in enumerate(pr.lens):
        want, size, magnitude = reference(pr, r)
        tol = ((2 * 2.0 ** -19 * magnitude + 2.0 ** -18 + n / 8 * 2.0 ** -23) * size)[:, :, None] + np.zeros_like(want)
        if pr.bf16:
            tol += np.exp2(np.floor(np.log2(np.maximum(np.abs(want) + tol, 1e-300))) - 8)
        far = np.abs(out[pr.starts[r]:pr.starts[r + 1]] - want)
        assert (far <= tol).all(), (r, (far / tol).max())


def set_v_scale(pr, page, head, factor):
    pr.scales[1][page, head] *= factor
    pr.v[page, head] *= factor


FAR = [8, 16, 32, 60]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("far", FAR)
@pytest.mark.parametrize("lens,new,heads,kv,d", [([130, 250], [1, 5], 4, 2, 64), ([130, 250], [1, 5], 8, 2, 128), ([130, 1010], [1, 20], 4, 2, 64), ([130, 600], [1, 100], 4, 2, 64),
                                                 ([130, 600], [1, 100], 4, 2, 128)])
def test_rows_that_do_not_see_a_page_are_blind_to_its_scale(torch, lens, new, heads, kv, d, far, code, dtype):  # noqa: F811
    """The last page's V scale is 2^far larger: nothing changes for the rows before it, and the rows that see it are right."""
    pr = Problem(torch, 41, lens, new, heads, kv, d, 16, dtype, code)
    clean, clean_lse = pr.call()
    first = (lens[1] - 1) // 16 * 16  # of the last page's tokens
    set_v_scale(pr, int(pr.table[1, first // 16]), 1, 2.0 ** far)
    out, lse = pr.call()
    assert pkg().sync_status() == 0
    group = heads // kv
    hit = torch.zeros(out.shape[0], heads, dtype=torch.bool, device="cuda")
    hit[1 + max(0, new[1] - (lens[1] - first)):, group:] = True
    same = (out == clean).view(-1, heads, d).all(2) & (lse == clean_lse)
    assert same[~hit].all()
    assert torch.equal(lse, clean_lse)  # scores have nothing to do with V
    check_rows(pr, out)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("far,key", [(8, 7), (16, 13), (32, 24), (60, 44), (60, 120)])
@pytest.mark.parametrize("new,heads,kv,d", [(1, 4, 2, 64), (5, 8, 4, 64), (7, 4, 1, 128), (90, 4, 2, 64), (90, 2, 1, 128)])
def test_a_page_of_large_values_and_small_weights(torch, new, heads, kv, d, far, key, code, dtype):  # noqa: F811
    """A page in the middle with V 2^far larger and scores `key` below the others': its part of the result is of the others' size (key about far log 2) or
    nothing (120), and either way nobody's bits are lost. The first page is as much smaller."""
    pr = Problem(torch, 43, [300, 170], [new, 1], heads, kv, d, 16, dtype, code)
    pr.q[:, :, 0] = 8.0
    pr.tq = dev(torch, pr.q.reshape(pr.q.shape[0], -1)).to(pr.td)
    pr.k[..., 0] = 0.0
    codes = pr.codes[0].to(torch.float32)
    codes[..., 0] = 0.0
    page = int(pr.table[0, 7])
    codes[page] = 0.0
    codes[page, ..., 0] = -key
    pr.codes[0] = codes.to(pr.codes[0].dtype)
    pr.scales[0][page] = d ** 0.5 / 8 if d == 64 else 1.5  # (one, and where d is 128 another number than a power of two: 8 * 1.5 * key / sqrt 128 is about key)
    pr.k[page] = 0.0
    pr.k[page, ..., 0] = -key * (1.0 if d == 64 else 1.5)
    for h in range(kv):
        set_v_scale(pr, page, h, 2.0 ** far)
        set_v_scale(pr, int(pr.table[0, 0]), h, 2.0 ** -far)
    out, _ = pr.call()
    assert pkg().sync_status() == 0
    check_rows(pr, out)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("new,heads,kv,d", [(1, 4, 4, 64), (1, 16, 1, 128), (5, 12, 4, 64), (5, 12, 4, 128), (3, 16, 2, 80), (40, 4, 4, 64), (70, 2, 1, 128)])
def test_weights_keep_the_bits_of_32(torch, new, heads, kv, d, dtype, code):  # noqa: F811
    """Scores close together (every token counts) over few tokens: weights rounded to 11 bits would be 2^-12 off each, which a bf16 result's own rounding
    does not cover where its last bit hangs on it or where values cancel."""
    pr = Problem(torch, 47, [new + 2, new + 19, 90], [new] * 3, heads, kv, d, 16, dtype, code)
    pr.scales[0].mul_(2.0 ** -5 if code == "int8" else 2.0 ** -4)
    pr.k = pr.k * (2.0 ** -5 if code == "int8" else 2.0 ** -4)
    out, _ = pr.call()
    assert pkg().sync_status() == 0
    check_rows(pr, out)


def test_scales_at_the_ends_of_the_number_range(torch):  # noqa: F811
    """Pages of zeros have the smallest scale (2^-126), pages of huge numbers one near 2^100; both in one request, and a scale of zero."""
    for new in (1, 6, 60):
        for d in (64, 128):
            pr = Problem(torch, 53, [200, 64, 40], [new, min(new, 64), 1], 4, 2, d, 16, "fp32", "int8")
            for r, (low, high) in enumerate(((2, 5), (1, 3), (0, 2))):
                for h in range(2):
                    page = int(pr.table[r, low])
                    pr.scales[1][page, h] = 2.0 ** -126
                    pr.codes[1][page, h] = 0
                    pr.v[page, h] = 0.0
                    page = int(pr.table[r, high])
                    was = pr.scales[1][page, h].item()
                    set_v_scale(pr, page, h, 2.0 ** 90 / was if r < 2 else 0.0)
            out, _ = pr.call()
            assert pkg().sync_status() == 0
            check_rows(pr, out)
