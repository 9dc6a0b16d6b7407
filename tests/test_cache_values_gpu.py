"""Attention over the 8-bit cache where weights must not lose bits: each row against 64 bits, relative to what that row adds up."""
import numpy as np
import pytest

from helpers import pkg
from test_cache_gpu import Problem, torch  # noqa: F401 (torch: the fixture)

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
    two parts 2^-23 each. All of it is relative to the row's own sum. bf16
    results are that, rounded once: half a unit in the last of 8 bits."""
    out = out.to(pr.torch.float64).cpu().numpy().reshape(-1, pr.heads, pr.d)
    for r, n in enumerate(pr.lens):
        want, size, magnitude = reference(pr, r)
        tol = ((2 * 2.0 ** -19 * magnitude + 2.0 ** -18 + n / 8 * 2.0 ** -23) * size)[:, :, None] + np.zeros_like(want)
        if pr.bf16:
            tol += np.exp2(np.floor(np.log2(np.maximum(np.abs(want) + tol, 1e-300))) - 8)
        far = np.abs(out[pr.starts[r]:pr.starts[r + 1]] - want)
        assert (far <= tol).all(), (r, (far / tol).max())


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
