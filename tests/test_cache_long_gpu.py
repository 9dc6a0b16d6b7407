"""Attention of many query rows over a long 8-bit cache: what long sums must not lose, and shapes whose parts of the work are long."""
import numpy as np
import pytest

from helpers import pkg
from test_cache_gpu import Problem, ints, torch  # noqa: F401 (torch: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,heads,length", [(64, 12, 80000), (128, 6, 80000), (96, 5, 60011)])
def test_sums_of_one_sign_over_many_tokens(torch, d, heads, length):  # noqa: F811
    """Values of one sign, so that every step's cut goes the same way. Tensor-core sums lose up to 2^-23 of themselves at each of 64 steps (8 stages of 64
    tokens, 4 steps of 16 each, two parts of a weight), then they are added up in rounded arithmetic (2^-18 with the exponentials); a score is within
    2^-19 of the sum of its magnitudes. Cut at every step of a CTA's part (400) it would be 2.4e-5."""
    p, page, rows = pkg(), 64, 40
    pages = -(-length // page)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(d)
    k = torch.randint(-127, 128, (pages, heads, page, d), generator=gen, device="cuda", dtype=torch.int32).to(torch.int8)
    v = torch.randint(64, 128, (pages, heads, page, d), generator=gen, device="cuda", dtype=torch.int32).to(torch.int8)
    scales = torch.full((pages, heads), 2.0 ** -6, device="cuda")
    q = torch.randn(rows, heads * d, generator=gen, device="cuda") * 0.05
    workspace = torch.zeros(p.CACHE_WORKSPACE_BYTES, dtype=torch.uint8, device="cuda")
    out, _ = p.cache_attention(q, k, v, scales, scales, torch.arange(pages, device="cuda", dtype=torch.int32)[None], ints(torch, [length]),
                               ints(torch, [0, rows]), heads, d ** -0.5, workspace)
    assert p.sync_status() == 0
    scale = float(np.float32(d ** -0.5))
    sees = torch.arange(length, device="cuda")[None] <= torch.arange(length - rows, length, device="cuda")[:, None]
    for h in range(heads):
        kh, vh = (x[:, h].reshape(-1, d)[:length].double() * 2.0 ** -6 for x in (k, v))
        qh = q.double().view(rows, heads, d)[:, h]
        s = (qh @ kh.t() * scale).masked_fill(~sees, float("-inf"))
        want = s.softmax(1) @ vh
        magnitude = float((qh.abs() @ kh.abs().t()).max()) * scale
        tol = 64 * 2.0 ** -23 + 2.0 ** -18 + 2 * 2.0 ** -19 * magnitude
        assert float(((out.double().view(rows, heads, d)[:, h] - want).abs() / want).max()) <= tol


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("shape", [([9000, 5000], [40, 33], 12, 12, 64, 16), ([7001, 1], [35, 1], 16, 8, 128, 32), ([3000] * 6, [200, 1, 90, 40, 0, 64], 8, 4, 112, 16)],
                         ids=lambda s: "x".join(map(str, s[2:])))
def test_long_parts_against_64_bits(torch, shape, dtype):  # noqa: F811
    pr = Problem(torch, 3, *shape, dtype, "e4m3")
    out, lse = pr.call()
    assert pkg().sync_status() == 0
    pr.check(out, lse)
    again, _ = pr.call()
    assert pkg().sync_status() == 0 and torch.equal(out, again)
