"""Requests' rows that overlap: starts that fall are refused by the kernels themselves, with the status that says so, and the next call is as ever."""
import pytest

from helpers import pkg
from test_cache_gpu import Problem, ints, torch  # noqa: F401 (torch: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("new", [1, 9, 70])
def test_starts_that_fall(torch, new, dtype):  # noqa: F811
    p = pkg()
    pr = Problem(torch, 59, [100, 200, 90], [new] * 3, 4, 2, 64, 16, dtype, "int8")
    good = pr.starts
    clean, clean_lse = pr.call()
    for starts in ([0, 2 * new, new, 3 * new], [0, new, 2 * new, 0], [5, 2, 1, 0], [0, 2 ** 31 - 1, -2 ** 31, 3]):
        pr.starts = starts
        out, lse = torch.full_like(clean, 3.0), torch.full_like(clean_lse, 3.0)
        pr.call(out=out, lse=lse)
        assert p.sync_status() == p.DF_ERR_DEVICE_BOUNDS
        assert (out == 3).all() and (lse == 3).all()
    pr.starts = good
    out, lse = pr.call()
    assert p.sync_status() == 0 and torch.equal(out, clean) and torch.equal(lse, clean_lse)


def test_starts_behind_the_rows_that_there_are(torch):  # noqa: F811
    """Ascending, but past the rows of q: what is there of a request is computed as if it had no more."""
    p = pkg()
    pr = Problem(torch, 60, [100, 200, 90], [1, 2, 1], 4, 2, 64, 16, "fp32", "int8")
    clean, _ = pr.call()
    pr.starts = [0, 1, 3, 10 ** 9]
    out, _ = pr.call()
    assert p.sync_status() == 0 and torch.equal(out, clean)
