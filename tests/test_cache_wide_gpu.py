"""Block tables so wide that the step's work cannot be counted in stages in 32 bits: whole segments are dealt out then, and the results are those of a narrow table."""
import pytest

from helpers import pkg
from test_cache_gpu import Problem, torch  # noqa: F401 (torch: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,new", [("fp32", 1), ("bf16", 1), ("fp32", 20), ("fp32", 40), ("bf16", 40)])
def test_wide_tables(torch, dtype, new):  # noqa: F811
    requests, kv, page, width = 160, 12, 256, 100000
    lens = [1 + 37 * r % 700 + new for r in range(requests)]
    pr = Problem(torch, 67, lens, [new] * requests, kv, kv, 32, page, dtype, "int8")
    # segments times the longest that a row of the table could be, as the launcher bounds them: past 2^31 (12 K/V heads, stages of 64 tokens in up to four units)
    assert (requests * new // 8 + requests) * kv * (width * page // 64 * 4) >= 2 ** 31
    out, lse = pr.call()
    pr.check(out, lse)
    wide = torch.full((requests, width), -1, dtype=torch.int32, device="cuda")
    wide[:, :pr.table.shape[1]] = torch.from_numpy(pr.table.astype("int32")).cuda()
    p = pkg()
    starts = torch.arange(0, (requests + 1) * new, new, dtype=torch.int32, device="cuda")
    got, got_lse = p.cache_attention(pr.tq, pr.codes[0], pr.codes[1], pr.scales[0], pr.scales[1], wide, torch.tensor(lens, dtype=torch.int32, device="cuda"),
                                     starts, kv, pr.scale, pr.workspace)
    assert p.sync_status() == 0
    pr.check(got, got_lse)
    again, _ = pr.call()
    assert p.sync_status() == 0 and torch.equal(out, again)
