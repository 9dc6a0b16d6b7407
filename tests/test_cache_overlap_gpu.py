"""Buffers that lie side by side without overlapping are taken, and two states that a program swaps give the same as new ones."""
import pytest

from helpers import pkg
from test_cache_gpu import ints, torch  # noqa: F401 (torch: the fixture)

pytestmark = pytest.mark.gpu


def test_results_right_behind_what_is_read(torch):  # noqa: F811
    p = pkg()
    room = torch.full((64,), -9, dtype=torch.int32, device="cuda")
    lens, new, lens_out, starts, slots, positions, state, count = room[0:2], room[2:4], room[4:6], room[6:9], room[9:14], room[14:19], room[19:21], room[21:22]
    free, table = room[22:30], room[30:38].view(2, 4)
    lens.copy_(ints(torch, [15, 3]))
    new.copy_(ints(torch, [3, 2]))
    free.copy_(ints(torch, range(10, 18)))
    table.copy_(ints(torch, [[1, 0, 0, 0], [2, 0, 0, 0]]))
    count.fill_(8)
    p.cache_plan(lens, new, table, free, count, 16, 5, lens_out=lens_out, starts=starts, slots=slots, positions=positions, state=state)
    assert p.sync_status() == 0
    assert lens_out.tolist() == [18, 5] and starts.tolist() == [0, 3, 5] and state.tolist() == [7, 0]
    assert slots.tolist() == [31, 17 * 16, 17 * 16 + 1, 35, 36] and positions.tolist() == [15, 16, 17, 3, 4]
    for kw in (dict(state=room[20:22]), dict(lens_out=new), dict(starts=room[5:8]), dict(positions=slots)):
        given = dict(lens_out=lens_out, starts=starts, slots=slots, positions=positions, state=state)
        given.update(kw)
        with pytest.raises(p.AttentionError):
            p.cache_plan(lens, new, table, free, count, 16, 5, **given)
    assert p.lib().df_attn_last_status() != p.DF_OK and p.sync_status() == 0


def test_two_states_in_turn(torch):  # noqa: F811
    """700 requests (several blocks), three steps with lengths and states swapped between two buffers each."""
    p = pkg()
    n = 700
    lens = [ints(torch, [r % 40 for r in range(n)]), torch.empty(n, dtype=torch.int32, device="cuda")]
    state = [ints(torch, [4 * n, 0]), ints(torch, [0, 0])]
    free, table = ints(torch, range(4 * n)), torch.zeros((n, 5), dtype=torch.int32, device="cuda")
    new, plain = ints(torch, [1 + r % 3 for r in range(n)]), None
    total = int(new.sum())
    want_lens, count, table2 = lens[0].clone(), state[0][:1].clone(), table.clone()
    for step in range(3):
        a, b = step % 2, 1 - step % 2
        _, _, slots, _, _ = p.cache_plan(lens[a], new, table, free, state[a][:1], 16, total, lens_out=lens[b], state=state[b])
        want_lens, _, plain, _, s = p.cache_plan(want_lens, new, table2, free, count, 16, total)
        count = s[:1]
        assert p.sync_status() == 0
        assert torch.equal(slots, plain) and torch.equal(lens[b], want_lens) and torch.equal(state[b], s) and torch.equal(table, table2)
    assert state[1].tolist()[1] == 0
