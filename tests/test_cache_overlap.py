"""Plan and release refuse, on the host, results that lie where they read or where another result goes (the pointers are never followed)."""
import ctypes

import pytest

from helpers import pkg

R, TOKENS, WIDTH, PAGES = 3, 5, 4, 12
SIZES = {"lens": R, "new_tokens": R, "block_table": R * WIDTH, "free_pages": PAGES, "free_count": 1, "lens_out": R, "starts": R + 1, "slots": TOKENS,
         "positions": TOKENS, "state": 2, "finished": R, "count_out": 1}
PLAN = ("lens", "new_tokens", "block_table", "free_pages", "free_count", "lens_out", "starts", "slots", "positions", "state")
RELEASE = ("lens", "finished", "block_table", "free_pages", "free_count", "lens_out", "count_out")
PLAN_OUT, RELEASE_OUT = PLAN[5:] + ("block_table",), ("lens_out", "count_out", "free_pages")


@pytest.fixture
def call():
    p = pkg()
    L = p.lib()
    memory = (ctypes.c_int32 * 1024)()
    base = ctypes.addressof(memory)

    def run(names, move):
        """`move`: {name: (other, entries)}: that argument lies so many entries behind the beginning of the other."""
        at = {n: base + 4 * 64 * i for i, n in enumerate(names)}
        for n, (other, by) in move.items():
            at[n] = at[other] + 4 * by
        f = L.df_cache_plan if names is PLAN else L.df_cache_release
        sizes = (R, TOKENS, WIDTH, 16, PAGES) if names is PLAN else (R, WIDTH, 16, PAGES)
        return f(*(ctypes.c_void_p(at[n]) for n in names), *sizes, None)

    L.df_attn_last_status()
    yield run
    L.df_attn_last_status()


@pytest.mark.parametrize("names,outputs", [(PLAN, PLAN_OUT), (RELEASE, RELEASE_OUT)], ids=["plan", "release"])
def test_results_apart_from_what_is_read(call, names, outputs):
    p = pkg()
    for out in outputs:
        for other in names:
            if other == out:
                continue
            for by in (0, SIZES[other] - 1, 1 - SIZES[out]):
                assert call(names, {out: (other, by)}) == p.DF_ERR_INVALID_ARG, (out, other, by)


def test_the_next_count_is_not_read_from_where_it_is_written(call):
    p = pkg()
    assert call(PLAN, {"free_count": ("state", 0)}) == p.DF_ERR_INVALID_ARG
    assert call(PLAN, {"lens_out": ("new_tokens", 0)}) == p.DF_ERR_INVALID_ARG
    assert call(RELEASE, {"lens_out": ("finished", 0)}) == p.DF_ERR_INVALID_ARG
