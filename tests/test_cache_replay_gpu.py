"""A captured step replayed while the requests grow, against attention over what the cache holds: the codes' own rounding apart, so that one token or page left out
shows."""
import numpy as np
import pytest

import cache_reference as ref
from helpers import pkg
from test_cache_gpu import dev, ints, torch  # noqa: F401 (torch: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_replays_attend_to_all_that_is_cached(torch, code):  # noqa: F811
    p = pkg()
    rng = np.random.RandomState(61)
    requests, heads, kv, d, page, width, steps = 3, 4, 2, 64, 16, 8, 40
    pages = requests * width
    type_of = torch.int8 if code == "int8" else torch.float8_e4m3fn
    table = torch.zeros((requests, width), dtype=torch.int32, device="cuda")
    lens, new = ints(torch, [0, 0, 0]), ints(torch, [1, 1, 1])
    free, count = ints(torch, rng.permutation(pages)), ints(torch, [pages])
    q, k, v = (torch.zeros((requests, n * d), device="cuda") for n in (heads, kv, kv))
    kc, vc = (torch.zeros((pages, kv, page, d), dtype=torch.int8, device="cuda").view(type_of) for _ in range(2))
    ks, vs = (torch.zeros((pages, kv), device="cuda") for _ in range(2))
    work = torch.zeros(p.CACHE_WORKSPACE_BYTES, dtype=torch.uint8, device="cuda")

    def step():
        lens_out, starts, slots, _, state = p.cache_plan(lens, new, table, free, count, page, requests)
        p.cache_append(k, v, slots, kc, vc, ks, vs)
        out, lse = p.cache_attention(q, kc, vc, ks, vs, table, lens_out, starts, heads, 0.125, work)
        lens.copy_(lens_out)
        count.copy_(state[:1])
        return out, lse

    step()  # kernels are loaded outside the capture
    torch.cuda.synchronize()
    lens.zero_()
    count.fill_(pages)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = step()
    given = [[], []]
    for t in range(steps):
        for x in (q, k, v):
            x.copy_(dev(torch, rng.standard_normal(tuple(x.shape)), torch.float32))
        graph.replay()
        assert p.sync_status() == 0
        for kept, x in zip(given, (k, v)):
            kept.append(x.cpu().numpy().reshape(requests, kv, d).astype(np.float64))
        held = [c.to(torch.float32).cpu().numpy().astype(np.float64) * s.cpu().numpy().astype(np.float64)[:, :, None, None] for c, s in ((kc, ks), (vc, vs))]
        where = table.cpu().numpy()
        want, want_lse, magnitude = ref.attention(q.cpu().numpy().reshape(requests, heads, d).astype(np.float64), *held, where, [t + 1] * requests,
                                                  np.arange(requests + 1), page, 0.125)
        tol = 2.0 ** -19 * magnitude  # a score; see Problem.check
        assert np.abs(out.cpu().numpy().reshape(want.shape) - want).max() <= (2 * tol + 2.0 ** -18) * np.abs(held[1]).max()
        assert np.abs(lse.cpu().numpy() - want_lse).max() <= tol + 2.0 ** -19 * (1 + np.abs(want_lse).max())
    # what is cached is what was given, within a step of its page's scale (e4m3: a step at the element's size, 2^-3 of it at most)
    for kept, values, scales in zip(given, held, (ks, vs)):
        for r in range(requests):
            for t in range(steps):
                page_of = where[r, t // page]
                step_of = scales[page_of].cpu().numpy().astype(np.float64)[:, None]
                each = step_of if code == "int8" else np.maximum(step_of * 2.0 ** -9, np.abs(kept[t][r]) / 8)
                assert (np.abs(values[page_of, :, t % page] - kept[t][r]) <= each).all()
