"""The 8-bit paged cache on the GPU: plan and release against the definition entry by entry, append code by code, attention against 64 bits."""
import numpy as np
import pytest

import cache_reference as ref
from helpers import pkg

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch


def dev(torch, x, dtype=None):
    return torch.from_numpy(np.ascontiguousarray(x)).to("cuda", dtype)


def ints(torch, x):
    return dev(torch, np.asarray(x, np.int32))


# ---------------------------------------------------------------- plan, release
def run_plan(torch, lens, new, table, free, count, page, n_tokens):
    p = pkg()
    tt = ints(torch, table)
    got = p.cache_plan(ints(torch, lens), ints(torch, new), tt, ints(torch, free), ints(torch, [count]), page, n_tokens)
    assert p.sync_status() == 0
    return [g.cpu().numpy() for g in got], tt.cpu().numpy()


def check_plan(torch, lens, new, table, free, count, page, n_tokens):
    want_table = table.copy()
    want = ref.plan(np.asarray(lens), np.asarray(new), want_table, free, count, page, n_tokens)
    got, got_table = run_plan(torch, lens, new, table, free, count, page, n_tokens)
    for g, w, name in zip(got, want, ("lens_out", "starts", "slots", "positions", "state")):
        assert np.array_equal(g, w), name
    assert np.array_equal(got_table, want_table)
    return got


@pytest.mark.parametrize("requests,prompt,page,spare", [(1, 1, 16, 0), (1, 5000, 16, 0), (3, 17, 7, 2), (64, 1, 16, 5), (255, 40, 32, 0), (257, 1, 16, 1),
                                                        (1000, 30, 64, 11), (1025, 9, 16, 0), (16384, 2, 16, 3)])
def test_plan_against_the_definition(torch, requests, prompt, page, spare):
    rng = np.random.RandomState(requests + page)
    lens = rng.randint(0, 6 * page, requests)
    new = rng.randint(0, prompt + 1, requests)
    lens[rng.rand(requests) < 0.1] = 0
    lens[rng.rand(requests) < 0.1] = 2 * page  # a page just full
    new[-1] = max(new[-1], 1)
    need = int((-(-(lens + new) // page) + lens // -page).sum())
    width = int(-(-(lens + new).max() // page)) + spare % 2
    pages = int((-(-lens // page)).sum()) + need + spare
    order = rng.permutation(pages)
    table, used = np.full((requests, max(width, 1)), -7), 0
    for r in range(requests):
        n = -(-lens[r] // page)
        table[r, :n] = order[used:used + n]
        used += n
    free = np.full(pages, -9)
    free[:pages - used] = order[used:]
    got = check_plan(torch, lens, new, table, free, pages - used, page, int(new.sum()) + spare)
    assert got[4][1] == 0


def test_plan_grants_everything_or_nothing(torch):
    lens, new, table, free = [5, 16, 30], [12, 1, 20], np.arange(12).reshape(3, 4), np.arange(100, 108)
    check_plan(torch, lens, new, table, free, 5, 16, 33)                # needs 1 + 1 + 2
    assert check_plan(torch, lens, new, table, free, 3, 16, 33)[4][1] == 1       # a page short
    assert check_plan(torch, lens, new, table, free, 8, 16, 32)[4][1] == -3      # the slot map is one short: request 2
    assert check_plan(torch, [5, 64, 30], new, table, free, 8, 16, 33)[4][1] == -2   # a table row of 64 tokens is full
    assert check_plan(torch, lens, new, table, free, -4, 16, 33)[4][1] == 4
    assert check_plan(torch, lens, new, table, free, 99, 16, 33)[4][0] == 4      # no more than the stack holds
    check_plan(torch, [-3, 16, 2 ** 31 - 1], [4, -5, 2 ** 31 - 1], table, free, 8, 16, 33)
    check_plan(torch, [], [], np.zeros((0, 4), int), free, 8, 16, 0)
    check_plan(torch, [], [], np.zeros((0, 4), int), free, 8, 16, 3)
    check_plan(torch, [0, 0], [0, 0], np.zeros((2, 0), int), free, 8, 16, 0)


@pytest.mark.parametrize("requests", [1, 7, 300, 3000])
def test_release_gives_pages_back_in_order(torch, requests):
    p = pkg()
    rng = np.random.RandomState(requests)
    page, width = 16, 5
    lens, finished = rng.randint(0, width * page + 1, requests), rng.randint(0, 2, requests)
    pages = requests * width
    table = rng.permutation(pages).reshape(requests, width)
    free, count = np.full(pages, -1), int(rng.randint(0, 2))
    want_free = free.copy()
    want = ref.release(lens, finished, table, want_free, count, page)
    tf = ints(torch, free)
    lens_out, count_out = p.cache_release(ints(torch, lens), ints(torch, finished), ints(torch, table), tf, ints(torch, [count]), page)
    assert p.sync_status() == 0
    assert np.array_equal(lens_out.cpu().numpy(), want[0]) and count_out.item() == want[1]
    assert np.array_equal(tf.cpu().numpy(), want_free)


def test_release_never_runs_past_the_stack(torch):
    p = pkg()
    free = torch.full((8,), -1, dtype=torch.int32, device="cuda")[:6]  # six entries, two behind them to watch
    whole = torch.full((8,), -1, dtype=torch.int32, device="cuda")
    free = whole[:6]
    _, count = p.cache_release(ints(torch, [1000, 64]), ints(torch, [1, 1]), ints(torch, np.arange(8).reshape(2, 4)), free, ints(torch, [3]), 16)
    assert p.sync_status() == 0
    assert count.item() == 6 and whole.cpu().tolist() == [-1, -1, -1, 0, 1, 2, -1, -1]


# ---------------------------------------------------------------- append
TORCH_CODE = {"int8": "int8", "e4m3": "float8_e4m3fn"}


def random_cache(torch, rng, pages, heads, page, d, code):
    """Codes as float64 values and as a tensor, scales alike: a random power of two per page and head."""
    if code == "int8":
        values = rng.randint(-127, 128, (pages, heads, page, d)).astype(np.float64)
    else:
        bits = rng.randint(0, 127, (pages, heads, page, d)) | (rng.randint(0, 2, (pages, heads, page, d)) << 7)
        values = torch.from_numpy(bits.astype(np.uint8)).view(torch.float8_e4m3fn).to(torch.float64).numpy()
    scales = 2.0 ** rng.randint(-9, -4, (pages, heads))
    if code == "e4m3":
        scales /= 4
    return values, scales, as_codes(torch, values, code), dev(torch, scales, torch.float32)


def as_codes(torch, values, code):
    return torch.from_numpy(values).to(torch.float32).to(getattr(torch, TORCH_CODE[code])).cuda()


def check_append(torch, k, v, slots, kc, vc, page, code, tk=None, tv=None):
    """kc, vc: (values, scales, codes tensor, scales tensor). Compares codes and scales exactly; the reference side is kept for a next call."""
    p = pkg()
    got = p.cache_append(tk if tk is not None else dev(torch, k.reshape(len(slots), -1), torch.float32),
                         tv if tv is not None else dev(torch, v.reshape(len(slots), -1), torch.float32), ints(torch, slots), kc[2], vc[2], kc[3], vc[3])
    assert p.sync_status() == 0
    assert got[0] is kc[2] and got[3] is vc[3]
    ref.append.code = code
    for x, c in ((k, kc), (v, vc)):
        ref.append(np.asarray(x, np.float64), slots, c[0], c[1], page)
        assert np.array_equal(c[3].cpu().numpy().astype(np.float64), c[1], equal_nan=True)
        assert np.array_equal(c[2].to(torch.float32).cpu().numpy().astype(np.float64), c[0])


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("heads,d,page", [(1, 16, 16), (3, 32, 32), (2, 48, 16), (12, 64, 16), (2, 80, 48), (1, 96, 256), (8, 128, 16), (2, 112, 64), (1, 128, 256)])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_append_is_exact_code_by_code(torch, code, heads, d, page, dtype):
    rng = np.random.RandomState(d + page)
    lens, new = [0, page - 1, 5, 2 * page, 3], [1, 1, 2 * page + 3, page, 0]
    per, n = 5, sum(new)
    pages = per * len(lens)
    table = rng.permutation(pages).reshape(len(lens), per)
    slots = [int(table[r, (lens[r] + j) // page]) * page + (lens[r] + j) % page for r in range(len(lens)) for j in range(new[r])]
    kc, vc = (random_cache(torch, rng, pages, heads, page, d, code) for _ in range(2))
    for size in (1.0, 100.0, 1e-3):  # as large as what is there, larger (older codes are rounded again), smaller
        k, v = (rng.standard_normal((n, heads, d)).astype(np.float32) * np.float32(size) for _ in range(2))
        td = torch.float32
        if dtype == "bf16":
            td = torch.bfloat16
            k, v = (torch.from_numpy(x).to(td).to(torch.float32).numpy() for x in (k, v))
        check_append(torch, k, v, slots, kc, vc, page, code, dev(torch, k.reshape(n, -1)).to(td), dev(torch, v.reshape(n, -1)).to(td))


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_append_token_by_token_stays_within_a_step(torch, code):
    """However a page is filled, an element differs from what was given by less than one step of its page's scale (e4m3: a step at the element's size)."""
    p = pkg()
    rng = np.random.RandomState(4)
    page, d = 32, 64
    x = (rng.standard_normal((page, d)) * np.exp2(np.linspace(-6, 6, page))[:, None]).astype(np.float32)  # the scale doubles again and again
    _, _, codes, scales = random_cache(torch, rng, 2, 1, page, d, code)
    vcodes, vscales = codes.clone(), scales.clone()
    for t in range(page):
        one = dev(torch, x[t:t + 1])
        p.cache_append(one, one, ints(torch, [page + t]), codes, vcodes, scales, vscales)
    assert p.sync_status() == 0
    scale = scales[1, 0].item()
    got = codes[1, 0].to(torch.float32).cpu().numpy().astype(np.float64)
    exact = x.astype(np.float64) / scale
    step = np.ones_like(exact) if code == "int8" else np.exp2(np.floor(np.log2(np.maximum(np.abs(exact), 2.0 ** -6))) - 3)
    assert scale == ref.scale_for(float(np.abs(x).max()), code)
    assert (np.abs(got - exact) < step).all()
    assert torch.equal(codes.view(torch.uint8), vcodes.view(torch.uint8)) and torch.equal(scales, vscales)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_append_at_the_ends_of_the_number_range(torch, code):
    rng = np.random.RandomState(5)
    page, d, heads = 16, 16, 2
    kc, vc = (random_cache(torch, rng, 6, heads, page, d, code) for _ in range(2))
    before = kc[0][5].copy()
    k = rng.standard_normal((6, heads, d)).astype(np.float32)
    k[0] = 0.0                       # a page of nothing but zeros: the smallest scale
    k[1] *= np.float32(1e-40)        # subnormal numbers
    k[2] *= np.float32(1e38)
    k[2, 0, 0] = np.finfo(np.float32).max
    k[3, 0] = ref.BIGGEST[code]      # just what a scale of one holds
    k[3, 1] = np.nextafter(np.float32(ref.BIGGEST[code]), np.float32(np.inf))
    k[4, 0, 3] = np.nan
    k[4, 1, 3] = -np.inf
    slots = [0 * page, 1 * page, 2 * page, 3 * page, 4 * page + 3, -1]
    check_append(torch, k, k, slots, kc, vc, page, code)
    assert np.array_equal(kc[0][5], before)
    assert np.isnan(kc[1][4]).all()
    # a poisoned page stays so, a slot behind the cache is left out, a page begun anew recovers
    check_append(torch, k[[3, 3, 0]], k[[3, 3, 0]], [4 * page + 4, 6 * page, 5 * page + 2], kc, vc, page, code)
    assert np.isnan(kc[1][4]).all()
    check_append(torch, k[:1], k[:1], [4 * page], kc, vc, page, code)
    assert not np.isnan(kc[1]).any()


def test_append_takes_strided_and_unaligned_rows(torch):
    rng = np.random.RandomState(6)
    page, heads, d, n = 16, 3, 80, 21
    slots = list(range(40, 40 + n))
    for dtype in (torch.float32, torch.bfloat16):
        for offset, extra in ((0, 4), (1, 0), (2, 3), (4, 8)):
            kc, vc = (random_cache(torch, rng, 5, heads, page, d, "int8") for _ in range(2))
            wide = torch.randn((n, heads * d + offset + extra), device="cuda").to(dtype)
            tk = wide[:, offset:offset + heads * d]
            k = tk.to(torch.float32).cpu().numpy().reshape(n, heads, d)
            tv = tk * 2
            check_append(torch, k, 2 * k, slots, kc, vc, page, "int8", tk, tv)


# ---------------------------------------------------------------- attention
class Problem:
    """Random requests over a shuffled pool; `given` = the tensors that a call takes."""

    def __init__(self, torch, seed, lens, news, heads, kv_heads, d, page, dtype, code, q_size=1.0):
        rng = np.random.RandomState(seed)
        self.torch, self.lens, self.page, self.heads, self.d, self.code = torch, lens, page, heads, d, code
        self.starts = np.concatenate(([0], np.cumsum(news))).astype(int)
        width = max(1, max(-(-max(n, 0) // page) for n in lens))
        pages = width * len(lens) + 2
        self.table = rng.permutation(pages)[:width * len(lens)].reshape(len(lens), width)
        kc, vc = (random_cache(torch, rng, pages, kv_heads, page, d, code) for _ in range(2))
        self.k, self.v = (c[0] * c[1][:, :, None, None] for c in (kc, vc))
        self.codes, self.scales = [kc[2], vc[2]], [kc[3], vc[3]]
        self.bf16 = dtype == "bf16"
        self.td = torch.bfloat16 if self.bf16 else torch.float32
        q = torch.from_numpy(rng.standard_normal((int(self.starts[-1]), heads * d)) * q_size).to(self.td)
        self.tq, self.q = q.cuda(), q.to(torch.float64).numpy().reshape(-1, heads, d)
        self.scale = float(np.float32(d ** -0.5))
        self.workspace = torch.zeros(pkg().CACHE_WORKSPACE_BYTES, dtype=torch.uint8, device="cuda")

    def call(self, **kw):
        p, torch = pkg(), self.torch
        return p.cache_attention(kw.pop("q", self.tq), self.codes[0], self.codes[1], self.scales[0], self.scales[1], ints(torch, self.table),
                                 ints(torch, self.lens), ints(torch, self.starts), self.heads, self.scale, self.workspace, **kw)

    def check(self, out, lse):
        """fp32: a score is a sum of d products (fp32, q in two half-precision parts of 22 bits together): its error is within 2^-19 of the sum of
        magnitudes; weights follow it (in natural units times their value), sums and exponentials add 2^-18. bf16 rounds the weights to 11 bits
        (2^-11 each way) and the result to 8."""
        want, want_lse, magnitude = ref.attention(self.q, self.k, self.v, self.table, self.lens, self.starts, self.page, self.scale)
        out, lse = out.to(self.torch.float64).cpu().numpy().reshape(want.shape), lse.cpu().numpy().astype(np.float64)
        d_score = 2.0 ** -19 * magnitude
        tol = (2 * d_score + 2.0 ** -18) * np.abs(self.v).max()
        each = 0.0
        if self.bf16:
            tol, each = tol + 2.0 ** -10 * np.abs(self.v).max(), 2.0 ** -8
        assert np.array_equal(np.isneginf(want_lse), np.isneginf(lse))
        seen = np.isfinite(want_lse)
        assert (np.abs(out - want) <= tol + each * np.abs(want)).all(), np.nanmax(np.abs(out - want)) / tol
        assert (out[~seen] == 0).all()
        assert (np.abs(lse - want_lse)[seen] <= d_score + 2.0 ** -19 * (1 + np.abs(want_lse[seen]))).all()


SHAPES = [  # lens, new tokens, heads, kv_heads, d, page
    ([1], [1], 1, 1, 64, 16),
    ([300], [1], 12, 12, 64, 16),
    ([15, 16, 17, 63, 64, 65, 129], [1] * 7, 4, 4, 128, 16),
    ([1000, 1, 3, 2500], [1] * 4, 8, 1, 128, 32),
    ([700, 33], [1, 1], 7, 1, 80, 48),
    ([257, 5], [1, 1], 32, 2, 32, 64),
    ([100, 511], [1, 1], 3, 3, 16, 256),
    ([90, 1030], [2, 3], 12, 4, 96, 16),
    ([640, 40, 17], [5, 8, 17], 16, 4, 64, 32),
    ([333, 1200], [70, 200], 4, 2, 128, 16),
    ([513], [513], 2, 2, 64, 16),
    ([2000, 50, 50, 3], [130, 1, 1, 3], 14, 2, 112, 16),
    ([48, 4000], [1, 1], 5, 5, 48, 16),
]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s[2:])) + "_%d" % s[0][0])
def test_attention_against_64_bits(torch, shape, code, dtype):
    pr = Problem(torch, sum(shape[0]), *shape, dtype, code)
    out, lse = pr.call()
    assert pkg().sync_status() == 0
    pr.check(out, lse)
    again, lse2 = pr.call()  # the workspace is ready again, the bits are the same
    assert pkg().sync_status() == 0
    assert torch.equal(out, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_attention_with_scores_far_apart(torch, dtype):
    pr = Problem(torch, 9, [900, 77], [1, 4], 4, 2, 64, 16, dtype, "int8", q_size=40.0)
    out, lse = pr.call()
    assert pkg().sync_status() == 0
    pr.check(out, lse)


def test_attention_rows_and_requests_that_see_nothing(torch):
    """Requests without tokens, without queries, shorter than their queries; rows behind the last request stay as they are."""
    pr = Problem(torch, 11, [0, 40, 3, 200, -5], [1, 0, 70, 2, 2], 6, 2, 64, 16, "fp32", "int8")
    extra = torch.cat([pr.tq, torch.ones_like(pr.tq[:3])])
    out = torch.full_like(extra, 7.0)
    lse = torch.full((extra.shape[0], 6), 7.0, device="cuda")
    pr.call(q=extra, out=out, lse=lse)
    assert pkg().sync_status() == 0
    assert (out[-3:] == 7).all() and (lse[-3:] == 7).all()
    pr.check(out[:-3], lse[:-3])
    assert torch.isneginf(lse[1:68]).all()


@pytest.mark.parametrize("new", [1, 3, 90])
@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_attention_is_blind_to_what_is_masked(torch, code, new):
    """Codes behind a request's end (every byte value), scales, table entries and pages that no row sees."""
    pr = Problem(torch, 13, [75, 200, 16 * 9], [min(new, 70), new, 1], 4, 2, 128, 16, "fp32", code)
    out, lse = pr.call()
    pr.check(out, lse)
    for r, n in enumerate(pr.lens):
        last = int(pr.table[r, (n - 1) // 16])
        for c in pr.codes:
            raw = c.view(torch.uint8)
            if n % 16:
                raw[last, :, n % 16:] = torch.arange(raw[last, :, n % 16:].numel(), device="cuda").to(torch.uint8).view_as(raw[last, :, n % 16:]) | 0x7C
        pr.table[r, -(-n // 16):] = [-1, 10 ** 6, -2 ** 31, 2 ** 31 - 1, 0, 1][r]
    unused = [i for i in range(pr.codes[0].shape[0]) if i not in {int(x) for r, n in enumerate(pr.lens) for x in pr.table[r, :-(-n // 16)]}]
    for s in pr.scales:
        s[unused] = float("nan")
    out2, lse2 = pr.call()
    assert pkg().sync_status() == 0
    assert torch.equal(out, out2) and torch.equal(lse, lse2)


@pytest.mark.parametrize("new", [1, 5, 100])
def test_attention_poison_reaches_who_sees_it_and_nobody_else(torch, new):
    """NaN scales of the last page: NaN for the rows that see a token of it, nothing changed for the others."""
    for which in (0, 1):
        pr = Problem(torch, 17, [130, 250], [1, new], 4, 2, 64, 16, "fp32", "int8")
        clean, clean_lse = pr.call()
        pr.scales[which][int(pr.table[1, 15]), 1] = float("nan")  # tokens 240 .. 249 of request 1, K/V head 1 = query heads 2, 3
        out, lse = pr.call()
        assert pkg().sync_status() == 0
        out, clean = out.view(-1, 4, 64), clean.view(-1, 4, 64)
        hit = torch.zeros(out.shape[:2], dtype=torch.bool, device="cuda")
        hit[1 + max(0, new - 10):, 2:] = True
        assert torch.isnan(out[hit]).all() and torch.equal(out[~hit], clean[~hit])
        assert torch.equal(lse[~hit], clean_lse[~hit]) and (which == 1 or torch.isnan(lse[hit]).all())


def test_attention_of_queries_that_are_not_finite(torch):
    pr = Problem(torch, 19, [130, 250], [1, 3], 4, 2, 64, 16, "fp32", "int8")
    clean, _ = pr.call()
    pr.tq[1, 64 * 3 + 5] = float("nan")
    pr.tq[2, 5] = float("inf")
    out, lse = pr.call()
    assert pkg().sync_status() == 0
    hit = torch.zeros((4, 4), dtype=torch.bool, device="cuda")
    hit[1, 3] = hit[2, 0] = True
    assert torch.isnan(out.view(4, 4, 64)[hit]).all() and torch.isnan(lse[hit]).all()
    assert torch.equal(out.view(4, 4, 64)[~hit], clean.view(4, 4, 64)[~hit])


def test_attention_takes_strided_queries_another_stream_and_given_outputs(torch):
    for dtype in ("fp32", "bf16"):
        pr = Problem(torch, 23, [300, 77], [1, 9], 6, 2, 80, 16, dtype, "e4m3")
        out, lse = pr.call()
        wide = torch.zeros((pr.tq.shape[0], pr.tq.shape[1] + 5), dtype=pr.td, device="cuda")
        wide[:, 3:-2] = pr.tq
        o2, l2 = torch.full_like(out, 9.0), torch.full_like(lse, 9.0)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            got = pr.call(q=wide[:, 3:-2], out=o2, lse=l2)
        side.synchronize()
        assert pkg().sync_status() == 0
        assert got[0] is o2 and torch.equal(out, o2) and torch.equal(lse, l2)


def test_attention_over_offsets_beyond_32_bits(torch):
    """A pool of more than 2^32 bytes, the request's pages at its end."""
    free, _ = torch.cuda.mem_get_info()
    heads, page, d = 16, 64, 128
    pages = (1 << 32) // (heads * page * d) + 40
    if free < 3 * pages * heads * page * d:
        pytest.skip("not enough memory")
    pr = Problem(torch, 29, [500], [1], heads, heads, d, page, "fp32", "int8")
    out, lse = pr.call()
    codes, scales = [], []
    for c, s in zip(pr.codes, pr.scales):
        big, wide = torch.empty((pages, heads, page, d), dtype=torch.int8, device="cuda"), torch.zeros((pages, heads), device="cuda")
        big[-c.shape[0]:], wide[-c.shape[0]:] = c, s
        codes.append(big)
        scales.append(wide)
    pr.table = pr.table + pages - pr.codes[0].shape[0]
    pr.codes, pr.scales = codes, scales
    out2, lse2 = pr.call()
    assert torch.equal(out, out2) and torch.equal(lse, lse2)
    # and a row put there
    p = pkg()
    x = torch.randn((1, heads * d), device="cuda")
    p.cache_append(x, x, ints(torch, [pages * page - page]), codes[0], codes[1], scales[0], scales[1])
    assert p.sync_status() == 0
    got = codes[0][-1, :, 0].float() * scales[0][-1][:, None]
    assert (got - x.view(heads, d)).abs().max() <= scales[0][-1].max() / 2


def test_a_step_as_a_graph_with_new_lengths(torch):
    """Plan, append and attention captured once and replayed while the requests grow: nothing of their lengths is fixed by the capture."""
    p = pkg()
    rng = np.random.RandomState(31)
    requests, heads, kv, d, page, width = 3, 4, 2, 64, 16, 8
    pages = requests * width
    table = torch.zeros((requests, width), dtype=torch.int32, device="cuda")
    lens, new = ints(torch, [0, 0, 0]), ints(torch, [1, 1, 1])
    free, count = ints(torch, rng.permutation(pages)), ints(torch, [pages])
    q, k, v = (torch.zeros((requests, n * d), device="cuda") for n in (heads, kv, kv))
    kc, vc = (torch.zeros((pages, kv, page, d), dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros((pages, kv), device="cuda") for _ in range(2))
    work = torch.zeros(p.CACHE_WORKSPACE_BYTES, dtype=torch.uint8, device="cuda")

    def step():
        lens_out, starts, slots, _, state = p.cache_plan(lens, new, table, free, count, page, requests)
        p.cache_append(k, v, slots, kc, vc, ks, vs)
        out, _ = p.cache_attention(q, kc, vc, ks, vs, table, lens_out, starts, heads, 0.125, work)
        lens.copy_(lens_out)
        count.copy_(state[:1])
        return out

    step()  # kernels are loaded outside the capture
    torch.cuda.synchronize()
    lens.zero_()
    count.fill_(pages)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    keys, vals = [[] for _ in range(requests)], [[] for _ in range(requests)]
    for t in range(40):
        for x in (q, k, v):
            x.copy_(dev(torch, rng.standard_normal(tuple(x.shape)), torch.float32))
        graph.replay()
        assert p.sync_status() == 0
        for r in range(requests):
            keys[r].append(k[r].cpu().numpy().reshape(kv, d).astype(np.float64))
            vals[r].append(v[r].cpu().numpy().reshape(kv, d).astype(np.float64))
            kk, vv, qq = np.stack(keys[r], 1), np.stack(vals[r], 1), q[r].cpu().numpy().reshape(heads, d)
            for h in range(heads):
                s = kk[h // 2] @ qq[h] * 0.125
                w = np.exp(s - s.max())
                want = w / w.sum() @ vv[h // 2]
                # codes are within half a step, once or twice rounded a step, of at most 2 * 4.5 / 127: scores move by
                # a step * sqrt(d) / 8, results by that and a step more
                assert np.abs(out[r].cpu().numpy().reshape(heads, d)[h] - want).max() < 0.25
    assert lens.cpu().tolist() == [40] * 3 and count.item() == pages - 9


# ---------------------------------------------------------------- refusals
def test_refusals(torch):
    p = pkg()
    pr = Problem(torch, 37, [40], [2], 4, 2, 64, 16, "fp32", "int8")
    kc, vc, ks, vs = pr.codes[0], pr.codes[1], pr.scales[0], pr.scales[1]
    table, lens, starts, q, ws = ints(torch, pr.table), ints(torch, pr.lens), ints(torch, pr.starts), pr.tq, pr.workspace

    def attend(**kw):
        a = dict(q=q, kc=kc, vc=vc, ks=ks, vs=vs, table=table, lens=lens, starts=starts, heads=4, scale=0.125, ws=ws)
        a.update(kw)
        return p.cache_attention(a["q"], a["kc"], a["vc"], a["ks"], a["vs"], a["table"], a["lens"], a["starts"], a["heads"], a["scale"], a["ws"],
                                 **{k: v for k, v in kw.items() if k in ("out", "lse")})

    attend()
    bad = [dict(q=q.double()), dict(q=q.cpu()), dict(q=q[:, :-1]), dict(q=q.t()), dict(heads=3), dict(heads=8), dict(kc=kc.float()), dict(kc=kc[0]),
           dict(vc=vc[:-1]), dict(vc=vc.view(torch.float8_e4m3fn)), dict(ks=ks[:-1]), dict(vs=vs.double()), dict(table=table.long()), dict(table=table[0]),
           dict(lens=lens.cpu()), dict(starts=starts[:-1]), dict(scale=float("nan")), dict(scale=float("inf")), dict(ws=ws[:1000]), dict(ws=ws[1:]),
           dict(out=torch.empty_like(q).bfloat16()), dict(out=torch.empty_like(q)[:1]), dict(lse=torch.empty((2, 3), device="cuda")),
           dict(kc=kc.transpose(1, 2))]
    for kw in bad:
        with pytest.raises(p.AttentionError):
            attend(**kw)
    for d, page in ((24, 16), (144, 16), (64, 24), (64, 8), (64, 272)):  # shapes that the cache does not have
        c, s = torch.zeros((2, 2, page, d), dtype=torch.int8, device="cuda"), torch.ones((2, 2), device="cuda")
        with pytest.raises(p.AttentionError):
            attend(q=torch.zeros((2, 4 * d), device="cuda"), kc=c, vc=c, ks=s, vs=s)
        with pytest.raises(p.AttentionError):
            p.cache_append(torch.zeros((1, 2 * d), device="cuda"), torch.zeros((1, 2 * d), device="cuda"), ints(torch, [0]), c, c.clone(), s, s.clone())
    k = torch.zeros((3, 128), device="cuda")
    slots = ints(torch, [0, 1, 2])
    for a in ((k, k.bfloat16(), slots), (k[:, :64], k[:, :64], slots), (k, k[:2], slots), (k, k, slots[:2]), (k, k, slots.long()), (k.half(), k.half(), slots)):
        with pytest.raises(p.AttentionError):
            p.cache_append(*a, kc, vc, ks, vs)
    n = ints(torch, [1])
    plan = lambda lens, new, table, free, count, page, tokens, **kw: p.cache_plan(lens, new, table, free, count, page, tokens, **kw)  # noqa: E731
    for a, kw in (((n, ints(torch, [1, 2]), ints(torch, [[0]]), n, n, 16, 1), {}), ((n, n, ints(torch, [0]), n, n, 16, 1), {}),
                  ((n, n, ints(torch, [[0]]), n, ints(torch, [1, 1]), 16, 1), {}), ((n, n, ints(torch, [[0]]), n, n, 0, 1), {}),
                  ((n, n, ints(torch, [[0]]), n, n, 16, -1), {}), ((n, n, ints(torch, [[0]]), n, n, 16, 1), {"lens_out": n}),
                  ((n.cpu(), n, ints(torch, [[0]]), n, n, 16, 1), {}), ((n, n, ints(torch, [[0]]), n, n, 16, 1), {"slots": ints(torch, [0, 0])})):
        with pytest.raises(p.AttentionError):
            plan(*a, **kw)
    big = torch.zeros(16385, dtype=torch.int32, device="cuda")
    with pytest.raises(p.AttentionError):
        plan(big, big, torch.zeros((16385, 1), dtype=torch.int32, device="cuda"), n, n, 16, 0)
    with pytest.raises(p.AttentionError):
        p.cache_release(n, n, ints(torch, [[0]]), n.clone(), n, 16, lens_out=n)
    assert p.lib().df_attn_last_status() != p.DF_OK and p.sync_status() == 0
