"""Measured cases of the operators that serve a batch of requests over a paged cache held in 8 bits, and score what comes out:

  plan       block tables, slot maps and positions of a step's new tokens, built on the GPU from request lengths; with
             "release" the pages of finished requests go back first
  append     the new tokens' K and V rows put into the cache: 8 bits each, one power-of-two scale per page and head
  attend     ragged queries of all requests against their cached tokens
  logprobs   log probabilities of given tokens with entropy and top alternatives; "backward" is its gradient

`run` computes a case in plain 32-bit torch operations, or, where `own` is set, by this library's calls.

Cache layout: codes [pages, kv_heads, page, head_dim] (torch.int8 or torch.float8_e4m3fn), scales [pages, kv_heads] fp32; the value of a
code is code * scale of its page and head. Token t of request r lies in page block_table[r, t // page] at row t % page.
"""
import math
import random

import torch

own = False

WORKSPACE_BYTES = 33554432  # what the attention call is lent: zeroed once, kept by the program


# ---------------------------------------------------------------- cases
def _attend(name, requests, heads, kv_heads, head_dim, shortest, longest, new, dtype, code, page):
    """Request lengths lie between `shortest` and `longest` (most of them short), each with `new` query tokens."""
    c = {"kind": "attend", "requests": requests, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "shortest": shortest, "longest": longest,
         "new": new, "dtype": dtype, "code": code, "page": page}
    return dict(c, name=name) if name else c


def _append(name, requests, new, kv_heads, head_dim, dtype, code, page):
    c = {"kind": "append", "requests": requests, "new": new, "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "code": code, "page": page}
    return dict(c, name=name) if name else c


def _plan(name, requests, longest, prompts, prompt, page, release):
    """`prompts` of the requests bring up to `prompt` new tokens each, the others one."""
    c = {"kind": "plan", "requests": requests, "longest": longest, "prompts": prompts, "prompt": prompt, "page": page, "release": release}
    return dict(c, name=name) if name else c


def _logprobs(name, rows, vocab, top, dtype, backward):
    c = {"kind": "logprobs", "rows": rows, "vocab": vocab, "top": top, "dtype": dtype, "backward": backward}
    return dict(c, name=name) if name else c


def listed():
    return [
        # Generating text for one user with GPT-2 small's heads: a few hundred cached tokens, where latency counts.
        _attend("attend_one_t300", 1, 12, 12, 64, 300, 300, 1, "fp32", "int8", 16),
        # A batch of chat requests of very different lengths, grouped heads, bf16 activations: ordinary serving.
        _attend("attend_b32_ragged", 32, 32, 8, 128, 200, 16000, 1, "bf16", "e4m3", 16),
        # One very long context with a K/V head for every query head: the cache's bytes alone.
        _attend("attend_long_t131073", 1, 16, 16, 128, 131073, 131073, 1, "fp32", "int8", 64),
        # Drafted tokens of many requests verified at once: five query tokens each.
        _attend("attend_verify_b16_q5", 16, 32, 8, 128, 1000, 6000, 5, "bf16", "e4m3", 32),
        # A further piece of two prompts over a long history: many query tokens, bound by arithmetic.
        _attend("attend_piece_q500", 2, 12, 12, 64, 6000, 9000, 500, "fp32", "int8", 16),
        # One token of each of 64 requests put into the cache.
        _append("append_b64", 64, 1, 8, 128, "bf16", "e4m3", 16),
        # The prompts of a step: 8 K tokens put into the cache.
        _append("append_prompts", 5, 1641, 12, 64, "fp32", "int8", 16),
        # Every request generates a token.
        _plan("plan_b64", 64, 4000, 0, 1, 16, False),
        # A busy server: finished requests leave, some bring prompts, the others a token.
        _plan("plan_b512_prompts", 512, 8000, 16, 2000, 16, True),
        # The log probabilities of a step of eight requests, with 20 alternatives for the user.
        _logprobs("logprobs_8x50257", 8, 50257, 20, "fp32", False),
        # Scoring a batch of texts in bf16 logits, five alternatives.
        _logprobs("logprobs_1024x50257", 1024, 50257, 5, "bf16", False),
        # The gradient of a policy's log probabilities and entropy over a chunk of logits.
        _logprobs("logprobs_grad_512x50257", 512, 50257, 0, "fp32", True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("attend", "attend", "attend", "append", "append", "plan", "logprobs", "logprobs"))
    code, dtype = rng.choice(("int8", "e4m3")), rng.choice(("fp32", "bf16"))
    if kind == "attend":
        kv_heads, group, head_dim = rng.choice((1, 2, 4, 8, 12)), rng.choice((1, 1, 2, 4, 7, 8)), rng.choice((32, 64, 64, 80, 96, 128, 128))
        page, new = rng.choice((16, 32, 48, 64, 128)), rng.choice((1, 1, 1, rng.randint(2, 8), _log(rng, 9, 400)))
        requests = _log(rng, 1, 64) if new <= 8 else rng.randint(1, 4)
        # the cached bytes stay below the longest listed context's, the scores of the plain form below 2 GB, the products below attend_piece_q500's
        most = min(100000, 130000 * 16 * 128 // (requests * kv_heads * head_dim), 500_000_000 // (requests * kv_heads * group * new),
                   6_000_000_000 // (requests * kv_heads * group * new * head_dim))
        longest = _log(rng, new, max(new + 1, most))
        return _attend(None, requests, kv_heads * group, kv_heads, head_dim, _log(rng, new, longest), longest, new, dtype, code, page)
    if kind == "append":
        requests = _log(rng, 1, 256)
        return _append(None, requests, rng.choice((1, 1, _log(rng, 2, max(3, 8000 // requests)))), rng.choice((1, 2, 4, 8, 12)), rng.choice((32, 64, 80, 128)),
                       dtype, code, rng.choice((16, 32, 64, 128)))
    if kind == "plan":
        requests = _log(rng, 1, 1000)
        return _plan(None, requests, _log(rng, 10, 8000), rng.randint(0, max(0, min(16, requests // 2))), _log(rng, 2, 2000), rng.choice((16, 32, 64)),
                     rng.random() < 0.5)
    vocab = _log(rng, 300, 130000)
    rows = _log(rng, 1, max(2, 25_000_000 // vocab))
    return _logprobs(None, rows, vocab, rng.choice((0, 1, 5, 20)), dtype, rng.random() < 0.4)


def _lengths(case):
    """The requests' lengths, part of the case itself: a long tail of short ones up to the longest."""
    rng = random.Random("%(requests)d %(shortest)d %(longest)d" % case)
    n = [_log(rng, case["shortest"], case["longest"]) for _ in range(case["requests"])]
    n[rng.randrange(len(n))] = case["longest"]
    return n


def _plan_lengths(case):
    """Lengths before the step, new tokens, and which requests have finished."""
    rng = random.Random("%(requests)d %(longest)d %(prompts)d %(prompt)d" % case)
    n = case["requests"]
    lens = [_log(rng, 1, case["longest"]) for _ in range(n)]
    new = [1] * n
    finished = [0] * n
    for r in rng.sample(range(n), case["prompts"]):
        finished[r] = 1 if case["release"] else 0
        new[r] = rng.randint(1, case["prompt"])
    return lens, new, finished


def _taken(codes, *index):
    """codes[index], moved as bytes."""
    return codes.view(torch.uint8)[index].view(codes.dtype)


# ---------------------------------------------------------------- inputs
def _generator(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _codes(gen, code, shape):
    """Codes as quantised activations have them: the largest of a page near the type's end."""
    x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    if code == "int8":
        return x.mul_(30.0).round_().clamp_(-127, 127).to(torch.int8)
    return x.mul_(110.0).clamp_(-448, 448).to(torch.float8_e4m3fn)


def _scales(gen, code, shape):
    e = torch.randint(-1, 2, shape, generator=gen, device="cuda", dtype=torch.int32) + (-5 if code == "int8" else -7)
    return torch.ldexp(torch.ones(shape, device="cuda"), e)


def prepare(case, seed):
    gen = _generator(seed)
    s = dict(case)
    kind = case["kind"]
    dtype = torch.bfloat16 if case.get("dtype") == "bf16" else torch.float32

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)

    if kind == "attend":
        lens, page, kv, d = _lengths(case), case["page"], case["kv_heads"], case["head_dim"]
        pages = [-(-n // page) for n in lens]
        n_pages = sum(pages) + 3
        order = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)
        table = torch.zeros((len(lens), max(pages)), dtype=torch.int32, device="cuda")
        used = 0
        for r, n in enumerate(pages):
            table[r, :n] = order[used:used + n]
            used += n
        s["table"] = table
        s["k_cache"], s["v_cache"] = (_codes(gen, case["code"], (n_pages, kv, page, d)) for _ in range(2))
        s["k_scale"], s["v_scale"] = (_scales(gen, case["code"], (n_pages, kv)) for _ in range(2))
        s["lens"] = _int32(lens)
        s["starts"] = _int32([case["new"] * r for r in range(len(lens) + 1)])
        s["q"] = normal(case["new"] * len(lens), case["heads"] * d)
        s["scale"] = d ** -0.5
        s["workspace"] = torch.zeros(WORKSPACE_BYTES, dtype=torch.uint8, device="cuda")
    elif kind == "append":
        n, new, page, kv, d = case["requests"], case["new"], case["page"], case["kv_heads"], case["head_dim"]
        rng = random.Random(seed)
        lens = [rng.randrange(4 * page) for _ in range(n)]
        per = -(-(4 * page + new) // page)
        n_pages = n * per
        table = torch.randperm(n_pages, generator=gen, device="cuda").view(n, per)
        pos = _int32(lens).long()[:, None] + torch.arange(new, device="cuda")[None]
        s["slots"] = (torch.gather(table, 1, pos // page) * page + pos % page).reshape(-1).to(torch.int32)
        s["k"], s["v"] = (normal(n * new, kv * d) for _ in range(2))
        s["k_cache"], s["v_cache"] = (_codes(gen, case["code"], (n_pages, kv, page, d)) for _ in range(2))
        s["k_scale"], s["v_scale"] = (_scales(gen, case["code"], (n_pages, kv)) for _ in range(2))
    elif kind == "plan":
        lens, new, finished = _plan_lengths(case)
        page = case["page"]
        width = -(-(case["longest"] + max(new)) // page) + 1
        held = [-(-n // page) for n in lens]
        need = sum(-(-(n + m) // page) for n, m in zip(lens, new))
        n_pages = need + sum(held) + 64
        order = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)
        s["table"] = torch.zeros((case["requests"], width), dtype=torch.int32, device="cuda")
        used = 0
        for r, n in enumerate(held):
            s["table"][r, :n] = order[used:used + n]
            used += n
        s["free"] = torch.zeros(n_pages, dtype=torch.int32, device="cuda")  # a stack: the first `count` entries are free pages
        s["free"][:n_pages - used] = order[used:]
        s["count"] = _int32([n_pages - used])
        s["lens"], s["new"], s["finished"] = _int32(lens), _int32(new), _int32(finished)
        s["n_tokens"] = sum(new)
        # where the step's results go, kept from step to step
        n, t = case["requests"], s["n_tokens"]
        s["kept"] = [torch.empty(m, dtype=torch.int32, device="cuda") for m in (n, n + 1, t, t, 2, n, 1)]
    else:
        rows, vocab = case["rows"], case["vocab"]
        x = torch.randn((rows, vocab), generator=gen, device="cuda", dtype=torch.float32).mul_(2.5)
        s["targets"] = torch.randint(0, vocab, (rows,), generator=gen, device="cuda", dtype=torch.int32)
        x.scatter_add_(1, s["targets"].long()[:, None], torch.full((rows, 1), 9.0, device="cuda"))  # a model that has learned something
        s["logits"] = x.to(dtype)
        s["inverse_temperature"] = 1.0 / 0.9
        if case["backward"]:
            z = s["logits"].float() * s["inverse_temperature"]
            m = z.max(1, keepdim=True).values
            e = torch.exp(z - m)
            total = e.sum(1, keepdim=True)
            s["lse"] = (m + torch.log(total)).squeeze(1)
            s["entropy"] = (torch.log(total) - (e * (z - m)).sum(1, keepdim=True) / total).squeeze(1)
            s["grad_logp"], s["grad_entropy"] = (torch.randn(rows, generator=gen, device="cuda") for _ in range(2))
            s["d_logits"] = torch.empty_like(s["logits"])
    return s


# ---------------------------------------------------------------- one pass
def run(s):
    return _own(s) if own else {"attend": _plain_attend, "append": _plain_append, "plan": _plain_plan, "logprobs": _plain_logprobs}[s["kind"]](s)


def _own(s):
    from __graft_entry__ import load_package
    df = load_package()
    if s["kind"] == "attend":
        return df.cache_attention(s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["table"], s["lens"], s["starts"], s["heads"], s["scale"],
                                  s["workspace"])
    if s["kind"] == "append":
        return df.cache_append(s["k"], s["v"], s["slots"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
    if s["kind"] == "plan":
        lens_out, starts, slots, positions, state, kept_lens, kept_count = s["kept"]
        lens, count = s["lens"], s["count"]
        if s["release"]:
            lens, count = df.cache_release(lens, s["finished"], s["table"], s["free"], count, s["page"], lens_out=kept_lens, count_out=kept_count)
        df.cache_plan(lens, s["new"], s["table"], s["free"], count, s["page"], s["n_tokens"], lens_out=lens_out, starts=starts, slots=slots,
                      positions=positions, state=state)
        return lens_out, starts, slots, positions, state, s["table"], s["free"]
    if s["backward"]:
        return df.token_logprobs_backward(s["logits"], s["targets"], s["lse"], s["entropy"], s["grad_logp"], s["grad_entropy"], s["inverse_temperature"],
                                          d_logits=s["d_logits"])
    return df.token_logprobs(s["logits"], s["targets"], s["inverse_temperature"], s["top"])


def _plain_attend(s):
    n, new, kv, d, page = s["requests"], s["new"], s["kv_heads"], s["head_dim"], s["page"]
    group, table = s["heads"] // kv, s["table"].long()
    tokens = table.shape[1] * page

    def cached(codes, scales):  # [request, head, token, dim]
        x = _taken(codes, table).float() * scales[table][..., None, None]
        return x.permute(0, 2, 1, 3, 4).reshape(n, kv, tokens, d)

    q = s["q"].float().view(n, new, kv, group, d).permute(0, 2, 1, 3, 4).reshape(n, kv, new * group, d)
    scores = (q @ cached(s["k_cache"], s["k_scale"]).transpose(2, 3)) * s["scale"]
    last = s["lens"].long()[:, None] - new + torch.arange(new, device="cuda")[None]  # the last key that a query token sees
    seen = torch.arange(tokens, device="cuda")[None, None] <= last[:, :, None]
    scores = scores.masked_fill(~seen.repeat_interleave(group, 1)[:, None], float("-inf"))
    top = scores.max(3, keepdim=True).values
    p = torch.exp(scores - top)
    total = p.sum(3, keepdim=True)
    out = (p @ cached(s["v_cache"], s["v_scale"])) / total
    lse = (top + torch.log(total)).squeeze(3)
    back = lambda x, *tail: x.view(n, kv, new, group, *tail).transpose(1, 2).reshape(n * new, -1)  # noqa: E731
    return back(out, d).to(s["q"].dtype), back(lse)


def _plain_append(s):
    page, kv, d = s["page"], s["kv_heads"], s["head_dim"]
    slots = s["slots"].long()
    pages, rows = slots // page, slots % page
    first = torch.ones_like(pages, dtype=torch.bool)
    first[1:] = pages[1:] != pages[:-1]  # the tokens of a page lie together
    run_of = torch.cumsum(first, 0) - 1
    touched, kept_rows = pages[first], rows[first]
    biggest, at_one = (127.0, 127 / 128) if s["code"] == "int8" else (448.0, 448 / 512)
    for x, codes, scales in ((s["k"], s["k_cache"], s["k_scale"]), (s["v"], s["v_cache"], s["v_scale"])):
        x = x.float().view(-1, kv, d)
        amax = torch.zeros((touched.shape[0], kv), device="cuda").index_reduce_(0, run_of, x.abs().amax(2), "amax")
        mantissa, exponent = torch.frexp(amax)
        exponent = exponent - math.frexp(biggest)[1] + (mantissa > at_one).int()
        exponent = torch.where(amax > 0, exponent, -126).clamp(min=-126)
        old = scales[touched]
        new = torch.ldexp(torch.ones_like(amax), exponent)
        new = torch.where(kept_rows[:, None] > 0, torch.maximum(old, new), new)
        ratio = torch.where(kept_rows[:, None] > 0, old / new, torch.ones_like(new))
        before = _taken(codes, touched)
        held = before.float() * ratio[..., None, None]
        fresh = x / new[run_of][..., None]
        if s["code"] == "int8":
            held, fresh = held.round(), fresh.round()
        keep = torch.arange(page, device="cuda")[None] < kept_rows[:, None]
        bits = torch.where(keep[:, None, :, None], held.to(codes.dtype).view(torch.uint8), before.view(torch.uint8))
        raw = codes.view(torch.uint8)
        raw[touched] = bits
        raw[pages, :, rows] = fresh.to(codes.dtype).view(torch.uint8)
        scales[touched] = new
    return s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]


def _plain_plan(s):
    page, table, free = s["page"], s["table"], s["free"]
    lens, new, count = s["lens"].long(), s["new"].long(), s["count"].long()
    if s["release"]:
        held = torch.where(s["finished"] > 0, (lens + page - 1) // page, 0)
        owner = torch.repeat_interleave(torch.arange(s["requests"], device="cuda"), held)
        nth = torch.arange(owner.shape[0], device="cuda") - (torch.cumsum(held, 0) - held)[owner]
        free[count + torch.arange(owner.shape[0], device="cuda")] = table[owner, nth]
        count = count + held.sum()
        lens = torch.where(s["finished"] > 0, 0, lens)
    starts = torch.nn.functional.pad(torch.cumsum(new, 0), (1, 0))
    has = (lens + page - 1) // page
    need = (lens + new + page - 1) // page - has
    owner = torch.repeat_interleave(torch.arange(s["requests"], device="cuda"), need)
    taken = torch.arange(owner.shape[0], device="cuda")
    nth = taken - (torch.cumsum(need, 0) - need)[owner]
    table[owner, has[owner] + nth] = free[count - 1 - taken]
    of = torch.repeat_interleave(torch.arange(s["requests"], device="cuda"), new)
    positions = lens[of] + torch.arange(of.shape[0], device="cuda") - starts[of]
    slots = table[of, positions // page].long() * page + positions % page
    state = torch.cat((count - need.sum(), torch.zeros(1, dtype=torch.long, device="cuda")))
    return tuple(x.int() for x in (lens + new, starts, slots, positions, state)) + (table, free)


def _plain_logprobs(s):
    x = s["logits"].float()
    z = x * s["inverse_temperature"]
    at = s["targets"].long()[:, None]
    if s["backward"]:
        logp = z - s["lse"][:, None]
        p = torch.exp(logp)
        g, h = s["grad_logp"][:, None], s["grad_entropy"][:, None]
        d = -p * (g + h * (logp + s["entropy"][:, None]))
        d.scatter_add_(1, at, g)
        return (d * s["inverse_temperature"]).to(s["logits"].dtype)
    m = z.max(1, keepdim=True).values
    e = torch.exp(z - m)
    total = e.sum(1, keepdim=True)
    lse = m + torch.log(total)
    entropy = torch.log(total) - (e * (z - m)).sum(1, keepdim=True) / total
    best = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :s["top"]]  # ties: the lowest index first
    return tuple(v.squeeze(1) for v in (z.gather(1, at) - lse, entropy, lse)) + (best.int(), z.gather(1, best) - lse)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    kind = case["kind"]
    elt = 2 if case.get("dtype") == "bf16" else 4
    if kind == "attend":
        lens, kv, d, page, new = _lengths(case), case["kv_heads"], case["head_dim"], case["page"], case["new"]
        rows = new * len(lens) * case["heads"]
        pages = sum(-(-n // page) for n in lens)
        pairs = sum(new * n - new * (new - 1) // 2 for n in lens) * case["heads"]
        return {"bytes": 2 * sum(lens) * kv * d + 8 * pages * kv + 4 * pages + rows * (2 * d * elt + 4), "flops": 4 * pairs * d}
    if kind == "append":
        n = case["requests"] * case["new"]
        return {"bytes": 2 * n * case["kv_heads"] * case["head_dim"] * (elt + 1) + 4 * n, "flops": 4 * n * case["kv_heads"] * case["head_dim"]}
    if kind == "plan":
        lens, new, finished = _plan_lengths(case)
        page = case["page"]
        freed = sum(-(-n // page) for n, f in zip(lens, finished) if f and case["release"])
        grown = sum(-(-(n + m) // page) - -(-n // page) for n, m in zip(lens, new))
        return {"bytes": 8 * sum(new) + 16 * len(new) + 8 * max(0, grown) + 8 * freed, "flops": 4 * sum(new)}
    elements = case["rows"] * case["vocab"]
    return {"bytes": elements * elt * (2 if case["backward"] else 1) + case["rows"] * (24 + 8 * case["top"]), "flops": 6 * elements}


# ---------------------------------------------------------------- in 64 bits
def exact(case, seed):
    if case["kind"] == "plan":
        return None  # whole numbers throughout
    return {"attend": _exact_attend, "append": _exact_append, "logprobs": _exact_logprobs}[case["kind"]](prepare(case, seed))


def _exact_attend(s):
    """Request by request and head by head, tokens gathered one after another."""
    new, kv, d, page = s["new"], s["kv_heads"], s["head_dim"], s["page"]
    group = s["heads"] // kv
    out = torch.zeros((s["q"].shape[0], s["heads"], d), dtype=torch.float64, device="cuda")
    lse = torch.zeros((s["q"].shape[0], s["heads"]), dtype=torch.float64, device="cuda")
    for r, n in enumerate(_lengths(s)):
        t = torch.arange(n, device="cuda")
        pages = s["table"][r].long()[t // page]
        for h in range(kv):
            k = _taken(s["k_cache"], pages, h, t % page).double() * s["k_scale"][pages, h].double()[:, None]
            v = _taken(s["v_cache"], pages, h, t % page).double() * s["v_scale"][pages, h].double()[:, None]
            for j0 in range(0, new, 64):
                j = torch.arange(j0, min(new, j0 + 64), device="cuda")
                q = s["q"].view(-1, s["heads"], d)[r * new + j, h * group:(h + 1) * group].double()
                score = torch.einsum("jgd,td->jgt", q, k) * s["scale"]
                score = score.masked_fill(t[None, None] > (n - new + j)[:, None, None], float("-inf"))
                l = torch.logsumexp(score, 2)
                lse[r * new + j, h * group:(h + 1) * group] = l
                out[r * new + j, h * group:(h + 1) * group] = torch.einsum("jgt,td->jgd", torch.exp(score - l[..., None]), v)
    return out.flatten(1), lse


def _exact_append(s):
    """Codes are whole numbers or 8-bit floats: the values they stand for follow from the scales, which are computed here page by page."""
    page, kv, d = s["page"], s["kv_heads"], s["head_dim"]
    slots = s["slots"].tolist()
    runs, at = [], 0
    while at < len(slots):
        end = at + 1
        while end < len(slots) and slots[end] // page == slots[at] // page:
            end += 1
        runs.append((at, end))
        at = end
    biggest = 127.0 if s["code"] == "int8" else 448.0
    found = []
    for x, codes, scales in ((s["k"], s["k_cache"], s["k_scale"]), (s["v"], s["v_cache"], s["v_scale"])):
        x = x.double().view(-1, kv, d)
        values, powers = codes.double(), scales.double()
        for a, b in runs:
            p, row = slots[a] // page, slots[a] % page
            need = torch.exp2(torch.ceil(torch.log2(x[a:b].abs().amax((0, 2)) / biggest)))
            if row:
                need = torch.maximum(need, powers[p])
                values[p, :, :row] = _rounded(values[p, :, :row] * (powers[p] / need)[:, None, None], s["code"])
            powers[p] = need
            values[p, :, row:row + b - a] = _rounded(x[a:b].transpose(0, 1) / need[:, None, None], s["code"])
        found.append((None if s["code"] == "int8" else values, powers))
    return found[0][0], found[1][0], found[0][1], found[1][1]


def _rounded(x, code):
    if code == "int8":
        return torch.round(x)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)  # three bits behind the first, none below 2^-9
    return torch.round(x / step) * step


def _exact_logprobs(s):
    x = s["logits"]
    rows = [[], [], [], []] if not s["backward"] else [[]]
    for r in range(0, x.shape[0], 64):
        z = x[r:r + 64].double() * s["inverse_temperature"]
        at = s["targets"][r:r + 64].long()
        logp = z - torch.logsumexp(z, 1, keepdim=True)
        picked = logp[torch.arange(len(at), device="cuda"), at]
        if s["backward"]:
            p, one = logp.exp(), torch.zeros_like(logp)
            one[torch.arange(len(at), device="cuda"), at] = 1
            g, h = s["grad_logp"][r:r + 64].double()[:, None], s["grad_entropy"][r:r + 64].double()[:, None]
            entropy = -(p * logp).sum(1, keepdim=True)
            rows[0].append(s["inverse_temperature"] * (g * (one - p) - h * p * (logp + entropy)))
            continue
        rows[0].append(picked)
        rows[1].append(-(logp.exp() * logp).sum(1))
        rows[2].append(torch.logsumexp(z, 1))
        rows[3].append(torch.topk(logp, s["top"], 1).values if s["top"] else logp[:, :0])
    if s["backward"]:
        return torch.cat(rows[0])
    logp, entropy, lse, best = (torch.cat(v) for v in rows)
    return logp, entropy, lse, None, best
