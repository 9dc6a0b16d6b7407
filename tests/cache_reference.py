"""Plain 64-bit forms of the paged-cache and log-probability operators, for their tests (numpy and torch on the CPU)."""
import numpy as np

BIGGEST = {"int8": 127.0, "e4m3": 448.0}


def round_to_code(x, code):
    """Nearest code value, ties to even, of float64 values already divided by their scale (and within the code's range)."""
    if code == "int8":
        return np.rint(x)
    step = np.exp2(np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** -6))) - 3)
    return np.rint(x / step) * step


def scale_for(amax, code):
    """Smallest power of two, 2^-126 or above, that holds amax."""
    e = -126
    if amax > 0:
        e = max(-126, int(np.ceil(np.log2(amax / BIGGEST[code]))) - 2)
        while amax > BIGGEST[code] * 2.0 ** e:
            e += 1
    return 2.0 ** e


def append(x, slots, values, scales, page):
    """One tensor (K or V): x [tokens, heads, d] float64, values [pages, heads, page, d] (what codes stand for without their scale) and scales
    [pages, heads], float64, changed in place. `code` of the values rides along in append.code."""
    code = append.code
    n_slots = values.shape[0] * page
    t = 0
    while t < len(slots):
        if not 0 <= slots[t] < n_slots:
            t += 1
            continue
        p, row = divmod(int(slots[t]), page)
        n = 1
        while t + n < len(slots) and row + n < page and slots[t + n] == slots[t] + n:
            n += 1
        for h in range(values.shape[1]):
            amax = np.abs(x[t:t + n, h]).max()
            need = scale_for(amax, code) if np.isfinite(amax) else np.nan
            if row and not need >= scales[p, h]:
                need = np.nan if np.isnan(need) else scales[p, h]
            if row and scales[p, h] < need:
                values[p, h, :row] = round_to_code(values[p, h, :row] * (scales[p, h] / need), code)
            scales[p, h] = need
            values[p, h, row:row + n] = 0.0 if np.isnan(need) else round_to_code(x[t:t + n, h] / need, code)
        t += n


append.code = "int8"


def plan(lens, new, table, free, count, page, n_tokens):
    """(lens_out, starts, slots, positions, state), table changed in place."""
    lens, new = np.maximum(lens, 0).astype(np.int64), np.maximum(new, 0).astype(np.int64)
    ends = np.cumsum(new)
    starts = np.minimum(np.concatenate(([0], ends)), n_tokens)
    slots, positions = np.full(n_tokens, -1), np.full(n_tokens, -1)
    count = min(max(int(count), 0), len(free))
    bad = [r for r in range(len(lens)) if lens[r] + new[r] > table.shape[1] * page or ends[r] > n_tokens]
    has = -(-lens // page)
    need = -(-(lens + new) // page) - has
    if bad or need.sum() > count:
        return lens, starts, slots, positions, np.array([count, -1 - bad[0] if bad else need.sum() - count])
    at = 0
    for r in range(len(lens)):
        for j in range(need[r]):
            count -= 1
            table[r, has[r] + j] = free[count]
        for j in range(new[r]):
            pos = lens[r] + j
            slots[at], positions[at] = table[r, pos // page] * page + pos % page, pos
            at += 1
    return lens + new, starts, slots, positions, np.array([count, 0])


def release(lens, finished, table, free, count, page):
    """(lens_out, count_out), free changed in place."""
    lens = lens.astype(np.int64).copy()
    for r in range(len(lens)):
        if finished[r]:
            for b in range(min(-(-max(int(lens[r]), 0) // page), table.shape[1])):
                free[count] = table[r, b]
                count += 1
            lens[r] = 0
    return lens, count


def attention(q, k, v, table, lens, starts, page, scale):
    """q [tokens, heads, d], k, v [pages, kv_heads, page, d] float64 (scales applied). Returns out [tokens, heads, d], lse [tokens, heads] and the largest
    sum of magnitudes of a visible score, which its rounding errors go by. Rows outside every request: NaN."""
    tokens, heads, d = q.shape
    group = heads // k.shape[1]
    out, lse, magnitude = np.full(q.shape, np.nan), np.full((tokens, heads), np.nan), 0.0
    for r in range(len(lens)):
        n = min(max(int(lens[r]), 0), table.shape[1] * page)
        pages = table[r, :-(-n // page)]
        if n:
            keys = k[pages].transpose(1, 0, 2, 3).reshape(k.shape[1], -1, d)[:, :n]
            vals = v[pages].transpose(1, 0, 2, 3).reshape(k.shape[1], -1, d)[:, :n]
        q_len = starts[r + 1] - starts[r]
        for j in range(q_len):
            row, see = starts[r] + j, n - q_len + j + 1
            if see <= 0:
                out[row], lse[row] = 0.0, -np.inf
                continue
            for h in range(heads):
                kk = keys[h // group, :see]
                s = kk @ q[row, h] * scale
                magnitude = max(magnitude, float((np.abs(kk) @ np.abs(q[row, h])).max()) * abs(scale))
                m = s.max()
                w = np.exp(s - m)
                lse[row, h] = m + np.log(w.sum())
                out[row, h] = w / w.sum() @ vals[h // group, :see]
    return out, lse, magnitude


def logprobs(x, targets, scale, top):
    """x [rows, cols] float64 without NaN and +inf. Returns logp, entropy, lse, ids, their log probabilities."""
    rows, cols = x.shape
    z = x * scale
    logp, entropy, lse = np.zeros(rows), np.zeros(rows), np.zeros(rows)
    ids, best = np.zeros((rows, top), int), np.zeros((rows, top))
    for r in range(rows):
        m = z[r].max()
        if m == -np.inf:
            lse[r], everything = -np.inf, np.full(cols, -np.inf)
        else:
            everything = (z[r] - m) - np.log(np.exp(z[r] - m).sum())  # from differences: m alone may be larger than 2^53 of them
            lse[r] = m + np.log(np.exp(z[r] - m).sum())
            seen = everything > -np.inf
            entropy[r] = -(np.exp(everything[seen]) * everything[seen]).sum()
        if 0 <= targets[r] < cols:
            logp[r] = everything[targets[r]]
        ids[r] = np.argsort(-x[r], kind="stable")[:top]
        best[r] = everything[ids[r]]
    return logp, entropy, lse, ids, best


def logprobs_backward(x, targets, scale, g, h):
    z = x * scale
    m = z.max(1, keepdims=True)
    lse = m + np.log(np.exp(z - m).sum(1, keepdims=True))
    logp = z - lse
    p = np.exp(logp)
    entropy = -(p * np.where(p > 0, logp, 0.0)).sum(1, keepdims=True)
    inside = (targets >= 0) & (targets < x.shape[1])
    g = np.where(inside, g, 0.0)[:, None]
    one = np.zeros_like(x)
    one[np.flatnonzero(inside), targets[inside]] = 1.0
    return scale * (g * (one - p) - h[:, None] * p * np.where(p > 0, logp + entropy, 0.0))
