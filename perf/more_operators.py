"""Measured cases of the operators that a training step needs behind its last block:

  head      softmax cross entropy of given tokens from hidden states and the output weight, over a vocabulary whose logits are
            not kept; "backward" is its gradient with respect to both
  orth      matrices orthogonalised by Newton-Schulz products
  muon      a step of an optimiser on matrices of one shape: momentum, orthogonalised, applied to the parameters

`run` computes a case in plain 32-bit torch operations, or, where `own` is set, by this library's calls.
"""
import math
import random

import torch

own = False

COEFFICIENTS = (3.4445, -4.7750, 2.0315)  # the odd polynomial of five steps that brings every singular value near 1
EPS = 1e-7


# ---------------------------------------------------------------- cases
def _head(name, rows, vocab, width, dtype, padded, backward):
    """`padded` percent of the rows have no target (-1), as the ends of texts of different lengths."""
    c = {"kind": "head", "rows": rows, "vocab": vocab, "width": width, "dtype": dtype, "padded": padded, "backward": backward}
    return dict(c, name=name) if name else c


def _orth(name, count, rows, cols, dtype, steps):
    c = {"kind": "orth", "count": count, "rows": rows, "cols": cols, "dtype": dtype, "steps": steps}
    return dict(c, name=name) if name else c


def _muon(name, count, rows, cols, nesterov, decay):
    c = {"kind": "muon", "count": count, "rows": rows, "cols": cols, "nesterov": nesterov, "decay": decay}
    return dict(c, name=name) if name else c


def listed():
    return [
        # The loss of a few tokens, one of each of eight short texts: latency and the weight's bytes.
        _head("loss_8x50257_bf16", 8, 50257, 768, "bf16", 0, False),
        # Evaluation of a batch of texts in bf16.
        _head("loss_4096x50257_bf16", 4096, 50257, 768, "bf16", 0, False),
        # The loss of a GPT-2 training step in fp32: 2048 rows.
        _head("loss_2048x50257_fp32", 2048, 50257, 768, "fp32", 0, False),
        # The gradient over a chunk of rows as the loss head takes them, fp32.
        _head("grad_512x50257_fp32", 512, 50257, 768, "fp32", 0, True),
        # The gradient of a whole batch of texts in bf16.
        _head("grad_8192x50257_bf16", 8192, 50257, 768, "bf16", 0, True),
        # Fine-tuning with padded texts, another tokenizer and an odd width.
        _head("grad_777x10007_fp32", 777, 10007, 330, "fp32", 30, True),
        # One attention projection of GPT-2 small: few tiles, where latency counts.
        _orth("orth_768x768", 1, 768, 768, "fp32", 5),
        # Small odd matrices of a narrow model, taller than wide.
        _orth("orth_6x515x131", 6, 515, 131, "fp32", 5),
        # The gradient of a large projection, held in bf16.
        _orth("orth_1024x4096_bf16", 1, 1024, 4096, "bf16", 5),
        # A step on the attention projections of GPT-2 small: 12 layers of four.
        _muon("muon_48x768x768", 48, 768, 768, True, 0.1),
        # The same on one layer of a narrow model: odd sides, momentum without a look ahead.
        _muon("muon_4x200x330", 4, 200, 330, False, 0.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("head", "head", "head", "head", "orth", "orth", "muon"))
    if kind == "head":
        backward = rng.random() < 0.5
        dtype = rng.choice(("fp32", "bf16"))
        width = rng.choice((64, 256, 512, 768, 768, 1024, _log(rng, 32, 2000)))
        vocab = rng.choice((50257, _log(rng, 300, 130000), _log(rng, 300, 130000)))
        # the products below those of the largest listed case (a third of them for fp32), the plain form's logits below 2 GB
        most = min((300_000_000_000 if dtype == "bf16" else 100_000_000_000) // (vocab * width), 400_000_000 // vocab, 8192)
        return _head(None, _log(rng, 1, max(2, most)), vocab, width, dtype, rng.choice((0, 0, 10, 50)), backward)
    count = rng.choice((1, 1, rng.randint(2, 12)))
    small = _log(rng, 16, 1200)
    large = min(4096, int(small * math.exp(rng.uniform(0.0, 2.0))))
    while count > 1 and count * small * small * large > 6_000_000_000:
        count -= 1
    rows, cols = rng.choice(((small, large), (large, small)))
    if kind == "orth":
        return _orth(None, count, rows, cols, rng.choice(("fp32", "bf16")), rng.choice((5, 5, 3, 1)))
    return _muon(None, count, rows, cols, rng.random() < 0.5, rng.choice((0.0, 0.1)))


# ---------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = dict(case)
    dtype = torch.bfloat16 if case.get("dtype") == "bf16" else torch.float32

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)

    if case["kind"] == "head":
        rows, vocab, width = case["rows"], case["vocab"], case["width"]
        s["weight"] = normal(vocab, width).mul_(width ** -0.5).to(dtype)
        targets = torch.randint(0, vocab, (rows,), generator=gen, device="cuda", dtype=torch.int32)
        # hidden states behind a norm, of a model that has learned something: its tokens' logits are above the others
        s["x"] = (normal(rows, width) + 7.0 * s["weight"][targets.long()].float()).to(dtype)
        padded = torch.randint(0, 100, (rows,), generator=gen, device="cuda") < case["padded"]
        s["targets"] = torch.where(padded, -1, targets).to(torch.int32)
        s["scale"] = 1.0
        if case["backward"]:
            s["lse"] = _statistics(s)[1]
            s["grad"] = normal(rows).mul_(0.25).add_(1.0) / rows  # a mean over the batch, rows weighted
    elif case["kind"] == "orth":
        # a gradient: a few strong directions and noise
        n, rows, cols = case["count"], case["rows"], case["cols"]
        s["update"] = (normal(n, rows, cols) * 1e-3 + 2e-3 * normal(n, rows, 4) @ normal(n, 4, cols)).to(dtype)
    else:
        n, rows, cols = case["count"], case["rows"], case["cols"]

        def gradient():
            return 1e-3 * normal(rows, cols) + 2e-3 * normal(rows, 4) @ normal(4, cols)

        # parameters and optimiser state lie in one buffer each, of which the matrices are parts
        s["held"] = [torch.stack(v) for v in ([normal(rows, cols) * 0.02 for _ in range(n)], [gradient() * 5.0 for _ in range(n)])]
        s["parameters"], s["moments"] = (list(v.unbind(0)) for v in s["held"])
        s["gradients"] = [gradient() for _ in range(n)]
        s["lr"], s["momentum"], s["update_scale"] = 0.02, 0.95, max(1.0, rows / cols) ** 0.5
    return s


# ---------------------------------------------------------------- one pass
def run(s):
    return _own(s) if own else {"head": _plain_head, "orth": _plain_orth, "muon": _plain_muon}[s["kind"]](s)


def _own(s):
    from __graft_entry__ import load_package
    df = load_package()
    if s["kind"] == "head":
        if s["backward"]:
            return df.linear_cross_entropy_backward(s["x"], s["weight"], s["targets"], s["lse"], s["grad"], s["scale"])
        return df.linear_cross_entropy(s["x"], s["weight"], s["targets"], s["scale"])
    if s["kind"] == "orth":
        return df.orthogonalize(s["update"], s["steps"], COEFFICIENTS, EPS)
    df.muon_update(s["parameters"], s["moments"], s["gradients"], s["lr"], s["momentum"], s["decay"], nesterov=s["nesterov"], update_scale=s["update_scale"],
                   steps=5, coefficients=COEFFICIENTS, eps=EPS)
    return s["held"]


def _statistics(s):
    """Loss and logsumexp of every row, 0 where there is no target."""
    z = (s["x"].float() @ s["weight"].float().t()) * s["scale"]
    m = z.max(1, keepdim=True).values
    lse = (m + torch.log(torch.exp(z - m).sum(1, keepdim=True))).squeeze(1)
    there = s["targets"] >= 0
    picked = z.gather(1, s["targets"].long().clamp(min=0)[:, None]).squeeze(1)
    return torch.where(there, lse - picked, 0.0), torch.where(there, lse, 0.0)


def _plain_head(s):
    if not s["backward"]:
        return _statistics(s)
    x, w = s["x"].float(), s["weight"].float()
    there = s["targets"] >= 0
    g = torch.exp((x @ w.t()) * s["scale"] - s["lse"][:, None])
    g.scatter_add_(1, s["targets"].long().clamp(min=0)[:, None], torch.full((x.shape[0], 1), -1.0, device="cuda"))
    g = g * torch.where(there, s["grad"] * s["scale"], 0.0)[:, None]
    return (g @ w).to(s["x"].dtype), (g.t() @ x).to(s["weight"].dtype)


def _newton_schulz(u, steps):
    """u [count, rows, cols] in its own precision."""
    a, b, c = COEFFICIENTS
    x = u / (torch.sqrt((u * u).sum((1, 2), keepdim=True)) + EPS)
    tall = x.shape[1] > x.shape[2]
    if tall:
        x = x.transpose(1, 2)
    for _ in range(steps):
        gram = x @ x.transpose(1, 2)
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.transpose(1, 2) if tall else x


def _plain_orth(s):
    return _newton_schulz(s["update"].float(), s["steps"]).to(s["update"].dtype).contiguous()


def _plain_muon(s):
    g = torch.stack(s["gradients"])
    p, m = s["held"]
    m.mul_(s["momentum"]).add_(g)
    o = _newton_schulz(g + s["momentum"] * m if s["nesterov"] else m, 5)
    p.mul_(1.0 - s["lr"] * s["decay"]).sub_((s["lr"] * s["update_scale"]) * o)
    return s["held"]


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    elt = 2 if case.get("dtype") == "bf16" else 4
    if case["kind"] == "head":
        rows, vocab, width = case["rows"], case["vocab"], case["width"]
        once = (rows + vocab) * width * elt
        if case["backward"]:  # the logits once more, and two products with their gradient
            return {"bytes": 2 * once + 12 * rows, "flops": 6 * rows * vocab * width}
        return {"bytes": once + 12 * rows, "flops": 2 * rows * vocab * width}
    n, rows, cols = case["count"], case["rows"], case["cols"]
    small, large = min(rows, cols), max(rows, cols)
    # two products are symmetric: half of each is enough
    flops = n * case.get("steps", 5) * (small * small * large + small ** 3 + 2 * small * small * large)
    return {"bytes": n * rows * cols * (2 * elt if case["kind"] == "orth" else 20), "flops": flops}


# ---------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "head":
        return _exact_head(s)
    if case["kind"] == "orth":
        return torch.stack([_exact_orth(u.double(), s["steps"]) for u in s["update"]])
    parameters, moments = [], []
    for p, m, g in zip(s["parameters"], s["moments"], s["gradients"]):
        m = s["momentum"] * m.double() + g.double()
        u = g.double() + s["momentum"] * m if s["nesterov"] else m
        parameters.append((1.0 - s["lr"] * s["decay"]) * p.double() - s["lr"] * s["update_scale"] * _exact_orth(u, 5))
        moments.append(m)
    return [torch.stack(parameters), torch.stack(moments)]


def _exact_orth(u, steps):
    """By the eigenvectors of the smaller Gram matrix: each singular value goes through the polynomial by itself."""
    a, b, c = COEFFICIENTS
    wide = u if u.shape[0] <= u.shape[1] else u.t()
    wide = wide / (torch.linalg.matrix_norm(wide) + EPS)
    squares, vectors = torch.linalg.eigh(wide @ wide.t())
    squares = squares.clamp(min=0.0)
    factor = torch.ones_like(squares)  # how much the singular value has been multiplied so far
    for _ in range(steps):
        now = squares * factor * factor
        factor = factor * (a + b * now + c * now * now)
    out = vectors @ (factor[:, None] * (vectors.t() @ wide))
    return out if u.shape[0] <= u.shape[1] else out.t()


def _exact_head(s):
    """Some rows at a time, only those that have a target."""
    x, w, scale = s["x"].double(), s["weight"].double(), s["scale"]
    rows = x.shape[0]
    loss, lse = (torch.zeros(rows, dtype=torch.float64, device="cuda") for _ in range(2))
    d_x, d_w = torch.zeros_like(x), torch.zeros_like(w)
    there = torch.nonzero(s["targets"] >= 0).squeeze(1)
    for r in there.split(max(1, 60_000_000 // w.shape[0])):
        logp = torch.einsum("rk,vk->rv", x[r], w) * scale
        at = s["targets"][r].long()
        of = torch.arange(len(r), device="cuda")
        picked = logp[of, at]
        if not s["backward"]:
            lse[r] = torch.logsumexp(logp, 1)
            loss[r] = lse[r] - picked
            continue
        p = torch.softmax(logp, 1)
        p[of, at] -= 1.0
        p *= (s["grad"][r].double() * scale)[:, None]
        d_x[r] = torch.einsum("rv,vk->rk", p, w)
        d_w += torch.einsum("rv,rk->vk", p, x[r])
    return (d_x, d_w) if s["backward"] else (loss, lse)
