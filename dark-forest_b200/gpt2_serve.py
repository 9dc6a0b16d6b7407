"""Serving a GPT-2 and learning from what it said: the caller side of the paged 8-bit cache and of the log probabilities.

A `Server` holds the model of gpt2_step.build and one cache per layer that share their pages' numbering. A step takes a batch of requests in which some
bring (a piece of) a prompt and the others one token: pages of finished requests go back (cache_release), the new tokens get their pages and slots
(cache_plan, once for all layers), and per layer LayerNorm -> Q, K, V projections -> cache_append -> cache_attention -> output projection with
residual -> LayerNorm -> MLP, all of this library but the MLP's second projection and the tied LM head (stock torch). The tokens that come out carry their log
probability, the entropy and the alternatives (token_logprobs). generate() reads those five results and the plan's state, once per step, and nothing else.

`policy_step` is the training side: the model's ordinary forward over the served sequences, the log probabilities of their tokens with token_logprobs
and its gradient, and an optimizer step on -advantage * log p - bonus * entropy.

    python dark-forest_b200/gpt2_serve.py --requests 12 --slots 8     # random weights of GPT-2 small, random prompts
"""
from __future__ import annotations


class Server:
    """Continuous batching over `slots` requests at a time. `n_pages` pages of `page_size` tokens are all the cache there is; a request is taken
    in when the pages that it can grow to are free, so that cache_plan grants every step. Prompts come in pieces of at most `piece` tokens."""

    def __init__(self, pkg, model, n_heads, slots=8, max_len=1024, n_pages=None, page_size=16, code="int8", piece=256, temperature=1.0, top_k=5, seed=0):
        import torch
        self.pkg, self.model, self.n_heads, self.page_size, self.piece = pkg, model, n_heads, page_size, piece
        self.temperature, self.top_k = temperature, top_k
        weight = model.tok.weight
        self.device, d_model = weight.device, weight.shape[1]
        d_head, width = d_model // n_heads, -(-max_len // page_size)
        self.max_len = min(max_len, model.pos.num_embeddings)
        self.n_pages = n_pages if n_pages is not None else slots * width
        dtype = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}[code]

        def pool():
            return (torch.zeros(self.n_pages, n_heads, page_size, d_head, dtype=torch.int8, device=self.device).view(dtype),
                    torch.zeros(self.n_pages, n_heads, device=self.device))

        self.caches = []
        for _ in model.blocks:
            (k, k_scale), (v, v_scale) = pool(), pool()
            self.caches.append((k, v, k_scale, v_scale))
        self.workspace = torch.zeros(pkg.CACHE_WORKSPACE_BYTES, dtype=torch.uint8, device=self.device)
        self.lens = torch.zeros(slots, dtype=torch.int32, device=self.device)
        self.held = [0] * slots  # the same on the host, so that a step that does not fit is refused before anything runs
        self.table = torch.zeros(slots, width, dtype=torch.int32, device=self.device)
        self.free = torch.arange(self.n_pages - 1, -1, -1, dtype=torch.int32, device=self.device)
        self.count = torch.full((1,), self.n_pages, dtype=torch.int32, device=self.device)
        self.random = torch.Generator(device=self.device)
        self.random.manual_seed(seed)

    def _forward(self, tokens, positions, starts, slots):
        """Hidden rows of a step's new tokens."""
        pkg, model = self.pkg, self.model
        x = model.tok(tokens) + model.pos(positions)
        for block, (k_cache, v_cache, k_scale, v_scale) in zip(model.blocks, self.caches):
            h = block.ln1(x)
            q, k, v = pkg.linear_qkv(h, block.wq.weight, block.wk.weight, block.wv.weight, block.wq.bias, block.wk.bias, block.wv.bias)
            pkg.cache_append(k, v, slots, k_cache, v_cache, k_scale, v_scale)
            a, _ = pkg.cache_attention(q, k_cache, v_cache, k_scale, v_scale, self.table, self.lens, starts, self.n_heads,
                                       (x.shape[1] / self.n_heads) ** -0.5, self.workspace)
            x = pkg.linear(a, block.wo.weight, block.wo.bias, residual=x)
            _, up = pkg.linear_gelu(block.ln2(x), block.w1.weight, block.w1.bias, keep_pre_activation=False)
            x = x + block.w2(up)
        return x

    def _lengths_after(self, new, finished):
        """The slots' lengths behind a step; ValueError for one that the cache or the model has no place for (their kernels would index behind it)."""
        if len(new) != len(self.held) or (finished is not None and len(finished) != len(self.held)):
            raise ValueError(f"a step has an entry for each of the {len(self.held)} slots")
        if not any(new):
            raise ValueError("a step needs a token of some slot (release() gives pages back without one)")
        vocab = self.model.tok.num_embeddings
        if any(not 0 <= t < vocab for tokens in new for t in tokens):
            raise ValueError(f"token ids are 0 to {vocab - 1}")
        after = [(0 if finished is not None and finished[s] else n) + len(new[s]) for s, n in enumerate(self.held)]
        if max(after) > self.max_len:
            raise ValueError(f"slot {after.index(max(after))}: {max(after)} tokens, {self.max_len} at most")
        pages = sum(-(-n // self.page_size) for n in after)
        if pages > self.n_pages:
            raise ValueError(f"the step needs {pages} pages, there are {self.n_pages}")
        return after

    def step(self, new, finished=None):
        """One step: `new` is a list, for each slot the tokens that it brings (possibly none, but not all of them); `finished` flags the slots whose request has
        left. Returns (tokens, logp, entropy, top_ids, top_logp), a row per slot, sampled behind the slot's last new token (rows of slots
        without any mean nothing). ValueError, and nothing changed, where the tokens or their pages do not fit."""
        import torch
        pkg, after = self.pkg, self._lengths_after(new, finished)
        with torch.no_grad():
            if finished is not None and any(finished):
                flags = torch.tensor([int(f) for f in finished], dtype=torch.int32, device=self.device)
                self.lens, self.count = pkg.cache_release(self.lens, flags, self.table, self.free, self.count, self.page_size)
            counts = torch.tensor([len(n) for n in new], dtype=torch.int32, device=self.device)
            tokens = torch.tensor([t for n in new for t in n], dtype=torch.int64, device=self.device)
            self.lens, starts, slots, positions, state = pkg.cache_plan(self.lens, counts, self.table, self.free, self.count, self.page_size,
                                                                        tokens.numel())
            self.count, self.held = state[:1], after
            x = self._forward(tokens, positions.long(), starts, slots)
            last = x[(starts[1:].long() - 1).clamp_(min=0)]
            logits = self.model.ln_f(last) @ self.model.tok.weight.t()
            noise = torch.empty_like(logits).exponential_(generator=self.random)
            chosen = torch.argmax(logits / self.temperature - noise.log(), dim=1).to(torch.int32)  # a draw from softmax(logits / temperature)
            logp, entropy, _, top_ids, top_logp = pkg.token_logprobs(logits, chosen, 1.0 / self.temperature, self.top_k)
        self.state = state
        return chosen, logp, entropy, top_ids, top_logp

    def generate(self, prompts, max_new, end=None):
        """Answers to `prompts` (lists of token ids), up to max_new tokens each or until `end`. Returns a dict per prompt: tokens, logp, entropy,
        alternatives (a list of (ids, logp) per token)."""
        slots = self.lens.numel()
        answers = [{"tokens": [], "logp": [], "entropy": [], "alternatives": []} for _ in prompts]
        waiting, owner = list(range(len(prompts))), [None] * slots
        if max_new < 1:
            raise ValueError("max_new is 1 or more")
        todo, pages, finished = [[] for _ in range(slots)], [0] * slots, [False] * slots

        def needs(i):
            return -(-(len(prompts[i]) + max_new) // self.page_size)

        for i in waiting:
            if not prompts[i] or len(prompts[i]) + max_new > self.max_len or needs(i) > self.n_pages:
                raise ValueError(f"prompt {i}: 1 to {self.max_len - max_new} tokens that fit {self.n_pages} pages are asked for")
        while waiting or any(o is not None for o in owner):
            for s in range(slots):
                if owner[s] is None and waiting and sum(pages) + needs(waiting[0]) <= self.n_pages:
                    owner[s] = waiting.pop(0)
                    todo[s], pages[s] = list(prompts[owner[s]]), needs(owner[s])
            new = [todo[s][:self.piece] if owner[s] is not None else [] for s in range(slots)]
            chosen, logp, entropy, top_ids, top_logp = (t.tolist() for t in self.step(new, finished))
            missing = int(self.state[1])
            if missing:
                raise RuntimeError(f"cache_plan granted nothing ({missing})")
            finished = [False] * slots
            for s in range(slots):
                if owner[s] is None:
                    continue
                todo[s] = todo[s][len(new[s]):]
                if todo[s]:
                    continue  # a piece of a prompt: more to come
                answer = answers[owner[s]]
                answer["tokens"].append(chosen[s])
                answer["logp"].append(logp[s])
                answer["entropy"].append(entropy[s])
                answer["alternatives"].append((top_ids[s], top_logp[s]))
                todo[s] = [chosen[s]]
                if len(answer["tokens"]) == max_new or chosen[s] == end:
                    owner[s], pages[s], finished[s], todo[s] = None, 0, True, []
        if any(finished):
            self.release(finished)
        return answers

    def release(self, finished):
        """Gives the pages of the flagged slots back without a step."""
        import torch
        flags = torch.tensor([int(f) for f in finished], dtype=torch.int32, device=self.device)
        self.lens, self.count = self.pkg.cache_release(self.lens, flags, self.table, self.free, self.count, self.page_size)
        self.held = [0 if f else n for f, n in zip(finished, self.held)]


def token_logprobs_function(pkg):
    """token_logprobs as an autograd.Function: apply(logits, targets, scale) -> (logp, entropy). Its gradient has none of its own: a second derivative
    raises instead of being left out."""
    import torch

    class TokenLogprobs(torch.autograd.Function):
        @staticmethod
        def forward(ctx, logits, targets, scale):
            logp, entropy, lse, _, _ = pkg.token_logprobs(logits, targets, scale)
            ctx.save_for_backward(logits, targets, lse, entropy)
            ctx.scale = scale
            return logp, entropy

        @staticmethod
        @torch.autograd.function.once_differentiable
        def backward(ctx, d_logp, d_entropy):
            logits, targets, lse, entropy = ctx.saved_tensors
            return pkg.token_logprobs_backward(logits, targets, lse, entropy, d_logp.contiguous(), d_entropy.contiguous(), ctx.scale), None, None

    return TokenLogprobs


def policy_step(pkg, model, opt, sequences, prompt_lens, advantages, bonus=0.0, temperature=1.0, lens=None):
    """One policy gradient step over sequences [batch, S] (int64 token ids, prompts first), of which the tokens behind prompt_lens [batch] were
    sampled; advantages [batch]. lens [batch]: the sequences' lengths where they differ, what lies behind is padding (no token attends to what comes
    after it, so every log probability is under the context that was served). Returns (loss, logp [batch, S - 1], 0 where a token is the prompt's or padding)."""
    import torch
    batch, S = sequences.shape
    x = model.tok(sequences) + model.pos(torch.arange(S, device=sequences.device))[None]
    for block in model.blocks:
        x = block(x)
    logits = model.ln_f(x)[:, :-1].reshape(batch * (S - 1), -1) @ model.tok.weight.t()
    place = torch.arange(1, S, device=sequences.device)[None]
    sampled = place >= prompt_lens[:, None]
    if lens is not None:
        sampled &= place < lens[:, None]
    targets = torch.where(sampled, sequences[:, 1:], -1).to(torch.int32).reshape(-1)  # -1: no log probability, and no gradient of one
    logp, entropy = token_logprobs_function(pkg).apply(logits, targets, 1.0 / temperature)
    logp, entropy = logp.view(batch, S - 1), entropy.view(batch, S - 1)
    loss = -((advantages[:, None] * logp + bonus * entropy) * sampled).sum() / sampled.sum()
    opt.zero_grad(set_to_none=False)
    loss.backward()
    opt.step()
    return loss.detach(), logp.detach()


def sequences_of(prompts, answers, device):
    """policy_step's sequences (padded behind with 0), prompt_lens and lens of prompts and what generate() answered to them."""
    import torch
    rows = [list(p) + a["tokens"] for p, a in zip(prompts, answers)]
    sequences = torch.zeros(len(rows), max(len(r) for r in rows), dtype=torch.int64)
    for i, row in enumerate(rows):
        sequences[i, :len(row)] = torch.tensor(row)
    return sequences.to(device), torch.tensor([len(p) for p in prompts], device=device), torch.tensor([len(r) for r in rows], device=device)


def main():
    import argparse
    import os
    import random
    import sys
    import time
    ap = argparse.ArgumentParser(description="Serve random prompts with random GPT-2 small weights; one policy step on the answers.")
    ap.add_argument("--requests", type=int, default=12)
    ap.add_argument("--slots", type=int, default=8)
    ap.add_argument("--new", type=int, default=32)
    ap.add_argument("--code", choices=("int8", "e4m3"), default="int8")
    args = ap.parse_args()
    sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    from __graft_entry__ import load_package
    pkg = load_package()
    import importlib

    import torch
    model, opt, _ = importlib.import_module("dark_forest_b200.gpt2_step").build(pkg, max_pos=1024)
    rng = random.Random(0)
    prompts = [[rng.randrange(50257) for _ in range(rng.randint(1, 400))] for _ in range(args.requests)]
    server = Server(pkg, model, 12, slots=args.slots, code=args.code)
    server.generate(prompts[:1], 2)  # first launches
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    answers = server.generate(prompts, args.new)
    seconds = time.perf_counter() - t0
    n = sum(len(a["tokens"]) for a in answers)
    print(f"{n} tokens of {args.requests} requests in {seconds * 1e3:.0f} ms, {n / seconds:.0f} a second; "
          f"mean log probability {sum(sum(a['logp']) for a in answers) / n:.3f}, mean entropy {sum(sum(a['entropy']) for a in answers) / n:.3f}")
    sequences, prompt_lens, lens = sequences_of(prompts, answers, "cuda")
    loss, _ = policy_step(pkg, model, opt, sequences, prompt_lens, torch.randn(args.requests, device="cuda"), bonus=0.01, lens=lens)
    print(f"policy step: loss {float(loss):.4f}")


if __name__ == "__main__":
    main()
