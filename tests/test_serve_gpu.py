"""The operators together, as a server uses them: gpt2_serve.Server against a plain 32-bit forward over what its caches hold, its pages, and the policy step.

Tolerance of the log probabilities: the projections run in TF32 (2^-11 a product), six a layer; over two layers some 5e-3 of a hidden value, and logits
are about 0.7 here: 3.5e-3. 1e-2 is asked for."""
import importlib

import pytest

from helpers import pkg

pytestmark = pytest.mark.gpu

D, HEADS, VOCAB = 128, 2, 500


@pytest.fixture(scope="module")
def torch_cuda():
    import torch
    assert torch.cuda.is_available(), "these tests need a GPU"
    torch.cuda.set_device(0)
    pkg().lib()
    yield torch
    assert pkg().sync_status() == 0


@pytest.fixture(scope="module")
def serve(torch_cuda):
    pkg()
    return importlib.import_module("dark_forest_b200.gpt2_serve")


def small_model():
    pkg()
    step = importlib.import_module("dark_forest_b200.gpt2_step")
    return step.build(pkg(), n_layers=2, d_model=D, n_heads=HEADS, d_ff=512, vocab=VOCAB, max_pos=256, seed=7)[:2]


def tokens_of(seed, n):
    return [(seed * 7919 + i * i * 31 + i) % VOCAB for i in range(n)]


def plain_logits(torch, server, slot, new):
    """Logits behind each of the slot's newest tokens, in fp32, keys and values as the caches hold them."""
    import torch.nn.functional as F
    m, length = server.model, int(server.lens[slot])
    first = length - len(new)
    x = m.tok(torch.tensor(new, device="cuda")) + m.pos(torch.arange(first, length, device="cuda"))
    pages = server.table[slot, :-(-length // server.page_size)].long()
    d = D // HEADS
    for block, (k_cache, v_cache, k_scale, v_scale) in zip(m.blocks, server.caches):
        h = F.layer_norm(x, (D,), block.ln1.weight, block.ln1.bias)
        q = (h @ block.wq.weight.t() + block.wq.bias).view(-1, HEADS, d)

        def held(cache, scale):  # [tokens, heads, d]
            codes = cache.view(torch.uint8)[pages].view(cache.dtype).float() * scale[pages][:, :, None, None]
            return codes.permute(0, 2, 1, 3).reshape(-1, HEADS, d)[:length]
        k, v = held(k_cache, k_scale), held(v_cache, v_scale)
        s = torch.einsum("qhd,thd->hqt", q, k) / d ** 0.5
        seen = torch.arange(length, device="cuda")[None] <= torch.arange(first, length, device="cuda")[:, None]
        a = torch.einsum("hqt,thd->qhd", s.masked_fill(~seen, float("-inf")).softmax(-1), v).reshape(-1, D)
        x = x + a @ block.wo.weight.t() + block.wo.bias
        h = F.layer_norm(x, (D,), block.ln2.weight, block.ln2.bias)
        x = x + F.gelu(h @ block.w1.weight.t() + block.w1.bias, approximate="tanh") @ block.w2.weight.t() + block.w2.bias
    return F.layer_norm(x, (D,), m.ln_f.weight, m.ln_f.bias) @ m.tok.weight.t()


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_steps_agree_with_a_plain_forward(torch_cuda, serve, code):
    torch = torch_cuda
    model, _ = small_model()
    server = serve.Server(pkg(), model, HEADS, slots=3, max_len=256, page_size=16, code=code, temperature=0.8, top_k=3)
    steps = [[tokens_of(1, 37), [], tokens_of(3, 100)], [tokens_of(4, 1), tokens_of(5, 16), tokens_of(6, 1)], [tokens_of(7, 20), tokens_of(8, 1), []]]
    allow = torch.backends.cuda.matmul.allow_tf32
    for new in steps:
        chosen, logp, entropy, top_ids, top_logp = server.step(new)
        torch.backends.cuda.matmul.allow_tf32 = False
        with torch.no_grad():
            for slot, tokens in enumerate(new):
                if not tokens:
                    continue
                z = torch.log_softmax(plain_logits(torch, server, slot, tokens)[-1] / 0.8, 0)
                assert abs(float(z[int(chosen[slot])] - logp[slot])) < 1e-2
                assert abs(float(-(z.exp() * z).sum() - entropy[slot])) < 1e-2
                assert float((z[top_ids[slot].long()] - top_logp[slot]).abs().max()) < 1e-2
                assert float(top_logp[slot, 0]) >= float(z.max()) - 1e-2
        torch.backends.cuda.matmul.allow_tf32 = allow


def test_requests_come_and_go(torch_cuda, serve):
    torch = torch_cuda
    prompts = [tokens_of(i, n) for i, n in enumerate((1, 60, 16, 33, 100, 7, 15))]
    runs = []
    for _ in range(2):
        server = serve.Server(pkg(), small_model()[0], HEADS, slots=3, max_len=128, n_pages=15, piece=24, seed=5)
        runs.append(server.generate(prompts, 6))
        assert sorted(server.free.tolist()) == list(range(15)) and int(server.count) == 15  # every page is back
        assert server.lens.tolist() == [0, 0, 0]
    assert runs[0] == runs[1]
    for answer in runs[0]:
        assert len(answer["tokens"]) == 6 and all(0 <= t < VOCAB for t in answer["tokens"])
        for t, lp, (ids, logps) in zip(answer["tokens"], answer["logp"], answer["alternatives"]):
            assert lp <= logps[0] and logps == sorted(logps, reverse=True)
            assert t not in ids or lp == logps[ids.index(t)]
    with pytest.raises(ValueError):
        server.generate([tokens_of(1, 123)], 6)
    with pytest.raises(ValueError):
        server.generate([[]], 6)
    assert torch.isfinite(server.caches[0][2]).all()


def test_policy_steps_raise_what_is_rewarded(torch_cuda, serve):
    torch = torch_cuda
    model, opt = small_model()
    sequences = torch.tensor([tokens_of(1, 40), tokens_of(2, 40)], device="cuda")
    prompt_lens = torch.tensor([10, 25], device="cuda")
    first = last = None
    for _ in range(8):
        _, logp = serve.policy_step(pkg(), model, opt, sequences, prompt_lens, torch.tensor([1.0, -1.0], device="cuda"), bonus=0.01)
        assert (logp[0, :9] == 0).all() and (logp[0, 9:] < 0).all() and (logp[1, :24] == 0).all()
        last = (float(logp[0, 9:].mean()), float(logp[1, 24:].mean()))
        first = first or last
    assert last[0] > first[0] + 0.05 and last[1] < first[1] - 0.05
