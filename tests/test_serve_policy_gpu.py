"""The policy step sees the tokens under the contexts that they were sampled in: its log probabilities are the server's."""
import importlib

import pytest

from helpers import pkg
from test_serve_gpu import HEADS, serve, small_model, tokens_of, torch_cuda  # noqa: F401 (serve, torch_cuda: the fixtures)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("code,step", [("int8", 2.0 ** -7), ("e4m3", 2.0 ** -4)])
def test_log_probabilities_are_those_of_the_served_tokens(torch_cuda, serve, code, step):  # noqa: F811
    """Keys and values are held within half a step of 8 bits: at most 2^-8 of a page's largest element (int8) or 2^-4 of the element itself (e4m3), which
    two layers' attention, a part of the residual stream, passes on to logits of 0.7: 2 * 0.7 * step bounds both sides of that, and the projections'
    TF32 adds the 3.5e-3 of the served steps' test."""
    torch = torch_cuda
    model, opt = small_model()
    prompts = [tokens_of(i, n) for i, n in enumerate((3, 60, 17, 33, 100))]
    server = serve.Server(pkg(), model, HEADS, slots=5, max_len=128, code=code, temperature=0.8, seed=3)
    answers = server.generate(prompts, 12)
    answers[1]["tokens"], answers[1]["logp"] = answers[1]["tokens"][:5], answers[1]["logp"][:5]  # one that ended earlier
    sequences, prompt_lens, lens = serve.sequences_of(prompts, answers, "cuda")
    assert lens.tolist() == [15, 65, 29, 45, 112] and prompt_lens.tolist() == [3, 60, 17, 33, 100]
    _, logp = serve.policy_step(pkg(), model, opt, sequences, prompt_lens, torch.ones(5, device="cuda"), temperature=0.8, lens=lens)
    for i, (p, a) in enumerate(zip(prompts, answers)):
        n = len(a["tokens"])
        got = logp[i, len(p) - 1:len(p) - 1 + n]
        assert (got - torch.tensor(a["logp"], device="cuda")).abs().max() < 2 * 0.7 * step / 0.8 + 3.5e-3
        assert (logp[i, :len(p) - 1] == 0).all() and (logp[i, len(p) - 1 + n:] == 0).all()


def test_padding_has_no_part_in_the_step(torch_cuda, serve):  # noqa: F811
    """The same step with other tokens behind the sequences' ends: the same loss and the same weights afterwards, bit for bit."""
    torch = torch_cuda
    kept = []
    for filler in (0, 77):
        model, opt = small_model()
        sequences = torch.full((2, 40), filler, device="cuda")
        sequences[0, :30] = torch.tensor(tokens_of(1, 30), device="cuda")
        sequences[1, :40] = torch.tensor(tokens_of(2, 40), device="cuda")
        loss, logp = serve.policy_step(pkg(), model, opt, sequences, torch.tensor([10, 25], device="cuda"), torch.tensor([1.0, -0.5], device="cuda"), bonus=0.01,
                                       lens=torch.tensor([30, 40], device="cuda"))
        kept.append((loss, logp, model.blocks[0].wq.weight.detach().clone(), model.blocks[1].wo.weight.detach().clone()))
    assert torch.equal(kept[0][0], kept[1][0]) and torch.equal(kept[0][1], kept[1][1])
    for a, b in zip(kept[0][2:], kept[1][2:]):
        assert torch.allclose(a, b, rtol=0, atol=1e-6)
    assert (kept[0][1][0, 29:] == 0).all()
