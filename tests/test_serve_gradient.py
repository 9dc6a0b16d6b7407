"""The autograd form of the log probabilities, over a stand-in for the library's calls on the CPU: first derivatives come through, second ones raise."""
import importlib
from types import SimpleNamespace

import pytest

from helpers import pkg


def stand_in():
    import torch

    def forward(logits, targets, scale):
        logs = (logits * scale).log_softmax(1)
        return logs.gather(1, targets.long()[:, None])[:, 0], -(logs.exp() * logs).sum(1), (logits * scale).logsumexp(1), None, None

    def backward(logits, targets, lse, entropy, d_logp, d_entropy, scale):
        logs = logits * scale - lse[:, None]
        one = torch.nn.functional.one_hot(targets.long(), logits.shape[1])
        return scale * (d_logp[:, None] * (one - logs.exp()) - d_entropy[:, None] * logs.exp() * (logs + entropy[:, None]))

    return SimpleNamespace(token_logprobs=forward, token_logprobs_backward=backward)


def test_second_derivatives_raise():
    import torch
    pkg()
    apply = importlib.import_module("dark_forest_b200.gpt2_serve").token_logprobs_function(stand_in()).apply
    torch.manual_seed(1)
    x, w, targets = torch.randn(3, 7, requires_grad=True), torch.randn(3, requires_grad=True), torch.tensor([1, 0, 6], dtype=torch.int32)
    logp, entropy = apply(x, targets, 0.8)
    first, = torch.autograd.grad((w * (logp + entropy)).sum(), x, create_graph=True)
    y = x.detach().clone().requires_grad_()
    logs = (y * 0.8).log_softmax(1)
    want, = torch.autograd.grad((w.detach() * (logs.gather(1, targets.long()[:, None])[:, 0] - (logs.exp() * logs).sum(1))).sum(), y)
    assert torch.allclose(first, want, atol=1e-6)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(first.square().sum(), x)
