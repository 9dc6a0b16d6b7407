"""The GPT-2 step harness with the loss from hidden states and the optimiser on matrices: the operators together, as a training step uses them."""
import importlib

import pytest

from helpers import pkg

pytestmark = pytest.mark.gpu
SIZES = dict(n_layers=2, d_model=64, n_heads=1, d_ff=256, vocab=1031, max_pos=128)


@pytest.fixture(scope="module")
def torch():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch


@pytest.fixture(scope="module")
def harness():
    pkg()
    return importlib.import_module("dark_forest_b200.gpt2_step")


def tokens(torch, seed=3):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return (torch.randint(0, SIZES["vocab"], (2, 100), device="cuda", generator=gen) for _ in range(2))


def test_loss_and_gradients_are_the_other_heads(torch, harness):
    """The same model with both heads: the head by library products rounds its operands to TF32 (2^-11 each), so losses differ by that of a logit, here below 1 in size,
    and gradients by 2^-10 of what the products sum up, of which a norm is at most a few times the gradient's; every parameter gets one. A shift of all keys moves a
    row's scores alike and its weights not at all: the exact gradient of the keys' biases is 0, what either head gives there is rounding and has no relative error."""
    out = []
    for linear_loss in (False, True):
        model, _, _ = harness.build(pkg(), linear_loss=linear_loss, optimizer=False, **SIZES)
        idx, tgt = tokens(torch)
        loss = model(idx, tgt)
        loss.backward()
        assert pkg().sync_status() == 0
        out.append((float(loss.detach()), {n: p.grad for n, p in model.named_parameters()}))
    assert abs(out[0][0] - out[1][0]) <= 2.0 ** -9
    for name, a in out[0][1].items():
        b = out[1][1][name]
        assert bool(b.isfinite().all())
        if name.endswith("wk.bias"):
            continue
        assert float((a.double() - b.double()).norm()) <= 2.0 ** -6 * float(a.double().norm()) + 1e-9


def test_second_derivative_is_refused(torch, harness):
    model, _, _ = harness.build(pkg(), linear_loss=True, optimizer=False, **SIZES)
    idx, tgt = tokens(torch)
    (g,) = torch.autograd.grad(model(idx, tgt), model.tok.weight, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_steps_together(torch, harness):
    """Three steps: every matrix of the blocks moves by the orthogonalised momentum (recomputed here in 64 bits), every other parameter as AdamW alone moves it."""
    model, opt, _ = harness.build(pkg(), linear_loss=True, optimizer="muon", **SIZES)
    assert sorted(len(g[0]) for g in opt.groups) == [2, 2, 8]
    for step in range(3):
        idx, tgt = tokens(torch, step)
        loss = model(idx, tgt)
        opt.zero_grad(set_to_none=True)
        loss.backward()
        before = [[(p.detach().double(), m.double()) for p, m in zip(*g)] for g in opt.groups]
        table = model.tok.weight.detach().clone()
        opt.step()
        assert pkg().sync_status() == 0
        assert not torch.equal(table, model.tok.weight)
        for (ps, ms), old in zip(opt.groups, before):
            for p, m, (p0, m0) in zip(ps, ms, old):
                want_m = 0.95 * m0 + p.grad.double()
                assert float((m.double() - want_m).norm()) <= 2.0 ** -22 * float(want_m.norm() + m0.norm())
                x = p.grad.double() + 0.95 * m.double()
                x = x / (x.norm() + 1e-7)
                tall = x.shape[0] > x.shape[1]
                x = x.t() if tall else x
                for _ in range(5):
                    g = x @ x.t()
                    x = 3.4445 * x + (-4.775 * g + 2.0315 * g @ g) @ x
                x = x.t() if tall else x
                scale = 0.02 * max(1.0, p.shape[0] / p.shape[1]) ** 0.5
                off = p.detach().double() - (p0 * (1 - 0.02 * 0.1) - scale * x)
                # the bound of tests/test_muon_gpu.py: 37 2^-19 sqrt(side) (1 + a + .. + a^4) / 4, and the parameter's own roundings
                assert float(off.norm()) <= scale * 37 * 2.0 ** -19 * 8 * 200 / 4 + 2.0 ** -22 * float(p0.norm() + scale * x.norm())


def test_runs_from_the_command_path(torch, harness):
    r = harness.run(pkg(), batch=2, seq=96, steps=2, warmup=1, linear_loss=True, optimizer="muon", **SIZES)
    assert r["loss_first_step"] > 0 and r["step_ms"] > 0
