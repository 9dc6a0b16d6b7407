"""Results that a call allocates while it runs on a stream given by name: neither work that the current stream still has to do nor what it does next may meet them."""
import pytest

from helpers import pkg

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch


def calls(torch):
    p = pkg()
    torch.manual_seed(1)
    x, w = torch.randn(64, 200, device="cuda"), torch.randn(900, 200, device="cuda") * 0.07
    targets = torch.randint(0, 900, (64,), device="cuda", dtype=torch.int32)
    lse = p.linear_cross_entropy(x, w, targets)[1]
    ones = torch.ones_like(lse)  # inputs are there before: a call on another stream does not wait for the current one
    u = torch.randn(2, 160, 240, device="cuda")
    return {"loss": lambda **kw: p.linear_cross_entropy(x, w, targets, **kw), "gradient": lambda **kw: p.linear_cross_entropy_backward(x, w, targets, lse, ones, **kw),
            "orthogonalised": lambda **kw: (p.orthogonalize(u, **kw),)}


@pytest.mark.parametrize("name", ["loss", "gradient", "orthogonalised"])
def test_blocks_that_the_current_stream_still_writes(torch, name):
    """Blocks of the results' sizes are freed while their writes still wait on the current stream; a call on another stream is done before these writes are."""
    call = calls(torch)[name]
    want = [t.clone() for t in call()]
    other = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        held = [torch.empty_like(t) for t in want for _ in range(4)]
        torch.cuda.synchronize()
        torch.cuda._sleep(40_000_000)  # about 20 ms, a bounded wait
        for t in held:
            t.fill_(7.0)
        del held, t
        got = call(stream=other)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        del got
    assert pkg().sync_status() == 0


@pytest.mark.parametrize("name", ["loss", "gradient", "orthogonalised"])
def test_results_that_are_dropped_early(torch, name):
    """Results of a call on another stream, read by the current stream behind a wait for that one, and dropped: the next call there does not write into them before they are read."""
    call = calls(torch)[name]
    want = [t.clone() for t in call()]
    other = torch.cuda.Stream()
    torch.cuda.synchronize()
    copies = []
    for _ in range(3):
        got = call(stream=other)
        torch.cuda.current_stream().wait_stream(other)
        torch.cuda._sleep(40_000_000)
        copies += [(t.clone(), w) for t, w in zip(got, want)]
        del got
        junk = []
        with torch.cuda.stream(other):  # whatever blocks the other stream gets now
            for w in want:
                junk += [torch.empty_like(w).fill_(9.0) for _ in range(2)]
        del junk
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in copies)
