"""Steps that do not fit the server's cache or model are refused on the host, before any call of the library (the stand-in for it here has none)."""
import importlib
from types import SimpleNamespace

import pytest

from helpers import pkg


@pytest.fixture(scope="module")
def server():
    import torch
    pkg()
    serve = importlib.import_module("dark_forest_b200.gpt2_serve")
    model = SimpleNamespace(tok=torch.nn.Embedding(50, 32), pos=torch.nn.Embedding(40, 32), blocks=[None])
    return serve.Server(SimpleNamespace(CACHE_WORKSPACE_BYTES=64), model, 2, slots=3, max_len=64, n_pages=5, page_size=16)


@pytest.mark.parametrize("new,finished", [([[], [], []], None), ([[], [], []], [1, 0, 0]), ([[1], []], None), ([[1], [], []], [0, 0]), ([[50], [], []], None), ([[1, -1], [], []], None),
                                          ([[1] * 41, [], []], None), ([[1] * 33, [1] * 33, []], None)])
def test_steps_that_do_not_fit(server, new, finished):
    before = (server.lens.tolist(), list(server.held), int(server.count))
    with pytest.raises(ValueError):
        server.step(new, finished)
    assert before == (server.lens.tolist(), server.held, int(server.count))


def test_what_slots_hold_counts(server):
    server.held = [40, 30, 0]
    try:
        assert server._lengths_after([[], [1, 2], []], None) == [40, 32, 0]
        for new, finished in (([[1], [], []], None), ([[], [1, 2, 3], []], None), ([[], [], [1]], None), ([[], [1] * 11, []], None), ([[7] * 40, [], [1]], [1, 0, 0])):
            with pytest.raises(ValueError):
                server._lengths_after(new, finished)
        assert server._lengths_after([[1], [], []], [1, 0, 0]) == [1, 30, 0]
    finally:
        server.held = [0, 0, 0]


def test_answers_have_a_token(server):
    for max_new in (0, -1):
        with pytest.raises(ValueError):
            server.generate([[1, 2]], max_new)
