"""How much memory the loss from hidden states and its gradient ask for, on the host."""
import pytest

from helpers import pkg


@pytest.mark.parametrize("rows,vocab,width,bf16", [(4096, 200000, 512, 0), (64, 130000, 1024, 0), (1, 10000, 800, 1), (8, 10000, 768, 1), (8, 50257, 768, 1), (1, 1, 1, 0), (16, 50257, 768, 0),
                                                   (2048, 50257, 768, 0), (8192, 50257, 768, 1)])
def test_the_size_for_the_gradient_is_enough_for_both(rows, vocab, width, bf16):
    """A program asks once and passes the same buffer to both calls."""
    size = pkg().lib().df_linear_cross_entropy_workspace_bytes
    assert size(rows, vocab, width, bf16, 1) >= size(rows, vocab, width, bf16, 0) > 0
