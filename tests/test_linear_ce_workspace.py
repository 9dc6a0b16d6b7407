"""Memory of the loss from hidden states and its gradient, on the host: how much they ask for, and what may not lie in what."""
import pytest

from helpers import pkg
from test_linear_ce_abi import at, grad, lib  # noqa: F401


@pytest.mark.parametrize("rows,vocab,width,bf16", [(4096, 200000, 512, 0), (64, 130000, 1024, 0), (1, 10000, 800, 1), (8, 10000, 768, 1), (8, 50257, 768, 1), (1, 1, 1, 0), (16, 50257, 768, 0),
                                                   (2048, 50257, 768, 0), (8192, 50257, 768, 1)])
def test_the_size_for_the_gradient_is_enough_for_both(rows, vocab, width, bf16):
    """A program asks once and passes the same buffer to both calls."""
    size = pkg().lib().df_linear_cross_entropy_workspace_bytes
    assert size(rows, vocab, width, bf16, 1) >= size(rows, vocab, width, bf16, 0) > 0


def test_a_gradient_of_no_rows_in_the_weight_is_refused(lib):  # noqa: F811
    """It would be set to 0."""
    assert grad(lib, rows=0, dw=at(1)) == pkg().DF_ERR_INVALID_ARG and grad(lib, rows=0, dw=at(1, 4 * 60)) == pkg().DF_ERR_INVALID_ARG
