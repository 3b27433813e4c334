"""Edges of the table lookup, its gradient and of gradient clipping that show without a GPU."""
import pytest
import torch


@pytest.mark.parametrize("dim,dtype", [(1, 0), (64, 1), (8192, 0), (8193, 0), (16384, 2), (16385, 1), (1 << 20, 2)])
def test_no_tokens_need_no_scratch(dim, dtype):
    """The gradient of no tokens is the zeros of the table, whatever the rows' width: nothing to sort."""
    from sparc_amd._lib import lib
    assert lib.sparc_embedding_grad_workspace_bytes(0, 9, dim, dtype) == 0
