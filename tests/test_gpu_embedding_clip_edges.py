"""Calls of the table lookup, its gradient, clipping and the Adam step at their edges: no tokens, sizes on both sides of a
rule, frozen tables, forward mode, version counters, memory that tensors share in part, captures beside living graphs.

Tolerances are those of test_gpu_embedding.py and test_gpu_clip.py."""
import pytest
import torch

from test_gpu_embedding import check_grad, gen, make_ids

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,dim,dtype", [(9, 8193, torch.float32), (5, 16385, torch.bfloat16), (3, 1 << 20, torch.float16), (7, 5, torch.float16),
                                            (2708, 64, torch.float32), (70_001, 700, torch.float32), (1, 1, torch.bfloat16)])
def test_gradient_of_no_tokens(rows, dim, dtype):
    """A table of zeros, also as the lookup's backward and inside a capture."""
    from sparc_amd.embedding import embedding_grad, embedding_lookup
    ids, g = torch.zeros(0, dtype=torch.int64, device="cuda"), torch.zeros(0, dim, dtype=dtype, device="cuda")
    torch.full((rows, dim), 3.0, dtype=dtype, device="cuda")              # what a new allocation may hold
    got = embedding_grad(ids, g, rows)
    assert got.shape == (rows, dim) and got.dtype == dtype and not bool((got != 0).any())
    table = torch.ones(rows, dim, dtype=dtype, device="cuda", requires_grad=True)
    embedding_lookup(ids.view(0, 2).int(), table, scale=2.0).sum().backward()
    assert not bool((table.grad != 0).any())
    del got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = embedding_grad(ids, g, rows)
    for _ in range(3):
        got.fill_(5.0)
        graph.replay()
        torch.cuda.synchronize()
        assert not bool((got != 0).any())


def test_every_clipped_gradient_counts_as_written():
    """Also one that requires no gradient itself and that another graph has saved."""
    from sparc_amd.optim import clip_grad_norm_
    p, x = (torch.randn(50, device="cuda", generator=gen(i)).requires_grad_() for i in (3, 4))
    p.grad = torch.randn(50, device="cuda", generator=gen(5))
    loss = (p.grad * x).sum()
    before = p.grad._version
    clip_grad_norm_([p], 0.1)
    assert p.grad._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        loss.backward()
    loss = (p.grad * x).sum()                                             # saved after the clipping: fine
    loss.backward()
    assert torch.equal(x.grad, p.grad)
