"""Edges of the table lookup, its gradient and of gradient clipping that show without a GPU."""
import pytest
import torch


@pytest.mark.parametrize("dim,dtype", [(1, 0), (64, 1), (8192, 0), (8193, 0), (16384, 2), (16385, 1), (1 << 20, 2)])
def test_no_tokens_need_no_scratch(dim, dtype):
    """The gradient of no tokens is the zeros of the table, whatever the rows' width: nothing to sort."""
    from sparc_amd._lib import lib
    assert lib.sparc_embedding_grad_workspace_bytes(0, 9, dim, dtype) == 0


def test_every_clipped_gradient_counts_as_written(monkeypatch):
    """clip_grad_norm_ raises the version of all gradients that it scales (the launch itself is left out here)."""
    from sparc_amd import optim
    monkeypatch.setattr(optim, "require_gpu", lambda device: None)
    monkeypatch.setattr(optim, "launch", lambda *a: None)
    monkeypatch.setattr(optim, "_dense_on", lambda *a: True)
    p, q = torch.nn.Parameter(torch.zeros(3)), torch.nn.Parameter(torch.zeros(2))
    p.grad, q.grad = torch.ones(3), torch.ones(2)
    x = torch.ones(3, requires_grad=True)
    loss = (p.grad * x).sum()
    optim.clip_grad_norm_([p, q], 1.0)
    assert p.grad._version > 0 and q.grad._version > 0
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        loss.backward()


def test_a_refused_adam_step_counts_for_no_group():
    from sparc_amd.optim import Adam
    ps = [torch.nn.Parameter(torch.zeros(3)) for _ in range(2)]
    opt = Adam([{"params": ps[:1]}, {"params": ps[1:]}])
    for p in ps:
        p.grad = torch.ones(3)
    with pytest.raises(RuntimeError):
        opt.step()                                                        # (host tensors)
    assert [group.get("step", 0) for group in opt.param_groups] == [0, 0]


def test_forward_mode_is_refused():
    """A tangent that the kernels would lose in silence: refused before the device is looked at, also by a frozen table."""
    from torch.autograd import forward_ad
    from sparc_amd.embedding import embedding_grad, embedding_lookup
    from sparc_amd.optim import adam_step_, clip_grad_norm_
    ids, t = torch.zeros(2, dtype=torch.int64), torch.randn(5, 3)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(t, torch.ones_like(t))
        p = torch.nn.Parameter(torch.zeros(5, 3))
        p.grad = d
        for call in (lambda: embedding_lookup(ids, d), lambda: embedding_grad(ids, d[:2], 5), lambda: clip_grad_norm_([p], 1.0)):
            with pytest.raises(NotImplementedError):
                call()
            with torch.no_grad(), pytest.raises(NotImplementedError):
                call()
        q = forward_ad.make_dual(t.clone().requires_grad_(), torch.ones_like(t))
        with pytest.raises(NotImplementedError):
            embedding_lookup(ids, q)


def test_gradient_of_a_gradient_is_refused():
    from sparc_amd.embedding import embedding_grad
    ids, g = torch.zeros(2, dtype=torch.int64), torch.randn(2, 3, requires_grad=True)
    with pytest.raises(RuntimeError, match="not differentiable"):
        embedding_grad(ids, g, 5)
