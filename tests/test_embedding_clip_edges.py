"""Edges of the table lookup, its gradient and of gradient clipping that show without a GPU."""
import ctypes

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


P = 1 << 20      # an address that no call below may touch: all are refused


def test_memory_written_twice_is_refused():
    """Before any launch, wherever in the tensors the overlap lies and whatever the order of the list."""
    from sparc_amd._lib import SparcOverlapError, check, lib
    records = lambda *rows: (ctypes.c_int64 * sum(map(len, rows)))(*(x for row in rows for x in row))  # noqa: E731
    clip = lambda *rows: lib.sparc_clip_grad_norm(len(rows), records(*rows), 1.0, P, 1 << 20, P, None)  # noqa: E731
    assert clip((P, 9, 0), (P + 4 * 5, 9, 0)) == -5                       # float32: bytes [0, 36) and [20, 56)
    assert clip((P + 4 * 5, 9, 0), (P, 9, 0)) == -5
    assert clip((P, 9, 0), (P, 9, 0)) == -5
    assert clip((P, 1000, 1), (P + 10_000, 7, 0), (P + 1998, 1, 2)) == -5  # the last two bytes of 1000 bfloat16
    assert clip((P, 100_000, 0), (P + 8, 1, 0), (P + 500_000, 3, 0)) == -5  # wholly inside
    assert clip(*((P + 4096 * i, 1024, 0) for i in range(300)), (P + 4096 * 300 - 4, 2, 0)) == -5
    adam = lambda *rows: lib.sparc_adam_step(len(rows), records(*rows), 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, None)  # noqa: E731
    clipped = lambda *rows: lib.sparc_adam_step_clipped(len(rows), records(*rows), 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, P, 1, 1.0, P, None)  # noqa: E731
    both = lambda *rows: lib.sparc_clip_adam_step(len(rows), records(*rows), 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, 1.0, P, 1 << 20, P, None)  # noqa: E731
    at = lambda i: P + 4096 * i  # noqa: E731
    every = lambda *rows: lib.sparc_adam_check(len(rows), records(*rows))  # noqa: E731
    assert every((at(0), at(1), at(2), at(3), 1024), (at(4), at(1), at(5), at(6), 1024), (0, 0, 0, 0, 0)) == 0    # a shared gradient
    assert every(*((at(4 * i), at(4 * i + 1), at(4 * i + 2), at(4 * i + 3), 1024) for i in range(200)), (at(799), at(900), at(901), at(902), 5)) == -5
    assert every((at(0), 0, at(2), at(3), 1)) == -1 and every((at(0), at(1), at(2), at(3), -1)) == -1
    for step in (adam, clipped, both, every):
        for bad in (((at(0), at(1), at(2), at(2) + 396, 100),),                       # moments that share an element
                    ((at(0), at(1), at(2), at(3), 100), (at(0) + 4, at(5), at(6), at(7), 100)),   # parameters
                    ((at(0), at(0) + 396, at(2), at(3), 100),),                       # a gradient's first element is a parameter's last
                    ((at(0), at(1), at(2), at(3), 100), (at(4), at(3) + 200, at(6), at(7), 100)),  # a gradient inside another's moment
                    ((at(0), at(1), at(2), at(3), 100), (at(4), at(1), at(6), at(1) + 8, 10))):    # a moment inside a shared gradient
            assert step(*bad) == -5, bad
    with pytest.raises(ValueError):
        check(-5, "a step")
    assert issubclass(SparcOverlapError, RuntimeError)


def test_a_model_pickled_before_there_was_a_node_table():
    import pickle
    from sparc_amd.SpectralTrainer import SpectralNetModel
    arch = {"n_layers": 2, "hidden_dim1": 16, "output_dim": 4}
    old = SpectralNetModel(arch, 12, torch.device("cpu"))
    del old.__dict__["node_table"]
    assert pickle.loads(pickle.dumps(old)).node_table is None
    new = pickle.loads(pickle.dumps(SpectralNetModel(arch, 12, torch.device("cpu"), node_table={"rows": 9, "dim": 6})))
    assert new.node_table.weight.shape == (9, 6) and "node_table.weight" in new.state_dict()
