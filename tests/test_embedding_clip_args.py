"""What the entry points of the table lookup and of gradient clipping refuse, before any launch (no GPU needed)."""
import ctypes

import pytest
import torch

P = 4096      # any address: no call below may touch it


def test_embedding_arguments():
    from sparc_amd._lib import lib
    fwd = lambda n=4, rows=5, dim=8, dtype=0, ids=P, table=P, ld=8, out=P, ldo=8: lib.sparc_embedding_fwd(  # noqa: E731
        n, rows, dim, dtype, ids, 0, table, ld, 1.0, out, ldo, None)
    for bad in (dict(n=-1), dict(rows=-1), dict(dim=-1), dict(dtype=3), dict(dtype=-1), dict(ids=None), dict(table=None),
                dict(out=None), dict(ld=7), dict(ldo=7)):
        assert fwd(**bad) == -1, bad
    for bad in (dict(n=1 << 31), dict(rows=1 << 31), dict(dim=(1 << 20) + 1, ld=1 << 21, ldo=1 << 21)):
        assert fwd(**bad) == -4, bad
    assert fwd(n=0) == 0 and fwd(dim=0, ld=0, ldo=0) == 0                    # nothing to do, nothing launched
    grad = lambda n=20000, rows=5, dim=8, dtype=0, ids=P, g=P, ldg=8, out=P, ws=P, nbytes=1 << 40: lib.sparc_embedding_grad(  # noqa: E731
        n, rows, dim, dtype, ids, 0, g, ldg, 1.0, -1, out, ws, nbytes, None)
    for bad in (dict(n=-1), dict(rows=-1), dict(dim=-1), dict(dtype=3), dict(ids=None), dict(g=None), dict(out=None),
                dict(ldg=7)):
        assert grad(**bad) == -1, bad
    for bad in (dict(n=1 << 31), dict(rows=1 << 31), dict(dim=(1 << 20) + 1, ldg=1 << 21)):
        assert grad(**bad) == -4, bad
    assert grad(nbytes=16) == -2 and grad(ws=P + 8) == -2 and grad(ws=None) == -2
    assert grad(rows=0) == 0 and grad(dim=0, ldg=0) == 0
    assert lib.sparc_embedding_grad_workspace_bytes(1 << 31, 5, 8, 0) == 0
    assert lib.sparc_embedding_grad_workspace_bytes(4, 5, 8, 7) == 0
    assert lib.sparc_embedding_grad_workspace_bytes(8192, 5, 8, 0) == 0        # one launch, without scratch
    assert lib.sparc_embedding_grad_workspace_bytes(8193, 5, 8, 0) > 0


def test_gradient_workspace_stays_near_its_operands():
    """A few words per token and row, and partial sums: never a multiple of the gradient for sizes that occur."""
    from sparc_amd._lib import lib
    for n, rows, dim, dtype, size in ((20437, 2708, 64, 0, 4), (48979, 2449029, 64, 0, 4), (262147, 50021, 512, 1, 2), (16385, 1, 1, 0, 4),
                                      (2_000_000_000, 1000, 1, 2, 2), (17000, 2_000_000_000, 1, 2, 2)):
        nbytes = lib.sparc_embedding_grad_workspace_bytes(n, rows, dim, dtype)
        assert 0 < nbytes <= 64 * (n + rows) + 4 * (n + rows) * dim * size + (1 << 26), (n, rows, dim)


def test_clip_arguments():
    from sparc_amd._lib import lib
    one = (ctypes.c_int64 * 3)(P, 100, 0)
    count = ctypes.c_int64(-5)
    norm = lambda n=1, t=one, parts=P, nbytes=1 << 20, c=ctypes.byref(count): lib.sparc_grad_norm(n, t, parts, nbytes, c, None)  # noqa: E731
    assert norm(n=-1) == -1 and norm(t=None) == -1 and norm(parts=None) == -1 and norm(c=None) == -1
    assert norm(nbytes=8) == -2 and norm(parts=P + 4) == -2
    for bad in ((P, -1, 0), (0, 1, 0), (P, 1, 3), (P, 1, -1), (P, (1 << 34) + 1, 0)):
        assert norm(t=(ctypes.c_int64 * 3)(*bad)) == -1, bad
    assert norm(n=0, t=None) == 0 and count.value == 0                       # an empty list has no partial sums
    clip = lambda n=1, t=one, limit=1.0, parts=P, nbytes=1 << 20, out=P: lib.sparc_clip_grad_norm(n, t, limit, parts, nbytes, out, None)  # noqa: E731
    for bad in (dict(n=-1), dict(t=None), dict(parts=None), dict(limit=-1.0), dict(limit=float("nan")), dict(out=None)):
        assert clip(**bad) == -1, bad
    assert clip(nbytes=8) == -2
    rec = (ctypes.c_int64 * 5)(P, P, P, P, 100)
    adam = lambda n=1, t=rec, b1=0.9, b2=0.999, eps=1e-8, step=1, parts=P, k=1, limit=1.0, out=P: lib.sparc_adam_step_clipped(  # noqa: E731
        n, t, 1e-3, b1, b2, eps, 0.0, step, parts, k, limit, out, None)
    for bad in (dict(n=-1), dict(t=None), dict(b1=1.0), dict(b2=-0.1), dict(eps=-1.0), dict(step=0), dict(parts=None), dict(k=2000),
                dict(limit=-2.0), dict(out=None), dict(t=(ctypes.c_int64 * 5)(P, 0, P, P, 4)), dict(t=(ctypes.c_int64 * 5)(P, P, P, P, -4))):
        assert adam(**bad) == -1, bad


def test_host_tensors_are_refused():
    from sparc_amd._lib import SparcHipError
    from sparc_amd.embedding import embedding_grad, embedding_lookup
    from sparc_amd.optim import adam_step_, clip_grad_norm_
    t, ids = torch.zeros(4, 3), torch.zeros(2, dtype=torch.int64)
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.ones(3)
    for call in (lambda: embedding_lookup(ids, t), lambda: embedding_grad(ids, t[:2], 4), lambda: clip_grad_norm_([p], 1.0),
                 lambda: adam_step_([t], [t], [t], [t], 1)):
        with pytest.raises(SparcHipError):
            call()


def test_trainer_configuration():
    from sparc_amd.SpectralTrainer import SpectralNetModel, SpectralTrainer
    arch = {"n_layers": 2, "hidden_dim1": 16, "output_dim": 4}
    net = SpectralNetModel(arch, 12, torch.device("cpu"), node_table={"rows": 9, "dim": 6, "scale": 2.0, "padding_idx": 1})
    assert set(net.state_dict()) == {"node_table.weight", "layers.0.0.weight", "layers.0.0.bias", "layers.1.0.weight", "layers.1.0.bias"}
    assert [id(p) for p in net.mlp_parameters()] == [id(p) for layer in net.layers for p in (layer[0].weight, layer[0].bias)]
    assert bool((net.node_table.weight[1] == 0).all())
    with pytest.raises(ValueError):
        SpectralNetModel(arch, 13, torch.device("cpu"), node_table={"rows": 9, "dim": 6})
    spectral = {"lr": 1e-3, "epochs": 1, "lr_decay": 0.5, "patience": 1, "batch_size": 1, "n_clusters": 1, "architecture": arch,
                "node_table": {"rows": 9, "dim": 6}, "max_grad_norm": 1.0, "min_lr": 0.0}
    tr = SpectralTrainer({"spectral": spectral, "dataset": "d"}, torch.device("cpu"))
    assert tr._input_dim(torch.zeros(5, 2, dtype=torch.int64)) == 12 and tr._input_dim(torch.zeros(5, dtype=torch.int32)) == 6
    with pytest.raises(ValueError):
        tr._to_device(torch.zeros(5, 2))
    tr._setup_model(12)
    with pytest.raises(ValueError):
        tr._setup_optimizer(False)


def test_clipping_step_arguments():
    from sparc_amd._lib import lib
    rec = (ctypes.c_int64 * 5)(P, P, P, P, 100)
    step = lambda n=1, t=rec, b1=0.9, b2=0.999, eps=1e-8, step=1, limit=1.0, parts=P, nbytes=1 << 20, out=P: lib.sparc_clip_adam_step(  # noqa: E731
        n, t, 1e-3, b1, b2, eps, 0.0, step, limit, parts, nbytes, out, None)
    for bad in (dict(n=-1), dict(t=None), dict(b1=1.0), dict(b2=-0.1), dict(eps=-1.0), dict(step=0), dict(parts=None), dict(limit=-2.0),
                dict(limit=float("nan")), dict(out=None), dict(t=(ctypes.c_int64 * 5)(P, 0, P, P, 4)),
                dict(t=(ctypes.c_int64 * 5)(P, P, P, P, -4)), dict(t=(ctypes.c_int64 * 5)(P, P, P, P, (1 << 34) + 1))):
        assert step(**bad) == -1, bad
    assert step(nbytes=8) == -2 and step(parts=P + 4) == -2
