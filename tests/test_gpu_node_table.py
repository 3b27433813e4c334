"""The table lookup, its gradient, the global norm and the clipped Adam step together, as the trainers use them: a SpectralNet
whose inputs are tokens (spectral.node_table) and whose gradients are clipped (max_grad_norm).

Tolerances.  Gradients of a whole step: those of the golden step (5e-5 of the largest entry, 5e-4 for the output layer's bias,
a sum that nearly cancels); the table's gradient goes through one more product and sum: twice that.  Trajectories over a few
steps: 1e-5, as for the same trainer without table and clipping."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

ARCH = {"n_layers": 4, "hidden_dim1": 64, "hidden_dim2": 64, "hidden_dim3": 32, "output_dim": 6}
ROWS, DIM, SCALE = 90, 5, 2.0


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def rel(a, b):
    a, b = np.asarray(a, dtype=np.float64), np.asarray(b, dtype=np.float64)
    return float(np.abs(a - b).max() / np.abs(b).max())


def problem(seed, m):
    """(support tuple, tokens [m, 2]): a random graph whose nodes carry two categories."""
    import scipy.sparse as sp
    from oracle import sparc_oracle as O
    A = sp.random(m, m, density=0.03, random_state=np.random.RandomState(seed), format="csr")
    A.data[:] = 1.0
    A = sp.triu(A, 1)
    rng = np.random.default_rng(seed)
    return O.as_support_tuple(sp.csr_matrix(A + A.T + sp.eye(m))), torch.tensor(rng.integers(0, ROWS, (m, 2)))


def table_config():
    return {"rows": ROWS, "dim": DIM, "scale": SCALE, "padding_idx": 3}


def test_step_gradients_through_the_table(dev):
    from oracle import sparc_oracle as O
    from sparc_amd.graph import ClusterBatch
    from sparc_amd.SpectralTrainer import SpectralNetLoss, SpectralNetModel
    support, t1 = problem(1, 300)
    _, t2 = problem(2, 200)
    torch.manual_seed(0)
    net = SpectralNetModel(ARCH, 2 * DIM, dev, node_table=table_config()).to(dev)
    batch = ClusterBatch.from_support(support, dev)
    Y = net.forward_pair(t2.to(dev).int(), t1.to(dev).int())
    loss = SpectralNetLoss()(batch, Y, is_normalized=True)
    loss.backward()
    ps = [p.detach().cpu().double().requires_grad_() for p in net.mlp_parameters()]
    table = net.node_table.weight.detach().cpu().double().requires_grad_()
    x1, x2 = ((table[t] * SCALE).flatten(1) for t in (t1, t2))
    Yr = O.mlp_forward(ps, x1) @ O.orthonorm_weights_qr(O.mlp_forward(ps, x2))
    ref = O.spectral_loss(O.valid_affinity(O.support_to_dense(support, torch.float64)), Yr, is_normalized=True)
    grads = torch.autograd.grad(ref, ps + [table])
    assert rel(loss.item(), ref.item()) < 1e-4 and rel(Y.detach().cpu(), Yr.detach()) < 1e-4
    for i, (p, g) in enumerate(zip(net.mlp_parameters(), grads)):
        assert rel(p.grad.cpu(), g) < (5e-4 if i == len(ps) - 1 else 5e-5), i
    want = grads[-1].clone()
    want[3] = 0.0                                        # the padding row
    assert rel(net.node_table.weight.grad.cpu(), want) < 1e-4 and bool((net.node_table.weight.grad[3] == 0).all())


def sharded(dev, seed=5, **kw):
    from sparc_amd.graph import ClusterBatch
    from sparc_amd.parallel import ShardedSpectralTrainer
    tr = ShardedSpectralTrainer(ARCH, 2 * DIM, dev, lr=1e-2, seed=seed, node_table=table_config(), **kw)
    for b in range(2):
        support, tokens = problem(10 + b, 260 + 30 * b)
        tr.add_batch(tokens, ClusterBatch.from_support(support, dev).warm(ARCH["output_dim"]))
    return tr


def run(tr, steps=6):
    rng = np.random.RandomState(0)
    losses = [float(tr.step(s % 2, (s // 2) % 2, rng.permutation(tr.batches[(s // 2) % 2].m)[:ARCH["output_dim"]])) for s in range(steps)]
    return np.array(losses), torch.cat([p.detach().flatten() for p in tr.params]).cpu().numpy()


def test_eager_and_graphed_steps_agree_and_clipping_bites(dev):
    free = run(sharded(dev))
    clipped_tr = sharded(dev, max_grad_norm=0.05)
    clipped = run(clipped_tr)
    assert float(clipped_tr.optimizer.grad_norm) > 0.05          # (the norm before clipping)
    assert rel(free[1], clipped[1]) > 1e-3
    other = sharded(dev, max_grad_norm=0.05, fused_adam=False)   # torch's Adam on gradients that clip_grad_norm_ left
    got = run(other)
    grads = torch.cat([p.grad.flatten() for p in other.params])
    assert float(grads.norm()) <= 0.05 * (1 + 1e-5)
    assert rel(got[0], clipped[0]) < 1e-5 and rel(got[1], clipped[1]) < 1e-5
    graphed = run(sharded(dev, max_grad_norm=0.05, hip_graph=True))
    assert rel(graphed[0], clipped[0]) < 1e-5 and rel(graphed[1], clipped[1]) < 1e-5
    same = sharded(dev, max_grad_norm=0.05)
    same.optimizer = torch.optim.Adam(same.net.parameters(), lr=torch.tensor(1e-2, device=dev), fused=True, capturable=True)
    same = run(same)                                             # eager steps with the graphs' optimiser: bit for bit
    assert np.array_equal(graphed[0], same[0]) and np.array_equal(graphed[1], same[1])


@pytest.mark.parametrize("hip_graph", [False, True])
def test_trainer_and_predict(dev, tmp_path, monkeypatch, hip_graph):
    from sparc_amd.SpectralNet import SpectralNet
    from sparc_amd.SpectralTrainer import SpectralTrainer
    monkeypatch.chdir(tmp_path)
    data = [problem(20 + b, 240 + 20 * b) for b in range(3)]
    parts = [np.arange(len(t)) for _, t in data]
    cfg = {"dataset": "tokens", "spectral": {
        "architecture": ARCH, "epochs": 2, "lr": 1e-3, "lr_decay": 0.1, "min_lr": 1e-7, "batch_size": 1024, "n_clusters": 6,
        "patience": 10, "hip_graph": hip_graph, "node_table": table_config(), "max_grad_norm": 0.1}}
    torch.manual_seed(1)
    np.random.seed(1)
    tr = SpectralTrainer(cfg, dev)
    train = (parts, [t for _, t in data], [s for s, _ in data], None, None)
    val = (parts[:1], [data[0][1]], [data[0][0]], None, None)
    net = tr.train(train, val)
    assert all(bool(p.isfinite().all()) for p in net.parameters())
    again = tr.load_model(tr._input_dim(data[0][1]))
    assert torch.equal(again.node_table.weight, torch.load(tr.weights_path, weights_only=True)["node_table.weight"].to(dev))
    facade = SpectralNet(6, cfg)
    facade.spec_net = net
    X = torch.cat([t for _, t in data])
    got = facade.predict(X, chunk_rows=100)
    with torch.no_grad():
        x = (net.node_table.weight[X.to(dev)] * SCALE).flatten(1)
        for layer in net.layers:
            x = layer(x)
        want = (x @ net.orthonorm_weights).cpu().numpy()
    assert rel(got, want) < 1e-4
    cfg["should_use_ae"] = True
    with pytest.raises(ValueError):
        SpectralNet(6, cfg).fit(train, val)


def test_autoencoder_clips(dev, tmp_path, monkeypatch):
    from sparc_amd.AETrainer import AE, AETrainer
    monkeypatch.chdir(tmp_path)
    arch = {"hidden_dim1": 64, "hidden_dim2": 32, "hidden_dim3": 16, "output_dim": 4}
    cfg = {"dataset": "ae", "ae": {"lr": 1e-2, "epochs": 2, "lr_decay": 0.1, "patience": 5, "n_samples": 10, "batch_size": 10,
                                   "architecture": arch, "min_lr": 1e-9, "max_grad_norm": 0.02}}
    x = torch.randn(200, 12, generator=torch.Generator().manual_seed(3))
    torch.manual_seed(4)
    net = AETrainer(cfg, dev).train([x], [x])
    torch.manual_seed(4)
    ref = AE(arch, 12).to(dev)
    opt = torch.optim.Adam(ref.parameters(), lr=1e-2, fused=True)
    xd = x.to(dev)
    for _ in range(2):
        opt.zero_grad()
        torch.nn.functional.mse_loss(ref.decoder(ref.encoder(xd)), xd).backward()
        assert float(torch.nn.utils.clip_grad_norm_(ref.parameters(), 0.02)) > 0.02
        opt.step()
    for a, b in zip(net.parameters(), ref.parameters()):
        # two Adam steps move every weight by about lr; a gradient entry near zero may take another sign of its last bits
        assert float((a - b).detach().abs().max()) <= 2 * 2 * 1e-2 * 1e-3 + 1e-5 * float(b.detach().abs().max())


def test_graphed_step_beside_a_living_eager_graph_is_refused(dev):
    tr = sharded(dev, max_grad_norm=0.05, hip_graph=True)
    head = np.arange(ARCH["output_dim"])
    kept = tr.net.forward_pair(tr.features[1], tr.features[0])    # on the default stream, and alive
    with pytest.raises(RuntimeError, match="is alive"):
        tr.step(0, 1, head)
    del kept
    tr.net.orthonorm_weights = None
    losses = [float(tr.step(0, 1, head)) for _ in range(4)]
    assert np.isfinite(losses).all()
