"""Calls of the table lookup, its gradient, clipping and the Adam step at their edges: no tokens, sizes on both sides of a
rule, frozen tables, forward mode, version counters, memory that tensors share in part, captures beside living graphs.

Tolerances are those of test_gpu_embedding.py and test_gpu_clip.py."""
import numpy as np
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


@pytest.mark.parametrize("groups", [1, 2])
@pytest.mark.parametrize("limit", [None, 1.0])
def test_adam_class_counts_as_written(limit, groups):
    """Parameters and moments: a graph that saved them refuses to go back, as with torch's Adam."""
    from sparc_amd.optim import Adam
    ps = [torch.nn.Parameter(torch.randn(50, device="cuda", generator=gen(3 + i))) for i in range(2)]
    opt = Adam([{"params": ps}] if groups == 1 else [{"params": [p]} for p in ps], max_grad_norm=limit)
    x = torch.ones(50, device="cuda", requires_grad=True)
    for turn in range(2):
        for p in ps:
            p.grad = torch.ones(50, device="cuda")
            saved = [(p * p).sum()] + [(x * m).sum() for m in opt.state[p].values()]
            opt.step()
            for loss in saved:
                with pytest.raises(RuntimeError, match="modified by an inplace"):
                    loss.backward()
    loss = (ps[0] * ps[0]).sum()                                          # made after the step: fine
    ps[0].grad = None
    loss.backward()
    assert torch.equal(ps[0].grad, 2 * ps[0].detach())


def test_adam_function_counts_moments_as_written():
    from sparc_amd.optim import adam_step_
    p, g, m, v = (torch.rand(50, device="cuda", generator=gen(i)) for i in range(4))
    x = torch.ones(50, device="cuda", requires_grad=True)
    for limit in (None, 1.0):
        saved = [(x * t).sum() for t in (p, m, v)]
        read = (x * g).sum()
        adam_step_([p], [g], [m], [v], 1, max_grad_norm=limit)
        for loss in saved:
            with pytest.raises(RuntimeError, match="modified by an inplace"):
                loss.backward()
        read.backward()                                                   # the gradient is only read


@pytest.mark.parametrize("limit", [None, 1.0])
def test_a_refused_adam_step_changes_nothing(limit):
    """The second group is refused: neither group moves or counts a step, and the next step is the one it would have been."""
    from sparc_amd.optim import Adam
    ps = [torch.nn.Parameter(torch.randn(6, 4, device="cuda", generator=gen(i))) for i in range(2)]
    opt = Adam([{"params": ps[:1]}, {"params": ps[1:]}], max_grad_norm=limit)
    for p in ps:
        p.grad = torch.ones_like(p)
    opt.step()
    kept = [t.clone() for p in ps for t in (p.detach(), *opt.state[p].values())]
    good = opt.state[ps[1]]["exp_avg"]
    opt.state[ps[1]]["exp_avg"] = good.t().contiguous().t()               # not laid out as the parameter
    with pytest.raises(ValueError):
        opt.step()
    assert [group["step"] for group in opt.param_groups] == [1, 1]
    assert all(torch.equal(a, b) for a, b in zip(kept, [t for p in ps for t in (p.detach(), *opt.state[p].values())]))
    opt.state[ps[1]]["exp_avg"] = good
    opt.step()
    assert [group["step"] for group in opt.param_groups] == [2, 2] and all(bool((p.detach() != k).all()) for p, k in zip(ps, kept[::3]))


def test_tangents_are_refused():
    """Forward mode, through the lookup, its backward and the steps behind it; beside a dual level everything works as ever."""
    from torch.autograd import forward_ad
    from sparc_amd.embedding import embedding_grad, embedding_lookup
    from sparc_amd.optim import Adam, adam_step_, clip_grad_norm_
    ids, t = torch.tensor([1, 4, 1], device="cuda"), torch.randn(5, 3, device="cuda", generator=gen(1))
    leaf = t.clone().requires_grad_()
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(t, torch.ones_like(t))
        w = forward_ad.make_dual(t[:3].clone(), torch.ones(3, 3, device="cuda"))
        p = torch.nn.Parameter(t.clone())
        p.grad = dual
        state = [torch.zeros_like(t) for _ in range(2)]
        for bad in (lambda: embedding_lookup(ids, dual), lambda: embedding_grad(ids, w, 5), lambda: clip_grad_norm_([p], 1.0),
                    lambda: adam_step_([p.detach()], [dual], state[:1], state[1:], 1), lambda: Adam([p]).step(),
                    lambda: embedding_lookup(ids, forward_ad.make_dual(leaf, torch.ones_like(t))),
                    lambda: embedding_lookup(ids, leaf).backward(w)):
            with pytest.raises(NotImplementedError):
                bad()
        assert torch.equal(embedding_lookup(ids, t), t[ids])
        embedding_lookup(ids, leaf).backward(t[:3])
        assert torch.equal(leaf.grad, embedding_grad(ids, t[:3], 5))
    g = t[:3].clone().requires_grad_()
    with pytest.raises(RuntimeError, match="not differentiable"):
        embedding_grad(ids, g, 5)
    with torch.no_grad():
        assert torch.equal(embedding_grad(ids, g, 5), leaf.grad)
    assert torch.equal(embedding_grad(ids, g.detach(), 5), leaf.grad)


def test_graphed_steps_with_a_frozen_table():
    """Rows that are not trained: graphed steps go as the eager ones with the same optimiser, and the table stays."""
    from test_gpu_node_table import ARCH, sharded
    dev = torch.device("cuda:0")
    heads = [np.random.RandomState(i).permutation(260)[:ARCH["output_dim"]] for i in range(6)]
    got = []
    for graphed in (True, False):
        tr = sharded(dev, max_grad_norm=0.05, hip_graph=graphed)
        if not graphed:
            tr.optimizer = torch.optim.Adam(tr.net.parameters(), lr=torch.tensor(1e-2, device=dev), fused=True, capturable=True)
        tr.net.node_table.weight.requires_grad_(False)
        table = tr.net.node_table.weight.clone()
        losses = [tr.step(s % 2, (s // 2) % 2, heads[s]) for s in range(6)]
        assert torch.equal(table, tr.net.node_table.weight) and tr.net.node_table.weight.grad is None
        got.append(torch.stack(losses + [p.detach().double().sum() for p in tr.net.parameters()]))
    assert torch.equal(*got) and bool(torch.isfinite(got[0]).all())


def test_capture_asks_for_the_stream_that_made_the_leafs_node():
    """Not for the stream of the first lookup: the node may be another operation's."""
    from sparc_amd.embedding import _leaf_stream, embedding_grad, embedding_lookup, refuse_capture_beside_eager_graph
    table = torch.randn(300, 24, device="cuda", generator=gen(70), requires_grad=True)
    ids, w = make_ids("zipf", 1000, 300, 71), torch.randn(1000, 24, device="cuda", generator=gen(72))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    assert _leaf_stream(table) == -1 and _leaf_stream(table.detach()) == -1 and _leaf_stream(table * 1) == -1
    other = (table * 2).sum()                                             # on the default stream, before any lookup
    with torch.cuda.stream(side):
        eager = embedding_lookup(ids, table)
    assert _leaf_stream(table) == 0
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="is alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            embedding_lookup(ids, table).backward(w)
    del eager, other
    torch.cuda.synchronize()
    assert _leaf_stream(table) == -1
    with torch.cuda.stream(side):
        other = (table * 2).sum()                                         # on a stream that can join a capture
    eager = embedding_lookup(ids, table)                                  # on the default stream
    assert _leaf_stream(table) > 0
    refuse_capture_beside_eager_graph(table)
    refuse_capture_beside_eager_graph(table.detach())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        embedding_lookup(ids, table).backward(w)
    for turn in range(3):
        w.copy_(torch.randn(w.shape, device="cuda", generator=gen(73 + turn)))
        graph.replay()
        assert torch.equal(table.grad, embedding_grad(ids, w, 300))
        torch.cuda.synchronize()


def test_graphed_steps_ask_for_every_parameter():
    from test_gpu_node_table import ARCH, sharded
    tr = sharded(torch.device("cuda:0"), hip_graph=True)
    head = np.arange(ARCH["output_dim"])
    for p in (tr.net.node_table.weight, tr.net.mlp_parameters()[0], tr.net.mlp_parameters()[-1]):
        kept = (p * 2).sum()                                              # on the default stream, and alive
        with pytest.raises(RuntimeError, match="is alive"):
            tr.step(0, 1, head)
        del kept
    assert np.isfinite([float(tr.step(0, 1, head)) for _ in range(3)]).all()


@pytest.mark.parametrize("n", [9, 5000, 300_000])
def test_gradients_that_overlap_in_part_are_refused(n):
    """And nothing is scaled; neighbours in one bucket, in any order, are no overlap."""
    from sparc_amd.optim import Adam, adam_step_, clip_grad_norm_
    from test_gpu_clip import check_clip, params_of
    for dtype in (torch.float32, torch.bfloat16):
        flat = torch.randn(2 * n, device="cuda", generator=gen(n)).to(dtype)
        kept = flat.clone()
        for bad in ([flat[:n], flat[n - 1:]], [flat[n - 1:], flat[:n]], [flat, flat[3:4]], [flat[1:2], flat[:n], flat[n:]]):
            with pytest.raises(ValueError):
                clip_grad_norm_(params_of(bad), 0.1)
        assert torch.equal(flat, kept)
        check_clip([flat[n:], flat[1:n], flat[:1]], 0.1)
    flat = torch.randn(4 * n, device="cuda", generator=gen(n + 1))
    g, kept = torch.ones(n, device="cuda"), flat.clone()
    for limit in (None, 1.0):
        for bad in ((flat[:n], g, flat[n - 1:2 * n - 1], flat[2 * n:3 * n]), (flat[:n], flat[n - 1:2 * n - 1], flat[2 * n:3 * n], flat[3 * n:]),
                    (flat[:n], g, flat[n:2 * n], flat[2 * n - 1:3 * n - 1])):
            with pytest.raises(ValueError):
                adam_step_(*([t] for t in bad), 1, max_grad_norm=limit)
        a, b = torch.nn.Parameter(flat[:n]), torch.nn.Parameter(flat[n - 1:2 * n - 1])
        a.grad, b.grad = g, g
        with pytest.raises(ValueError):
            Adam([a, b], max_grad_norm=limit).step()
        many = [[torch.zeros(3, device="cuda") for _ in range(40)] for _ in range(3)]   # (more than one launch takes)
        many[0][39] = many[1][38][1:]
        many[1][39], many[2][39] = torch.zeros(2, device="cuda"), torch.zeros(2, device="cuda")
        with pytest.raises(ValueError):
            adam_step_(many[0], [torch.ones_like(t) for t in many[0]], *many[1:], 1, max_grad_norm=limit)
        assert not any(bool((t != 0).any()) for of in many for t in of)
    assert torch.equal(flat, kept)
    adam_step_([flat[:n]], [g], [flat[n:2 * n].zero_()], [flat[2 * n:3 * n].zero_()], 1)      # neighbours: fine
    assert bool((flat[:n] != kept[:n]).all()) and torch.equal(flat[3 * n:], kept[3 * n:])


def test_the_norm_of_no_gradient_is_on_the_device():
    from sparc_amd.optim import clip_grad_norm_
    p = torch.nn.Parameter(torch.zeros(3, device="cuda"))
    norm = clip_grad_norm_((x for x in [p]), 1.0)
    assert norm.device == p.device and norm.dtype == torch.float32 and norm.shape == () and float(norm) == 0.0
    assert float(clip_grad_norm_([], 1.0)) == 0.0                         # (no tensor to say which device)


@pytest.mark.parametrize("groups", [1, 2])
def test_a_shared_transposed_gradient_counts_once(groups):
    """As clip_grad_norm_ counts it, though Adam copies it into the parameters' layout."""
    from sparc_amd.optim import Adam, clip_grad_norm_
    ps = [torch.nn.Parameter(torch.zeros(6, 4, device="cuda")) for _ in range(3)]
    g = torch.randn(4, 6, device="cuda", generator=gen(1)).t()
    ps[0].grad, ps[1].grad, ps[2].grad = g, g, torch.randn(6, 4, device="cuda", generator=gen(2))
    opt = Adam([{"params": ps}] if groups == 1 else [{"params": ps[:1]}, {"params": ps[1:]}], max_grad_norm=0.5)
    opt.step()
    moments = [opt.state[p]["exp_avg"] for p in ps]
    assert torch.equal(moments[0], moments[1])
    kept = [p.grad.clone() for p in ps]
    assert torch.equal(opt.grad_norm, clip_grad_norm_(ps, 0.5))
    for m, p, k in zip(moments, ps, kept):    # 0.1 of the clipped gradient: factor, product, difference and sum in float32
        assert bool(((m.double() - 0.1 * p.grad.double()).abs() <= 8 * 2.0 ** -24 * k.double().abs()).all())


@pytest.mark.parametrize("pattern", ["uniform", "one", "zipf"])
@pytest.mark.parametrize("n,rows,dim,dtype", [
    (8192, 3000, 512, torch.float32), (8192, 3000, 513, torch.float32), (8192, 3000, 1024, torch.float16), (8192, 3000, 1025, torch.float16),
    (8192, 900, 1024, torch.bfloat16), (8191, 900, 1025, torch.bfloat16), (512, 70, 8192, torch.float32), (513, 70, 8192, torch.float32),
    (512, 70, 16384, torch.bfloat16), (513, 70, 16384, torch.bfloat16), (4096, 3000, 1024, torch.float32), (4097, 3000, 1024, torch.float32)])
def test_gradient_on_both_sides_of_the_one_launch_rule(pattern, n, rows, dim, dtype):
    """One launch takes up to 8192 tokens and 16 MiB of gradient, in rows of up to 32 KiB."""
    from sparc_amd._lib import lib
    from sparc_amd.embedding import DTYPES, embedding_grad
    size = 4 if dtype == torch.float32 else 2
    sorts = lib.sparc_embedding_grad_workspace_bytes(n, rows, dim, DTYPES[dtype]) > 0
    assert sorts == (n * dim * size > 16 << 20)
    ids = make_ids(pattern, n, rows, n + dim)
    g = torch.randn(n, dim, device="cuda", generator=gen(n + rows)).to(dtype)
    got = embedding_grad(ids, g, rows, scale=-1.5)
    check_grad(got, ids, g, rows, -1.5)
    assert torch.equal(got, embedding_grad(ids.int(), g, rows, scale=-1.5))


@pytest.mark.parametrize("limit", [None, 1.0])
def test_memory_that_groups_share_is_refused_before_any_moves(limit):
    from sparc_amd.optim import Adam
    flat = torch.randn(3000, device="cuda", generator=gen(8))
    kept = flat.clone()
    for second in (flat[999:2000], flat[:1000]):
        ps = [torch.nn.Parameter(flat[:1000]), torch.nn.Parameter(second)]
        for p in ps:
            p.grad = torch.ones_like(p)
        opt = Adam([{"params": [p]} for p in ps], max_grad_norm=limit)
        with pytest.raises(ValueError):
            opt.step()
        assert torch.equal(flat, kept) and [group.get("step", 0) for group in opt.param_groups] == [0, 0]
    ps = [torch.nn.Parameter(flat[:1000]), torch.nn.Parameter(flat[1000:2000])]
    for p in ps:
        p.grad = torch.ones_like(p)
    Adam([{"params": [p]} for p in ps], max_grad_norm=limit).step()
    assert bool((flat[:2000] != kept[:2000]).all()) and torch.equal(flat[2000:], kept[2000:])
