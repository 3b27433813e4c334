"""The global gradient norm, clipping and the clipped Adam step (sparc_amd/optim.py) against their formulas in 64 bits.

Tolerances.  u = 2^-24.  Norm: float64 sums, one rounding to float32 (u).  Clipped gradients: the coefficient rounded to
float32 (u), one float32 product (u), one rounding to the type (its half step h; half subnormals 2^-25).  Adam: g' carries
3 u (coefficient, product, weight decay) of |g| + |weight_decay p|; m is a sum of three terms, v of two products: the bounds
are in adam_bounds."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U, SLACK = 2.0 ** -24, 1.01
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def params_of(grads):
    out = []
    for g in grads:
        p = torch.nn.Parameter(torch.empty(g.shape, dtype=g.dtype, device="cuda"))
        p.grad = g
        out.append(p)
    return out


def norm64(grads):
    return math.sqrt(sum(float(g.double().square().sum()) for g in grads))


def check_clip(grads, max_norm):
    from sparc_amd.optim import clip_grad_norm_
    before = [g.clone().double() for g in grads]
    norm = clip_grad_norm_(params_of(grads), max_norm)
    want = norm64(before)
    assert norm.dtype == F32 and norm.dim() == 0 and abs(float(norm) - want) <= SLACK * U * want + 2.0 ** -149
    coef = min(1.0, max_norm / (want + 1e-6))
    for g, b in zip(grads, before):
        w = b * coef
        h = (0.0 if coef == 1.0 else SLACK * (2 * U + (HALF[g.dtype] if g.dtype != F32 else 0.0)))
        assert bool(((g.double() - w).abs() <= h * w.abs() + TINY[g.dtype]).all())
    return norm


@pytest.mark.parametrize("sizes,dtypes", [
    ([1], [F32]), ([3, 0, 5], [F32]), ([4096], [F32]), ([4097, 1, 8191, 0], [F32, BF16, F16, F32]),
    ([10 * 1024, 1024, 1024 * 1024, 1024, 512 * 1024, 512, 47 * 512, 47], [F32]), ([100003], [BF16]), ([65537, 8192], [F16]),
    ([0], [F32]), ([7] * 300, [F32, BF16]), ([60_000_001], [F32]), ([500_003] * 130, [F32]), ([3, 130_000_000, 9], [BF16]), (list(range(1, 129)), [F16]), ([33333] * 129, [F32]), ([5_000_011], [F32, BF16])])
def test_clip(sizes, dtypes):
    for max_norm in (0.5, 1e9):
        grads = [(torch.randn(s, device="cuda", generator=gen(i)) * 2.0 ** (i % 5)).to(dtypes[i % len(dtypes)]) for i, s in enumerate(sizes)]
        check_clip(grads, max_norm)


def test_clip_repeats_bit_for_bit_and_agrees_with_the_bound():
    from sparc_amd.optim import clip_grad_norm_
    grads = [torch.randn(s, device="cuda", generator=gen(s)) for s in (3_000_000, 77, 1_000_001)]
    copies = [[g.clone() for g in grads] for _ in range(2)]
    norms = [clip_grad_norm_(params_of(c), 2.0) for c in copies]
    assert torch.equal(*norms) and all(torch.equal(a, b) for a, b in zip(*copies))
    assert abs(norm64(copies[0]) - 2.0) < 2.0 * 1e-6


def test_clip_ranges_that_leave_float32():
    """Squares below and above float32's range: the sums are in float64."""
    for size in (1e-30, 1e25):
        grads = [torch.full((1000,), size, device="cuda"), torch.full((77,), 3 * size, device="cuda")]
        want = norm64(grads)
        norm = check_clip(grads, want / 2 if size > 1 else 1.0)
        assert float(norm) > 0


def test_clip_of_what_is_not_finite():
    from sparc_amd.optim import clip_grad_norm_
    a, b = torch.tensor([1.0, float("inf")], device="cuda"), torch.ones(5000, device="cuda")
    assert math.isinf(float(clip_grad_norm_(params_of([a, b]), 1.0)))
    assert float(a[0]) == 0.0 and math.isnan(float(a[1])) and bool((b == 0).all())
    a, b = torch.tensor([float("nan")], device="cuda"), torch.ones(5000, device="cuda")
    assert math.isnan(float(clip_grad_norm_(params_of([a, b]), 1.0))) and bool(b.isnan().all())
    a = torch.tensor([1.0, float("inf")], device="cuda")
    assert math.isinf(float(clip_grad_norm_(params_of([a]), float("inf")))) and a.tolist() == [1.0, float("inf")]
    z = torch.zeros(100, device="cuda")
    assert float(clip_grad_norm_(params_of([z]), 0.0)) == 0.0 and bool((z == 0).all())
    g = torch.ones(100, device="cuda")
    clip_grad_norm_(params_of([g]), 0.0)
    assert bool((g == 0).all())


def test_clip_layouts_views_and_duplicates():
    from sparc_amd.optim import clip_grad_norm_
    bucket = torch.randn(1000, device="cuda", generator=gen(1))
    for dtype in (F32, BF16, F16):
        flat = bucket.to(dtype).clone()
        views = [flat[1:8].view(7, 1), flat[8:608].view(20, 30).t(), flat[609:609 + 24].view(2, 3, 4).permute(2, 0, 1)]
        kept = flat.clone()
        check_clip(views, 0.25)
        assert torch.equal(flat[[0, 608]], kept[[0, 608]]) and torch.equal(flat[633:], kept[633:])
    p, q = torch.nn.Parameter(torch.zeros(9, device="cuda")), torch.nn.Parameter(torch.zeros(3, device="cuda"))
    assert float(clip_grad_norm_([q], 1.0)) == 0.0                     # no gradient at all
    p.grad = torch.full((9,), 2.0, device="cuda")
    assert float(clip_grad_norm_([p, q, p], 3.0)) == 6.0               # the same gradient twice counts and is scaled once
    assert bool((p.grad == 2.0 * np.float32(3.0 / (6.0 + 1e-6))).all())
    p.grad.fill_(2.0)
    assert float(clip_grad_norm_(p, 3.0)) == 6.0                       # one tensor
    assert float(clip_grad_norm_((x for x in [p]), 1e9)) > 0           # a generator


def adam_bounds(p0, g, m0, v0, coef, step, lr, b1, b2, eps, wd):
    """(p, m, v) after the step in 64 bits and how far float32 may be off."""
    p0, g, m0, v0 = (t.double() for t in (p0, g, m0, v0))
    size = (coef * g).abs() + (wd * p0).abs()
    g = coef * g + wd * p0
    m, v = b1 * m0 + (1 - b1) * g, b2 * v0 + (1 - b2) * g * g
    # m = m0 + (1 - b1) (g - m0): g off by 3 u, difference, constant, sum
    dm = SLACK * U * (4 * (1 - b1) * (size + m0.abs()) + 2 * m.abs() + 2 * (1 - b1) * (g.abs() + m0.abs()))
    # v = b2 v0 + (1 - b2) g g: g twice, constants, products, sum
    dv = SLACK * U * (4 * b2 * v0.abs() + (1 - b2) * (6 * size * g.abs() + 4 * g * g) + 2 * v)
    step_size, root = lr / (1 - b1 ** step), 1 / math.sqrt(1 - b2 ** step)
    denom = v.sqrt() * root + eps
    # sqrt off by dv / (2 sqrt v); square root, its factor, eps and sum, quotient, rate, difference
    drel = dv / (2 * v).clamp(min=1e-300) + 10 * U
    move = step_size * m / denom
    dp = SLACK * (move.abs() * drel + step_size * dm / denom + U * (p0.abs() + move.abs()) * 2)
    return (p0 - move, m, v), (dp, dm, dv)


@pytest.mark.parametrize("sizes", [[1], [1000, 0, 3], [5, 1023, 1024, 1025, 300001], [47] * 130, [2_000_003], [9, 13_000_001]])
@pytest.mark.parametrize("max_norm,wd", [(0.5, 0.0), (2.0, 0.01), (1e9, 0.1)])
def test_adam_step(sizes, max_norm, wd):
    from sparc_amd.optim import adam_step_
    p = [torch.randn(s, device="cuda", generator=gen(s + 1)) for s in sizes]
    g = [torch.randn(s, device="cuda", generator=gen(s + 2)) for s in sizes]
    m = [torch.randn(s, device="cuda", generator=gen(s + 3)) * 0.1 for s in sizes]
    v = [torch.rand(s, device="cuda", generator=gen(s + 4)) * 0.01 for s in sizes]
    start = [[t.clone() for t in of] for of in (p, g, m, v)]
    norm = adam_step_(p, g, m, v, 7, lr=0.01, weight_decay=wd, max_grad_norm=max_norm)
    want = norm64(g)
    assert abs(float(norm) - want) <= SLACK * U * want
    assert all(torch.equal(a, b) for a, b in zip(g, start[1]))
    coef = min(1.0, max_norm / (want + 1e-6))
    for i in range(len(sizes)):
        exact, off = adam_bounds(*(of[i] for of in start), coef, 7, 0.01, 0.9, 0.999, 1e-8, wd)
        for name, got, w, d in zip("pmv", (p[i], m[i], v[i]), exact, off):
            assert bool(((got.double() - w).abs() <= d + 1e-37).all()), (name, float(((got.double() - w).abs() - d).max()))
    if max_norm > 1e6:     # nothing to clip: the unclipped update's bits
        q = [[t.clone() for t in of] for of in start]
        assert adam_step_(*q, 7, lr=0.01, weight_decay=wd) is None
        assert all(torch.equal(a, b) for got, ref in zip((p, m, v), (q[0], q[2], q[3])) for a, b in zip(got, ref))


def test_adam_class_clips_over_all_groups():
    from sparc_amd.optim import Adam, adam_step_
    shapes = [(40, 30), (30,), (5,)]
    a = [torch.nn.Parameter(torch.randn(s, device="cuda", generator=gen(7))) for s in shapes]
    b = [torch.nn.Parameter(x.detach().clone()) for x in a]
    opt = Adam([{"params": a[:1], "lr": 0.01}, {"params": a[1:], "lr": 0.1}], max_grad_norm=0.7)
    ms, vs = [torch.zeros_like(x) for x in b], [torch.zeros_like(x) for x in b]
    for step in (1, 2, 3):
        grads = [torch.randn(s, device="cuda", generator=gen(70 + step)) for s in shapes]
        for x, g in zip(a, grads):
            x.grad = g.t().contiguous().t() if g.dim() == 2 else g          # (a transposed gradient too)
        opt.step()
        assert abs(float(opt.grad_norm) - norm64(grads)) <= SLACK * U * norm64(grads)
        coef = np.float32(min(1.0, 0.7 / (norm64(grads) + 1e-6)))
        clipped = [g * float(coef) for g in grads]
        data = [x.detach() for x in b]
        adam_step_(data[:1], clipped[:1], ms[:1], vs[:1], step, lr=0.01)
        adam_step_(data[1:], clipped[1:], ms[1:], vs[1:], step, lr=0.1)
    for x, y in zip(a, b):   # the products are rounded here and fused there: 3 steps of at most 10 u of a move of about lr
        assert float((x - y).abs().max()) < 3 * 0.1 * 64 * U + 3 * U * float(y.abs().max())
    import copy
    import pickle
    assert pickle.loads(pickle.dumps(opt)).defaults["max_grad_norm"] == 0.7 and copy.deepcopy(opt).param_groups[0]["max_grad_norm"] == 0.7
    state = opt.state_dict()
    for group in state["param_groups"]:
        del group["max_grad_norm"]                                          # a state from before it existed
    opt.load_state_dict(state)
    assert opt.param_groups[1]["max_grad_norm"] == 0.7
    opt.param_groups[1]["max_grad_norm"] = 3.0
    with pytest.raises(ValueError):
        opt.step()


def test_clip_captured_twice_and_on_other_streams():
    from sparc_amd.optim import clip_grad_norm_
    sets = [params_of([torch.zeros(s, device="cuda") for s in sizes]) for sizes in ((70_001, 33), (5, 1_000_000))]
    graphs = []
    torch.cuda.synchronize()
    for ps in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            norm = clip_grad_norm_(ps, 0.3)
        graphs.append((graph, norm))
    for turn in range(4):
        fresh = [[torch.randn(p.shape, device="cuda", generator=gen(turn + i)) for i, p in enumerate(ps)] for ps in sets]
        for ps, of in zip(sets, fresh):
            for p, g in zip(ps, of):
                p.grad.copy_(g)
        for graph, _ in graphs:
            graph.replay()
        for (_, norm), ps, of in zip(graphs, sets, fresh):
            ref = params_of([g.clone() for g in of])
            assert torch.equal(clip_grad_norm_(ref, 0.3), norm)
            assert all(torch.equal(p.grad, q.grad) for p, q in zip(ps, ref))
        torch.cuda.synchronize()
    work = [[torch.randn(2_000_000, device="cuda", generator=gen(80 + i))] for i in range(2)]
    want = [[g.clone() for g in of] for of in work]
    norms = [clip_grad_norm_(params_of(of), 1.0) for of in want]
    torch.cuda.synchronize()
    got = []
    for of in work:
        with torch.cuda.stream(torch.cuda.Stream()):
            got.append(clip_grad_norm_(params_of(of), 1.0))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(norms, got)) and all(torch.equal(a[0], b[0]) for a, b in zip(work, want))


def test_refusals_on_the_device():
    from sparc_amd.optim import Adam, adam_step_, clip_grad_norm_
    g = torch.randn(8, 8, device="cuda")
    with pytest.raises(ValueError):
        clip_grad_norm_(params_of([g]), -1.0)
    with pytest.raises(ValueError):
        clip_grad_norm_(params_of([g]), float("nan"))
    with pytest.raises(ValueError):
        clip_grad_norm_(params_of([g.double()]), 1.0)
    p = torch.nn.Parameter(torch.zeros(8, 4, device="cuda"))
    p.grad = g[:, ::2]                                     # gaps between its elements
    with pytest.raises(ValueError):
        clip_grad_norm_([p], 1.0)
    with pytest.raises(ValueError):
        Adam([p], max_grad_norm=-1.0)
    z = torch.zeros(4, device="cuda")
    with pytest.raises(ValueError):
        adam_step_([z], [z.double()], [z], [z], 1)
    with pytest.raises(ValueError):
        adam_step_([z], [z], [z], [z[:3]], 1, max_grad_norm=1.0)
    with pytest.raises(ValueError):
        adam_step_([z], [], [z], [z], 1)


def test_gradients_that_share_memory():
    """Counted and scaled once, by whatever tensors the memory is met; an overlap from the same element on is refused."""
    from sparc_amd.optim import adam_step_, clip_grad_norm_
    flat = torch.full((70_000,), 2.0, device="cuda")
    ps = params_of([flat, flat.view(700, 100), flat.view(100, 700).t()])
    want = norm64([flat])
    coef = np.float32(3.0 / (want + 1e-6))
    assert abs(float(clip_grad_norm_(ps, 3.0)) - want) <= SLACK * U * want
    assert bool((flat == 2.0 * coef).all())
    with pytest.raises(ValueError):
        clip_grad_norm_(params_of([flat, flat[:5]]), 1.0)
    empty = [torch.zeros(0, device="cuda") for _ in range(3)]
    assert float(clip_grad_norm_(params_of(empty), 1.0)) == 0.0
    assert float(clip_grad_norm_(params_of([*empty, torch.full((4,), 3.0, device="cuda")]), 100.0)) == 6.0
    new = lambda: [torch.ones(33, device="cuda") for _ in range(2)]  # noqa: E731
    g = torch.full((33,), 5.0, device="cuda")
    p, m, v = new(), new(), new()
    norm = adam_step_(p, [g, g], m, v, 1, max_grad_norm=1.0)
    assert abs(float(norm) - 5.0 * math.sqrt(33.0)) <= SLACK * U * 5.0 * math.sqrt(33.0)
    p1, m1, v1 = (t[:1] for t in (new(), new(), new()))
    adam_step_(p1, [g], m1, v1, 1, max_grad_norm=1.0)
    assert torch.equal(p[0], p1[0]) and torch.equal(p[1], p1[0]) and torch.equal(v[1], v1[0])
    t = new()
    for bad in (([t[0], t[0]], new(), new(), new()), (new(), new(), [t[0], t[0]], new()), (new(), new(), [t[0], t[1]], [t[1], new()[0]]),
                ([t[0]], [t[0]], new()[:1], new()[:1])):
        with pytest.raises(ValueError):
            adam_step_(*bad, 1)


def test_what_is_written_counts_as_written():
    """Autograd refuses to go back through values that a step or a clipping has replaced."""
    from sparc_amd.optim import adam_step_, clip_grad_norm_
    p = torch.randn(50, device="cuda", generator=gen(3)).requires_grad_()
    state = [torch.zeros(50, device="cuda") for _ in range(3)]
    for limit in (None, 1.0):
        loss = (p * p).sum()
        adam_step_([p], state[:1], state[1:2], state[2:], 1, max_grad_norm=limit)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            loss.backward()
    loss = (p ** 3).sum()
    loss.backward(create_graph=True)
    penalty = (p.grad * p.grad).sum()
    clip_grad_norm_([p], 1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        penalty.backward()
    p.grad = None


@pytest.mark.parametrize("sizes", [[1], [3, 0, 5], [16384], [255, 256, 257, 1023], [131072], [2048] * 60, [1] * 64, [1] * 65, [131073], [7, 2049, 100_001],
                                   [256] * 64, [257] * 32, [16385], [0, 0], [32768],
                                   [32769], [65536], [65537], [1024] * 32, [1023] * 64])
def test_short_lists_and_the_first_longer_ones(sizes):
    """What one workgroup holds (128 KiB of gradients to clip, 16384 parameters to update) and what is just beyond it."""
    from sparc_amd.optim import adam_step_, clip_grad_norm_
    bucket = {d: torch.randn(sum(sizes) + len(sizes) + 1, device="cuda", generator=gen(5)).to(d) for d in (F32, BF16, F16)}
    for kinds in ([F32], [BF16], [F16], [F32, BF16, F16]):
        for odd in (0, 1):                                     # one after another in memory, at any element
            views, at = [], 0
            kept = {d: t.clone() for d, t in bucket.items()}
            for i, s in enumerate(sizes):
                views.append(kept[kinds[i % len(kinds)]][at + odd:at + odd + s])
                at += s + 1
            check_clip(views, 0.25)
            touched = {d: torch.ones(t.numel(), dtype=torch.bool, device="cuda") for d, t in kept.items()}
            at = 0
            for i, s in enumerate(sizes):
                touched[kinds[i % len(kinds)]][at + odd:at + odd + s] = False
                at += s + 1
            assert all(torch.equal(kept[d][touched[d]], bucket[d][touched[d]]) for d in kept)
    new = lambda seed: [torch.randn(s, device="cuda", generator=gen(seed + i)) for i, s in enumerate(sizes)]  # noqa: E731
    p, g, m = new(100), new(200), new(300)
    v = [t * t for t in new(400)]
    want = norm64(g)
    before = [[t.clone() for t in c] for c in (p, g, m, v)]
    norm = adam_step_(p, g, m, v, 3, lr=0.01, weight_decay=0.02, max_grad_norm=0.5)
    assert abs(float(norm) - want) <= SLACK * U * want + 2.0 ** -149
    coef = min(1.0, 0.5 / (want + 1e-6))
    for i in range(len(sizes)):
        if sizes[i] == 0:
            continue
        exact, bounds = adam_bounds(*(c[i] for c in before), coef, 3, 0.01, 0.9, 0.999, 1e-8, 0.02)
        for got, w, off in zip((p[i], m[i], v[i]), exact, bounds):
            assert bool(((got.double() - w).abs() <= off + 1e-37).all())
        assert torch.equal(g[i], before[1][i])


@pytest.mark.parametrize("sizes", [[300, 5], [70_001, 33], [64] * 20])
def test_adam_step_captured_and_on_another_stream(sizes):
    """Replays with new gradients, eager work between them: the same bits as eager calls (the number of the step is the
    capture's)."""
    from sparc_amd.optim import adam_step_, clip_grad_norm_
    new = lambda seed: [torch.randn(s, device="cuda", generator=gen(seed + i)) for i, s in enumerate(sizes)]  # noqa: E731
    p, g, m, v = new(1), new(2), new(3), [t * t for t in new(4)]
    q, n, w = ([t.clone() for t in c] for c in (p, m, v))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = adam_step_(p, g, m, v, 5, lr=0.02, max_grad_norm=0.7)
    for turn in range(4):
        fresh = new(10 * turn + 20)
        for a, b in zip(g, fresh):
            a.copy_(b)
        graph.replay()
        if turn % 2:
            with torch.cuda.stream(torch.cuda.Stream()):
                torch.cuda.current_stream().wait_stream(torch.cuda.default_stream())
                eager = adam_step_(q, fresh, n, w, 5, lr=0.02, max_grad_norm=0.7)
                torch.cuda.default_stream().wait_stream(torch.cuda.current_stream())
        else:
            eager = adam_step_(q, fresh, n, w, 5, lr=0.02, max_grad_norm=0.7)
        assert torch.equal(eager, norm) and all(torch.equal(a, b) for x, y in ((p, q), (m, n), (v, w)) for a, b in zip(x, y))
        want = norm64(fresh)
        assert abs(float(clip_grad_norm_(params_of(fresh), 0.7)) - want) <= SLACK * U * want
        torch.cuda.synchronize()
