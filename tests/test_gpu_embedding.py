"""Table lookup by token and its gradient (sparc_amd/embedding.py) against their definitions in 64 bits.

Tolerances.  u = 2^-24 is half a step of float32, h half a step of the result's type (2^-24, 2^-8, 2^-11).  Lookup: one
float32 product (u) and one rounding (h).  Gradient: a row of c places is a float32 sum of c terms, off by at most
(c - 1) u sum |g| in any order, then one product with the scale (u) and one rounding (h).  Half: results below 2^-14 are
multiples of 2^-24, off by 2^-25 at most.  SLACK covers the products of these errors."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U, SLACK = 2.0 ** -24, 1.01
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def make_ids(pattern, n, rows, seed):
    g = gen(seed)
    if pattern == "uniform":
        return torch.randint(rows, (n,), generator=g, device="cuda")
    if pattern == "zipf":
        u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
        return (torch.exp(u * np.log(rows + 1.0)) - 1.0).long().clamp_(0, rows - 1)
    if pattern == "one":
        return torch.full((n,), rows // 2, device="cuda")
    if pattern == "falling":
        return (torch.arange(n - 1, -1, -1, device="cuda") * rows) // max(n, 1)
    if pattern == "lengths":   # rows of 0, 1, 63, 64, 65, 127, 128, 129 and 1000 places, shuffled
        lens = torch.tensor([0, 1, 63, 64, 65, 0, 127, 128, 129, 1000], device="cuda")
        ids = torch.repeat_interleave(torch.arange(10, device="cuda"), lens)
        ids = ids * max(rows // 10, 1) % rows
        return ids[torch.randperm(ids.numel(), generator=g, device="cuda")]
    if pattern == "stray":     # tokens that are no rows, next to ones that are
        ids = torch.randint(-3, rows + 3, (n,), generator=g, device="cuda")
        ids[::7] = 2 ** 62 if rows > 2 else -1
        return ids
    raise ValueError(pattern)


def grad64(ids, g, rows, scale, padding_idx=None):
    """(the gradient, sum |g| per row, places per row) in 64 bits."""
    ids, g = ids.reshape(-1), g.reshape(-1, g.shape[-1]).double()
    ok = (ids >= 0) & (ids < rows)
    if padding_idx is not None:
        ok &= ids != padding_idx
    ids, g = ids[ok].long(), g[ok]
    out = torch.zeros(rows, g.shape[1], dtype=torch.float64, device=g.device)
    size = torch.zeros_like(out)
    places = torch.zeros(rows, dtype=torch.float64, device=g.device)
    out.index_add_(0, ids, g)
    size.index_add_(0, ids, g.abs())
    places.index_add_(0, ids, torch.ones(ids.numel(), dtype=torch.float64, device=g.device))
    s = float(np.float32(scale))
    return out * s, size * abs(s), places


def check_grad(got, ids, g, rows, scale=1.0, padding_idx=None):
    want, size, places = grad64(ids, g, rows, scale, padding_idx)
    assert got.shape == want.shape and got.dtype == g.dtype
    bound = SLACK * (places[:, None] * U * size + HALF[g.dtype] * want.abs()) + TINY[g.dtype]
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), float((off - bound).max())
    # (elementwise: torch's selection of 70 million rows returned rows that it had not written)
    assert not bool(((got != 0).any(1) & (places == 0)).any())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,rows,dim", [(1, 1, 1), (5, 3, 2), (1, 2708, 64), (700, 33, 47), (1000, 19717, 100), (257, 50, 7),
                                        (65, 70000, 4), (3, 9, 1030), (20000, 40, 8), (0, 5, 4), (4, 5, 0)])
def test_lookup(n, rows, dim, dtype):
    from sparc_amd.embedding import embedding_lookup
    table = torch.randn(rows, dim, device="cuda", generator=gen(n + dim)).to(dtype)
    for id_dtype in (torch.int32, torch.int64):
        ids = make_ids("uniform", n, rows, 5).to(id_dtype)
        for scale in (1.0, 11.3137085):
            out = embedding_lookup(ids, table, scale=scale)
            want = table[ids.long()].double() * float(np.float32(scale))
            assert out.shape == (n, dim) and out.dtype == dtype
            h = 0.0 if scale == 1.0 else SLACK * (HALF[dtype] + (U if dtype != torch.float32 else 0.0))
            assert bool(((out.double() - want).abs() <= h * want.abs() + TINY[dtype]).all())


def test_lookup_shapes_strides_and_strays():
    from sparc_amd.embedding import embedding_lookup
    base = torch.randn(50, 61, device="cuda", generator=gen(1))
    for dtype in DTYPES:
        wide = base.to(dtype)
        for table in (wide[:, 3:50], wide[1::2, :60], wide[:, :1], wide[7:8, 5:], wide[:, 2:5]):
            ids = make_ids("uniform", 24, table.shape[0], 2).view(2, 3, 4)
            assert torch.equal(embedding_lookup(ids, table), table[ids])
            assert torch.equal(embedding_lookup(ids.transpose(0, 2), table), table[ids.transpose(0, 2)])
            assert embedding_lookup(ids[0, 0, 0], table).shape == (table.shape[1],)
            ids = torch.tensor([0, -1, table.shape[0], -2 ** 40, 2 ** 40, table.shape[0] - 1], device="cuda")
            out = embedding_lookup(ids, table, scale=2.0)
            assert bool(out[1:5].isnan().all()) and torch.equal(out[[0, 5]], (table[[0, -1]] * 2.0).to(dtype))
    special = torch.tensor([[float("inf"), -float("inf"), float("nan"), -0.0]], device="cuda")
    out = embedding_lookup(torch.zeros(2, dtype=torch.int64, device="cuda"), special)
    assert torch.equal(out.view(torch.int32), special.expand(2, 4).contiguous().view(torch.int32))


def test_lookup_far_into_a_large_table():
    from sparc_amd.embedding import embedding_lookup
    rows, dim = 9_000_000, 250          # 2.25e9 elements: offsets beyond 32 bits
    table = torch.zeros(rows, dim, dtype=torch.bfloat16, device="cuda")
    ids = torch.tensor([rows - 1, 0, 8_600_000, rows - 2], device="cuda")
    table[ids] = torch.arange(4 * dim, device="cuda").view(4, dim).to(torch.bfloat16)
    assert torch.equal(embedding_lookup(ids, table, scale=2.0), table[ids] * 2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pattern,n,rows,dim", [
    ("uniform", 0, 7, 5), ("uniform", 1, 1, 1), ("uniform", 3, 2, 3), ("uniform", 140, 2708, 64), ("uniform", 2437, 2708, 64),
    ("uniform", 6600, 19717, 47), ("uniform", 2049, 3000, 16), ("uniform", 5000, 10, 130), ("uniform", 300, 70001, 9),
    ("zipf", 20000, 5000, 257), ("zipf", 70001, 30000, 33), ("zipf", 4096, 64, 1024),
    ("one", 1, 9, 8), ("one", 64, 9, 8), ("one", 65, 9, 8), ("one", 20000, 3, 47), ("one", 9000, 1, 600),
    ("falling", 4000, 4000, 20), ("falling", 9999, 700, 3), ("lengths", 0, 10, 64), ("lengths", 0, 4001, 72),
    ("stray", 5000, 90, 12), ("stray", 100, 1, 4),
    # one launch or the sort: 8192 tokens, 4 MiB of gradient
    ("zipf", 8192, 900, 5), ("zipf", 8193, 900, 5), ("one", 8193, 9, 3), ("one", 8192, 900, 7), ("uniform", 8192, 3000, 128),
    ("uniform", 8192, 3000, 129), ("zipf", 2000, 100_000, 1), ("falling", 8000, 9_000, 16), ("zipf", 16384, 900, 5), ("falling", 16400, 5000, 3), ("stray", 40000, 70, 6),
    ("lengths", 0, 200, 1030), ("zipf", 30000, 20000, 65), ("uniform", 17000, 1, 2), ("uniform", 66000, 2050, 1),
    ("zipf", 300000, 70000, 2)])
def test_gradient(pattern, n, rows, dim, dtype):
    from sparc_amd.embedding import embedding_grad
    ids = make_ids(pattern, n, rows, 3)
    g = torch.randn(ids.numel(), dim, device="cuda", generator=gen(4)).to(dtype)
    got = embedding_grad(ids, g, rows, scale=0.7)
    check_grad(got, ids, g, rows, 0.7)
    if pattern != "stray":
        assert torch.equal(got, embedding_grad(ids.int(), g, rows, scale=0.7))     # and the same bits again
    pad = rows // 2
    check_grad(embedding_grad(ids, g, rows, padding_idx=pad), ids, g, rows, 1.0, pad)


@pytest.mark.parametrize("n,rows,dim", [(5000, 9_000_001, 1), (300, 140_000_000, 1), (300, 70_000_000, 4), (4_500_000, 1000, 1), (3000, 4_300_000, 2), (49_000, 2_449_029, 4)])
def test_gradient_of_many_rows_or_tokens(n, rows, dim):
    from sparc_amd.embedding import embedding_grad
    ids = make_ids("uniform", n, rows, 6)
    g = torch.randn(n, dim, device="cuda", generator=gen(7))
    check_grad(embedding_grad(ids, g, rows), ids, g, rows)


@pytest.mark.parametrize("n,rows,dim,dtype", [(20000, 800_001, 64, torch.float32), (200_003, 1000, 256, torch.float32),
                                              (120_001, 500_000, 1024, torch.bfloat16)])
def test_gradients_that_outgrow_the_cache(n, rows, dim, dtype):
    """The table's zeros, the gradient, both: with streaming accesses."""
    from sparc_amd.embedding import embedding_grad
    ids = make_ids("zipf", n, rows, 16)
    g = torch.randn(n, dim, device="cuda", generator=gen(17)).to(dtype)
    out = embedding_grad(ids, g, rows, padding_idx=1)
    keep = torch.cat([ids.unique()[:3000], torch.randint(rows, (3000,), generator=gen(18), device="cuda")]).unique()
    slot = torch.full((rows,), -1, dtype=torch.int64, device="cuda")
    slot[keep] = torch.arange(keep.numel(), device="cuda")
    of = slot[ids]
    of[ids == 1] = -1
    check_grad(out[keep], of[of >= 0], g[of >= 0], keep.numel())
    touched = torch.zeros(rows, dtype=torch.bool, device="cuda")
    touched[ids] = True
    touched[1] = False
    assert int(((out != 0).any(1) != touched).sum()) == 0


def test_lookup_that_outgrows_the_cache():
    from sparc_amd.embedding import embedding_lookup
    table = torch.randn(5000, 1000, device="cuda", generator=gen(19)).half()
    ids = make_ids("zipf", 110_000, 5000, 20)
    assert torch.equal(embedding_lookup(ids, table, scale=0.5), (table * 0.5)[ids])


def test_gradient_past_32_bit_offsets():
    from sparc_amd.embedding import embedding_grad
    rows, dim = 9_000_000, 250
    ids = torch.tensor([rows - 1, 3, rows - 1, 8_600_000], device="cuda")
    g = torch.randn(4, dim, device="cuda", generator=gen(8)).bfloat16()
    out = embedding_grad(ids, g, rows)
    assert torch.equal(out[rows - 1], (g[0].float() + g[2].float()).bfloat16()) and torch.equal(out[3], g[1])
    assert torch.equal(out[8_600_000], g[3]) and int((out != 0).any(1).sum()) == 3
    del out
    n = 9_000_000                                           # and a gradient of that many elements
    g = torch.zeros(n, dim, dtype=torch.bfloat16, device="cuda")
    g[-1] = 1.5
    ids = torch.arange(n, device="cuda") % 1000
    out = embedding_grad(ids, g, 1000)
    assert bool((out[(n - 1) % 1000] == 1.5).all()) and int((out != 0).any(1).sum()) == 1


def test_gradient_layouts():
    from sparc_amd.embedding import embedding_grad
    ids = make_ids("zipf", 1200, 300, 9)
    for dtype in DTYPES:
        wide = torch.randn(1200, 60, device="cuda", generator=gen(10)).to(dtype)
        for g in (wide[:, 3:50], wide[:, 1:2], wide.flip(0)[:, ::2], wide.t().contiguous().t()):
            check_grad(embedding_grad(ids, g, 300), ids, g, 300)
        one = torch.ones(1, 1, device="cuda", dtype=dtype).expand(1200, 24)          # what sum() sends back
        check_grad(embedding_grad(ids, one, 300), ids, one, 300)
        g3 = wide.view(20, 60, 60)
        check_grad(embedding_grad(ids.view(20, 60), g3, 300), ids, g3, 300)
        assert torch.equal(embedding_grad(ids.view(20, 60).t(), g3.transpose(0, 1), 300),
                           embedding_grad(ids.view(20, 60).t().contiguous(), g3.transpose(0, 1).contiguous(), 300))


def test_autograd_accumulates_and_stops_at_second_order():
    from sparc_amd.embedding import embedding_lookup
    rows, dim = 40, 12
    table = torch.randn(rows, dim, device="cuda", generator=gen(11), requires_grad=True)
    a, b = make_ids("zipf", 300, rows, 12).view(30, 10), make_ids("uniform", 77, rows, 13)
    wa = torch.randn(30, 10, dim, device="cuda", generator=gen(14))
    wb = torch.randn(77, dim, device="cuda", generator=gen(15))

    def loss(t, look):
        return (look(a, t, 1.5) * wa).sum() + (look(b, t, -2.0) * wb).sum()
    loss(table, embedding_lookup).backward()
    plain = table.detach().double().requires_grad_()
    value = loss(plain, lambda i, t, s: t[i] * s)
    value.backward()
    pa, pb = grad64(a, wa, rows, 1.5), grad64(b, wb, rows, -2.0)
    bound = SLACK * ((pa[2] + 1)[:, None] * U * pa[1] + (pb[2] + 1)[:, None] * U * pb[1] + U * plain.grad.abs())
    assert bool(((table.grad.double() - plain.grad).abs() <= bound).all())
    # against differences: the loss is linear in the table, so a difference of any size is its slope
    for r, c in ((0, 0), (3, 11), (39, 5)):
        moved = plain.detach().clone()
        moved[r, c] += 1.0
        slope = float(loss(moved, lambda i, t, s: t[i] * s) - value)
        assert abs(slope - float(table.grad[r, c])) <= float(bound[r, c]) + 1e-9 * float(value.detach().abs() + 1)
    with torch.no_grad():
        assert not embedding_lookup(a, table).requires_grad
    out = embedding_lookup(b, table)
    (first,) = torch.autograd.grad((out * out).sum(), table, create_graph=True)
    with pytest.raises(RuntimeError):
        first.sum().backward()


def test_other_streams_do_not_share_scratch():
    from sparc_amd.embedding import embedding_grad
    rows = 5000
    jobs = [(make_ids("zipf", 30000, rows, 20 + i), torch.randn(30000, 64, device="cuda", generator=gen(30 + i))) for i in range(2)]
    want = [embedding_grad(ids, g, rows) for ids, g in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(embedding_grad(*jobs[i], rows))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(w, want[i]) for w in got[i])


def test_two_captured_graphs():
    """Forward and backward of two lookups captured into two graphs, replayed in turn with new tokens and eager work
    between: every replay equals the eager result bit for bit."""
    from sparc_amd.embedding import EmbeddingLookup, embedding_grad, embedding_lookup
    rows, dim = 700, 48
    table = torch.randn(rows, dim, device="cuda", generator=gen(40), requires_grad=True)
    graphs = []
    for i, n in enumerate((5000, 333)):
        ids, w = torch.zeros(n, dtype=torch.int64, device="cuda"), torch.zeros(n, dim, device="cuda")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(side):
            torch.autograd.grad(embedding_lookup(ids, table, 0.5), table, w)     # (nothing of it lives at the capture)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            out = embedding_lookup(ids, table, 0.5)
            (grad,) = torch.autograd.grad(out, table, w)
            out = out.detach()
        graphs.append((graph, ids, w, out, grad))
    for turn in range(4):
        for i, (graph, ids, w, out, grad) in enumerate(graphs):
            ids.copy_(make_ids("zipf" if turn % 2 else "uniform", ids.numel(), rows, 50 + turn + i))
            w.copy_(torch.randn(w.shape, device="cuda", generator=gen(60 + turn + i)))
            graph.replay()
        for graph, ids, w, out, grad in graphs:
            assert torch.equal(out, embedding_lookup(ids, table.detach(), 0.5))
            assert torch.equal(grad, embedding_grad(ids, w, rows, 0.5))
        torch.cuda.synchronize()
    assert EmbeddingLookup is not None


def test_refusals_on_the_device():
    from sparc_amd.embedding import NodeTable, embedding_grad, embedding_lookup
    table = torch.zeros(4, 8, device="cuda")
    ids = torch.zeros(3, dtype=torch.int64, device="cuda")
    for bad in (lambda: embedding_lookup(ids.float(), table), lambda: embedding_lookup(ids.cpu(), table),
                lambda: embedding_lookup(ids, table.double()), lambda: embedding_lookup(ids, table.t()),
                lambda: embedding_lookup(ids, table[0]), lambda: embedding_lookup(ids, table[:1].expand(4, 8)),
                lambda: embedding_lookup(ids, table, padding_idx=4), lambda: embedding_grad(ids, table, 4),
                lambda: embedding_grad(ids, table[:3].double(), 4), lambda: embedding_grad(ids, table[:3], 4, padding_idx=-1),
                lambda: embedding_grad(ids, table[:3], -1), lambda: NodeTable(0, 3), lambda: NodeTable(3, 3, padding_idx=3)):
        with pytest.raises(ValueError):
            bad()


def test_capture_beside_a_living_eager_graph_is_refused():
    """The earlier graph's leaf keeps the default stream, which no capture may make wait; without it the capture works."""
    from sparc_amd.embedding import embedding_grad, embedding_lookup
    table = torch.randn(300, 24, device="cuda", generator=gen(70), requires_grad=True)
    ids, w = make_ids("zipf", 1000, 300, 71), torch.randn(1000, 24, device="cuda", generator=gen(72))
    want = embedding_grad(ids, w, 300)
    eager = embedding_lookup(ids, table)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="is alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            embedding_lookup(ids, table).backward(w)
    with torch.cuda.graph(torch.cuda.CUDAGraph()):                # a forward alone is no matter
        embedding_lookup(ids, table)
    eager.backward(w)
    assert torch.equal(table.grad, want)
    del eager
    table.grad = None
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        embedding_lookup(ids, table).backward(w)
    for turn in range(3):
        w.copy_(torch.randn(w.shape, device="cuda", generator=gen(73 + turn)))
        graph.replay()
        assert torch.equal(table.grad, embedding_grad(ids, w, 300))
        torch.cuda.synchronize()


def test_lookup_of_more_rows_than_one_launch_takes():
    """A launch has fewer than 2^32 threads along x: 268435440 rows of 33 vectors."""
    from sparc_amd.embedding import embedding_lookup
    n, rows, dim, one = 268_500_000, 1000, 264, 268_435_440
    if torch.cuda.mem_get_info()[0] < 160e9:
        pytest.skip("142 GB of output")
    table = torch.randn(rows, dim, device="cuda", generator=gen(80)).bfloat16()
    ids = torch.arange(n, dtype=torch.int32, device="cuda").remainder_(997)
    out = embedding_lookup(ids, table)
    for a in (0, one // 2, one - 50_000, n - 20_000):
        assert torch.equal(out[a:a + 100_000], table[ids[a:a + 100_000].long()]), a
    del out, ids
    torch.cuda.empty_cache()


@pytest.mark.parametrize("pattern", ["uniform", "zipf", "one", "falling", "stray"])
@pytest.mark.parametrize("n,rows,dim,dtype", [(8192, 11, 2, torch.float32), (8192, 300, 1, torch.float32), (8191, 40_000, 64, torch.float32),
                                              (8000, 2_449_029, 3, torch.bfloat16), (4096, 2, 512, torch.bfloat16), (257, 1, 33, torch.float32),
                                              (1500, 7, 700, torch.float16), (8192, 4000, 256, torch.float16), (513, 3, 1000, torch.float32),
                                              (6000, 100_000_000, 1, torch.float32), (300, 19, 8, torch.bfloat16)])
def test_gradient_of_few_tokens_however_they_fall(pattern, n, rows, dim, dtype):
    """What one launch takes: all tokens in one workgroup or none, runs of every length, in order and out of it."""
    from sparc_amd.embedding import embedding_grad
    ids = make_ids(pattern, n, rows, n + dim)
    g = torch.randn(n, dim, device="cuda", generator=gen(n + rows)).to(dtype)
    got = embedding_grad(ids, g, rows, scale=0.75, padding_idx=rows // 3)
    check_grad(got, ids, g, rows, 0.75, rows // 3)
    assert torch.equal(got, embedding_grad(ids, g, rows, scale=0.75, padding_idx=rows // 3))
    check_grad(embedding_grad(ids.clamp(-1, rows).int(), g, rows, scale=0.75), ids, g, rows, 0.75)


@pytest.mark.parametrize("n", [3, 1001, 8190, 20_001])
def test_tokens_at_any_element_and_nan_in_places_left_out(n):
    """Tokens and gradients that start at any element; what padding and stray tokens carry reaches no row."""
    from sparc_amd.embedding import embedding_grad, embedding_lookup
    rows, pad = 500, 7
    for offset in (1, 2, 3):
        ids = make_ids("stray", n + offset, rows, n)
        g = torch.randn(n + offset, 37, device="cuda", generator=gen(n))
        left_out = (ids < 0) | (ids >= rows) | (ids == pad)
        g[left_out] = torch.tensor([float("nan"), float("inf"), -float("inf")], device="cuda").repeat(13)[:37]
        kept = torch.where(left_out[:, None], torch.zeros_like(g), g)
        for dtype in DTYPES:
            tokens, some, clean = ids[offset:], g.to(dtype)[offset:, 1:], kept.to(dtype)[offset:, 1:]
            got = embedding_grad(tokens, some, rows, padding_idx=pad)
            check_grad(got, tokens, clean, rows, padding_idx=pad)
            assert torch.equal(got, embedding_grad(ids.clamp(-1, rows).int()[offset:], some, rows, padding_idx=pad))
        table = torch.randn(rows, 37, device="cuda", generator=gen(1))
        out = embedding_lookup(ids.clamp(-1, rows).int()[offset:], table)
        assert torch.equal(out.nan_to_num(5.0), embedding_lookup(ids[offset:], table).nan_to_num(5.0))


@pytest.mark.parametrize("rows,dim,dtype", [(300_001, 127, torch.float16), (420_000, 47, torch.float32), (300_000, 256, torch.float16),
                                            (64_000_001, 1, torch.bfloat16), (90_001, 601, torch.float32), (1_500_000, 32, torch.float32)])
def test_gradient_of_few_tokens_in_a_large_table(rows, dim, dtype):
    """Zeros in the same launch and in one of their own."""
    from sparc_amd.embedding import embedding_grad
    for n in (0, 5, 3000):
        ids = make_ids("zipf", n, rows, 90 + n)
        g = torch.randn(n, dim, device="cuda", generator=gen(91)).to(dtype)
        torch.full((rows, dim), 3.0, dtype=dtype, device="cuda")          # what a new allocation may hold
        check_grad(embedding_grad(ids, g, rows), ids, g, rows)


@pytest.mark.parametrize("pattern", ["one", "zipf", "uniform", "lengths"])
@pytest.mark.parametrize("n,rows,dim,dtype", [(30_000, 3, 1, torch.float32), (30_000, 3, 3, torch.float16), (40_001, 5, 70, torch.float32),
                                              (262_147, 3, 47, torch.float32), (20_000, 2, 515, torch.bfloat16), (9_000, 1, 1030, torch.float16),
                                              (70_000, 120, 8, torch.bfloat16), (300_000, 30, 16, torch.float32)])
def test_gradient_of_rows_that_many_workgroups_share(pattern, n, rows, dim, dtype):
    """One piece per worker at a long row's ends, one per workgroup inside it; few long rows and many."""
    from sparc_amd.embedding import embedding_grad
    ids = make_ids(pattern, n, rows, n + dim)
    if pattern == "lengths":
        ids = torch.cat([ids % rows, torch.arange(n, device="cuda") * rows // n])
    g = torch.randn(ids.numel(), dim, device="cuda", generator=gen(n + rows)).to(dtype)
    got = embedding_grad(ids, g, rows, scale=-1.5)
    check_grad(got, ids, g, rows, -1.5)
    assert torch.equal(got, embedding_grad(ids, g, rows, scale=-1.5))


@pytest.mark.parametrize("dim,dtype", [(8192, torch.float32), (8193, torch.float32), (16384, torch.float16), (16385, torch.bfloat16), (1 << 20, torch.float16)])
def test_gradient_of_very_wide_rows(dim, dtype):
    from sparc_amd.embedding import embedding_grad, embedding_lookup
    for pattern, n, rows in (("zipf", 37, 9), ("one", 90, 4), ("uniform", 1, 3)):
        if n * dim > 1 << 23:
            n = 5
        ids = make_ids(pattern, n, rows, dim)
        g = torch.randn(n, dim, device="cuda", generator=gen(dim)).to(dtype)
        check_grad(embedding_grad(ids, g, rows, scale=3.0), ids, g, rows, 3.0)
        assert torch.equal(embedding_lookup(ids, g[:min(n, rows)]).isnan().any(1), ids >= min(n, rows))
