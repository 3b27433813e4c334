"""The table lookup, its gradient, the global gradient norm with clipping and the clipped Adam step: the cases on which
they are timed, their plain forms and their values in 64 bits.  `own` selects the framework's operators."""
import math
import random

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16,
          "int32": torch.int32, "int64": torch.int64}
BETAS, EPS, LR, WEIGHT_DECAY, STEP = (0.9, 0.999), 1e-8, 1e-3, 0.01, 100


def listed():
    lookup = {"op": "lookup", "ids": "uniform", "id_dtype": "int64", "scale": 1.0}
    grad = {"op": "lookup_grad", "ids": "uniform", "id_dtype": "int64", "scale": 1.0, "padded": False}
    clip = {"op": "clip", "layout": "mlp", "din": 10, "rows": 0, "dim": 0, "dtype": "float32", "max_norm": 1.0}
    return [
        # one node's row out of the Cora graph's table: what embedding a single node costs
        dict(lookup, name="lookup-one-node", n=1, rows=2708, dim=64, dtype="float32"),
        # one Amazon2M-shape cluster batch, as many columns as that graph's embedding has (rows of 188 bytes)
        dict(lookup, name="lookup-amazon-batch", n=24490, rows=2449029, dim=47, dtype="float32"),
        # token sequences over a vocabulary, frequent tokens first, rows scaled by the root of their width
        dict(lookup, name="lookup-tokens-bf16", n=262147, rows=50021, dim=1024, dtype="bfloat16", ids="zipf",
             id_dtype="int32", scale=32.0),
        # a step on the shipped Cora graph: every training node once or twice
        dict(grad, name="grad-cora", n=2437, rows=2708, dim=64, dtype="float32"),
        # odd width and 16-bit gradients on the PubMed graph's nodes
        dict(grad, name="grad-pubmed-fp16", n=6600, rows=19717, dim=47, dtype="float16", id_dtype="int32", scale=0.5),
        # both batches of an Amazon2M-shape step: few of the table's rows are met, all have to be written
        dict(grad, name="grad-amazon-step", n=48979, rows=2449029, dim=64, dtype="float32"),
        # token sequences with padding: the most frequent token has thousands of places, most have a few
        dict(grad, name="grad-tokens-bf16", n=262147, rows=50021, dim=512, dtype="bfloat16", ids="zipf", id_dtype="int32",
             scale=22.627417, padded=True),
        # the gradients of the benchmark's MLP
        dict(clip, name="clip-mlp"),
        # many tensors of uneven sizes in 16 bits
        dict(clip, name="clip-uneven-bf16", layout="uneven", count=48, total=9000001, dtype="bfloat16", max_norm=0.5),
        # the MLP and a table with a row for every node of the Amazon2M shape
        dict(clip, name="clip-amazon-table", din=64, rows=2449029, dim=64),
        # the optimiser step of the benchmark's MLP
        dict(clip, name="adam-mlp", op="adam"),
        # the MLP and a table with a row for every node of the Reddit shape
        dict(clip, name="adam-reddit-table", op="adam", din=128, rows=232965, dim=128),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("lookup", "lookup_grad", "lookup_grad", "clip", "adam"))
    if op in ("lookup", "lookup_grad"):
        dtype = rng.choice(("float32", "bfloat16", "float16"))
        size = 4 if dtype == "float32" else 2
        case = {"op": op, "dim": _log(rng, 1, 1024), "dtype": dtype, "id_dtype": rng.choice(("int32", "int64")),
                "ids": rng.choice(("uniform", "uniform", "zipf", "zipf", "one")), "scale": rng.choice((1.0, 0.5, 11.3137085))}
        most = 268435456 // (case["dim"] * size)     # elements: a drawn case stays below the largest listed ones
        case["rows"] = min(_log(rng, 2, 2449029), most)
        case["n"] = min(_log(rng, 1, 262147), most)
        if op == "lookup_grad":
            case["padded"] = rng.random() < 0.3
        return case
    case = {"op": op, "dtype": "float32", "layout": "uneven", "count": _log(rng, 1, 60 if op == "clip" else 20)}
    if op == "clip":
        case["dtype"] = rng.choice(("float32", "bfloat16", "float16"))
    case["total"] = max(case["count"], _log(rng, 64, 60000000 if op == "clip" else 25000000))
    # below, around and far above the norm that such gradients have
    case["max_norm"] = rng.choice((0.1, 0.5, 1000.0)) * math.sqrt(case["total"])
    return case


def _shapes(case):
    """The parameter tensors of a training program."""
    if case["layout"] == "mlp":
        sizes = [case["din"], 1024, 1024, 512, 47]       # the benchmark's MLP
        shapes = [s for a, b in zip(sizes, sizes[1:]) for s in ((b, a), (b,))]
        return ([(case["rows"], case["dim"])] if case["rows"] else []) + shapes
    rng = random.Random("%(count)d of %(total)d" % case)
    parts = [rng.random() ** 4 + 1e-9 for _ in range(case["count"])]
    return [(max(1, int(case["total"] * p / sum(parts))),) for p in parts]


def _elements(case):
    return sum(math.prod(s) for s in _shapes(case))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    state = dict(case)
    if case["op"] in ("lookup", "lookup_grad"):
        n, rows, dim = case["n"], case["rows"], case["dim"]
        if case["ids"] == "one":        # one token everywhere
            ids = torch.randint(rows, (1,), generator=gen, device="cuda").expand(n)
        elif case["ids"] == "zipf":     # token t with a chance of about 1 / (t + 1)
            u = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)
            ids = (torch.exp(u * math.log(rows + 1.0)) - 1.0).long().clamp_(0, rows - 1)
        else:
            ids = torch.randint(rows, (n,), generator=gen, device="cuda")
        state["padding_idx"] = None
        if case.get("padded"):          # about an eighth of the places hold no token
            state["padding_idx"] = 0
            ids = ids * (torch.rand(n, generator=gen, device="cuda") > 0.125)
        state["ids_"] = ids.to(DTYPES[case["id_dtype"]]).contiguous()
        values = rows if case["op"] == "lookup" else n
        state["values"] = torch.randn(values, dim, generator=gen, device="cuda", dtype=torch.float32).to(dtype)
        return state
    tensors = []
    for i, shape in enumerate(_shapes(case)):       # gradients of different layers differ in size
        tensors.append((torch.randn(shape, generator=gen, device="cuda") * 10.0 ** -(i % 4)).to(dtype))
    if case["op"] == "clip":
        state["params"] = [torch.nn.Parameter(torch.empty_like(g)) for g in tensors]
        for p, g in zip(state["params"], tensors):
            p.grad = g
        return state
    state["grads"] = tensors
    state["params"] = [torch.randn(g.shape, generator=gen, device="cuda") * 0.1 for g in tensors]
    state["m"] = [torch.randn(g.shape, generator=gen, device="cuda") * 0.01 for g in tensors]
    state["v"] = [torch.rand(g.shape, generator=gen, device="cuda") * 0.001 + 1e-6 for g in tensors]
    return state


def _norm_and_coef(grads, max_norm):
    norm = torch.stack([g.float().square().sum() for g in grads]).sum().sqrt()
    return norm, (max_norm / (norm + 1e-6)).clamp(max=1.0)


def _adam(p, g, m, v, coef):
    g = g * coef + WEIGHT_DECAY * p
    m.add_((1.0 - BETAS[0]) * (g - m))
    v.mul_(BETAS[1]).add_((1.0 - BETAS[1]) * g * g)
    denom = v.sqrt() / math.sqrt(1.0 - BETAS[1] ** STEP) + EPS
    p.sub_(LR / (1.0 - BETAS[0] ** STEP) * m / denom)


def run(state):
    op = state["op"]
    if op == "lookup":
        ids, table = state["ids_"], state["values"]
        if own:
            from sparc_amd.embedding import embedding_lookup
            return embedding_lookup(ids, table, scale=state["scale"])
        return (table[ids.long()].float() * state["scale"]).to(table.dtype)
    if op == "lookup_grad":
        ids, g = state["ids_"], state["values"]
        if own:
            from sparc_amd.embedding import embedding_grad
            return embedding_grad(ids, g, state["rows"], scale=state["scale"], padding_idx=state["padding_idx"])
        rows = torch.arange(state["rows"], device=g.device)
        if state["ids"] == "uniform" and state["n"] < 64 * state["rows"]:
            out = torch.zeros(state["rows"], state["dim"], device=g.device).index_add_(0, ids.long(), g.float())
        else:
            # a row that collects thousands of places is a long sum: running sums of the sorted places in 64 bits
            by_row, order = ids.long().sort()
            sums = torch.nn.functional.pad(g[order].t().contiguous().double().cumsum(1), (1, 0))
            ends, starts = torch.searchsorted(by_row, rows, right=True), torch.searchsorted(by_row, rows)
            out = (sums[:, ends] - sums[:, starts]).t().contiguous()
        if state["padding_idx"] is not None:
            out[state["padding_idx"]] = 0
        return (out * state["scale"]).to(g.dtype)
    if op == "clip":
        params = state["params"]
        if own:
            from sparc_amd.optim import clip_grad_norm_
            return [clip_grad_norm_(params, state["max_norm"])] + [p.grad for p in params]
        norm, coef = _norm_and_coef([p.grad for p in params], state["max_norm"])
        return [norm] + [p.grad.copy_(p.grad.float() * coef) for p in params]
    params, grads, m, v = state["params"], state["grads"], state["m"], state["v"]
    if own:
        from sparc_amd.optim import adam_step_
        norm = adam_step_(params, grads, m, v, STEP, lr=LR, betas=BETAS, eps=EPS, weight_decay=WEIGHT_DECAY,
                          max_grad_norm=state["max_norm"])
    else:
        norm, coef = _norm_and_coef(grads, state["max_norm"])
        [_adam(*of_one, coef) for of_one in zip(params, grads, m, v)]
    return [norm] + params + m + v


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"] in ("lookup", "lookup_grad"):
        ids = case["n"] * (4 if case["id_dtype"] == "int32" else 8)
        read = min(case["n"], case["rows"]) if case["op"] == "lookup" else case["n"]
        written = case["n"] if case["op"] == "lookup" else case["rows"]
        return {"bytes": ids + (read + written) * case["dim"] * size, "flops": case["n"] * case["dim"]}
    n = _elements(case)
    if case["op"] == "clip":
        return {"bytes": 2 * n * size + 4, "flops": 3 * n}
    return {"bytes": 28 * n + 4, "flops": 18 * n}


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "lookup":
        return state["values"].double().index_select(0, state["ids_"].long()).mul_(case["scale"])
    if case["op"] == "lookup_grad":
        ids, g = state["ids_"].long(), state["values"].double()
        if state["padding_idx"] is not None:
            kept = ids != state["padding_idx"]
            ids, g = ids[kept], g[kept]
        out = torch.zeros(case["rows"], case["dim"], dtype=torch.float64, device=g.device)
        return out.index_put_((ids,), g * case["scale"], accumulate=True)
    grads = [p.grad for p in state["params"]] if case["op"] == "clip" else state["grads"]
    norm = math.sqrt(sum(float(torch.linalg.vector_norm(g.double())) ** 2 for g in grads))
    coef = min(1.0, case["max_norm"] / (norm + 1e-6))
    total = torch.tensor(norm, dtype=torch.float64)
    if case["op"] == "clip":
        return [total] + [g.double() * coef for g in grads]
    p, m, v = [], [], []
    for p0, g, m0, v0 in zip(state["params"], grads, state["m"], state["v"]):
        g = g.double() * coef + WEIGHT_DECAY * p0.double()
        m.append(BETAS[0] * m0.double() + (1.0 - BETAS[0]) * g)
        v.append(BETAS[1] * v0.double() + (1.0 - BETAS[1]) * g.square())
        root = torch.sqrt(v[-1] / (1.0 - BETAS[1] ** STEP))
        p.append(p0.double() - LR * m[-1] / (1.0 - BETAS[0] ** STEP) / (root + EPS))
    return [total] + p + m + v
