"""The selection products of a language model, as they are measured: the embedding lookup and its
gradient, and the tokens sorted by expert and brought back.

Each case is one call (or the run of calls that belong together) of a program that trains or
serves such a model.  ``run`` computes it in a plain form with elementary torch operations, or,
where ``own`` is true, with this package's kernels; ``exact`` computes it in 64 bits.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
INDEX = {"i32": torch.int32, "i64": torch.int64}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}

# ------------------------------------------------------------------------------------------------
# cases.  kind:
#   embed   rows of the table for `n` tokens, scaled
#   grad    the table's gradient from the gradients of `n` looked-up rows: a new dense one
#           (beta 0), or added to the one that earlier micro-batches left (beta 1)
#   there   the plan of a batch (tokens sorted by expert) and its rows in that order
#   trip    the plan, the rows in that order, and the experts' results back with their weights
#   back    the plan (a program that recomputes its activations makes it again) and the gradients
#           of the way back and of the way there
# pad: elements between the rows of the inputs (a slice of a wider buffer).  drop: share of the
# entries that are masked (-1): positions another rank holds, or assignments over capacity.
# ------------------------------------------------------------------------------------------------


def _embed(name, n, vocab, dim, dtype, index="i64", draw="zipf", drop=0.0, pad=0):
    return dict(name=name, kind="embed", n=n, vocab=vocab, dim=dim, dtype=dtype, index=index,
                draw=draw, drop=drop, pad=pad)


def _grad(name, n, vocab, dim, dtype, out, beta, index="i64", draw="zipf", drop=0.0, pad=0):
    return dict(name=name, kind="grad", n=n, vocab=vocab, dim=dim, dtype=dtype, out=out,
                beta=beta, index=index, draw=draw, drop=drop, pad=pad)


def _route(name, kind, n, k, experts, dim, dtype, weight="fp32", index="i64", drop=0.0, pad=0):
    return dict(name=name, kind=kind, n=n, k=k, experts=experts, dim=dim, dtype=dtype,
                weight=weight, index=index, drop=drop, pad=pad)


def listed():
    return [
        # one decoding step of 64 sequences: latency counts
        _embed("embed step", 64, 32000, 4096, "bf16"),
        # the prompts of a serving batch, a large vocabulary
        _embed("embed prompts", 16384, 131072, 4096, "bf16"),
        # an odd width, some tokens held by another rank of a split vocabulary
        _embed("embed odd", 5003, 50257, 1001, "fp16", index="i32", drop=0.3, pad=3),
        # fine-tuning on a few hundred tokens, gradient added to a float32 one
        _grad("grad small", 256, 32000, 1024, "bf16", "fp32", 1.0),
        # a training micro-batch: a new dense gradient of a large table
        _grad("grad dense", 16384, 131072, 2048, "bf16", "bf16", 0.0),
        # micro-batch after micro-batch into a float32 gradient
        _grad("grad added", 32768, 32000, 4096, "bf16", "fp32", 1.0),
        # a padded batch of an odd width: one token holds a third of the positions
        _grad("grad odd", 6001, 50257, 771, "fp32", "fp32", 0.0, draw="padded", drop=0.1),
        # one decoding step of 64 sequences, 8 of 256 experts
        _route("there step", "there", 64, 8, 256, 4096, "bf16"),
        # the prompts of a serving batch, 8 of 128 experts
        _route("trip prompts", "trip", 8192, 8, 128, 4096, "bf16"),
        # few large experts, an odd width, some assignments over capacity
        _route("trip odd", "trip", 1537, 3, 11, 1005, "fp16", weight="fp16", index="i32",
               drop=0.1, pad=5),
        # a training micro-batch, 4 of 64 experts
        _route("back batch", "back", 16384, 4, 64, 2048, "bf16"),
        # float32 training of a small model, 2 of 8 experts
        _route("back small", "back", 1000, 2, 8, 520, "fp32", drop=0.05),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng):
    """A model's width: mostly multiples of 64, now and then of 8, or odd."""
    d = _spread(rng, 256, 4096)
    style = rng.random()
    return max(64, d // 64 * 64) if style < 0.6 else d // 8 * 8 if style < 0.8 else d | 1


def draw(rng):
    kind = rng.choice(["embed", "grad", "there", "trip", "back"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    index = rng.choice(["i32", "i64"])
    drop = rng.choice([0.0, 0.0, round(rng.uniform(0.01, 0.5), 3)])
    pad = rng.choice([0, 0, 8, rng.randrange(1, 16)])
    dim = _width(rng)
    if kind in ("embed", "grad"):
        n, vocab = _spread(rng, 1, 16384), _spread(rng, 1000, 131072)
        how = rng.choice(["zipf", "even", "padded"])
        if kind == "embed":
            case = _embed("", n, vocab, dim, dtype, index, how, drop, pad)
        else:
            while vocab * dim > 131072 * 2048:
                vocab //= 2
            out = rng.choice([dtype, "fp32"])
            case = _grad("", n, vocab, dim, dtype, out, rng.choice([0.0, 1.0]), index, how,
                         drop, pad)
    else:
        experts = _spread(rng, 4, 512)
        k = rng.randrange(1, min(8, experts) + 1)
        n = _spread(rng, 1, 16384)
        while n * k * dim * SIZE[dtype] > 1 << 29:
            n = max(1, n // 2)
        weight = rng.choice(["fp32", dtype])
        case = _route("", kind, n, k, experts, dim, dtype, weight, index, drop, pad)
    del case["name"]
    return case


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _matrix(g, rows, dim, dtype, pad=0, std=1.0):
    wide = torch.empty(rows, dim + pad, dtype=DTYPES[dtype], device="cuda")
    wide.normal_(0.0, std, generator=g)
    return wide[:, :dim]


def _tokens(g, case):
    n, vocab = case["n"], case["vocab"]
    u = torch.rand(n, dtype=torch.float64, device="cuda", generator=g)
    if case["draw"] == "even":
        rank = u * vocab
    else:  # the frequency of the r-th most frequent token falls as 1 / r
        rank = torch.exp(u * math.log(vocab + 1.0)) - 1.0
    tokens = torch.randperm(vocab, device="cuda", generator=g)[rank.long().clamp_(0, vocab - 1)]
    if case["draw"] == "padded":  # the tails of the sequences hold one token
        tokens[n - n // 3:] = vocab // 2
    tokens = _dropped(g, case, tokens)
    return tokens.to(INDEX[case["index"]])


def _dropped(g, case, ids):
    if case["drop"]:
        gone = torch.rand(ids.shape, device="cuda", generator=g) < case["drop"]
        ids = ids.masked_fill(gone, -1)
    return ids


def prepare(case, seed):
    g = _generator(seed)
    dim, dtype, pad = case["dim"], case["dtype"], case["pad"]
    state = {"case": case}
    if case["kind"] in ("embed", "grad"):
        state["tokens"] = _tokens(g, case)
        state["ignore"] = -1 if case["drop"] else None
        state["alpha"] = math.sqrt(dim)
        if case["kind"] == "embed":
            state["table"] = _matrix(g, case["vocab"], dim, dtype, pad, 0.02)
        else:
            state["grad"] = _matrix(g, case["n"], dim, dtype, pad)
            state["out"] = None
            if case["beta"]:
                state["out"] = _matrix(g, case["vocab"], dim, case["out"])
        return state
    n, k = case["n"], case["k"]
    # the router's scores: some experts are asked for more often than others
    score = torch.randn(n, case["experts"], device="cuda", generator=g)
    score += 0.5 * torch.randn(case["experts"], device="cuda", generator=g)
    top, experts = torch.topk(score, k, dim=1)
    state["experts"] = _dropped(g, case, experts).to(INDEX[case["index"]])
    weights = torch.softmax(top, dim=1)
    state["weights"] = weights.to(DTYPES[case["weight"]])
    if case["kind"] != "back":
        state["x"] = _matrix(g, n, dim, dtype, pad)
    if case["kind"] != "there":
        state["y"] = _matrix(g, n * k, dim, dtype, pad)
    if case["kind"] == "back":
        state["grad_out"] = _matrix(g, n, dim, dtype, pad)
        state["grad_rows"] = _matrix(g, n * k, dim, dtype, pad)
    return state


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    import flagsparse_b200 as fs

    case = s["case"]
    kind = case["kind"]
    if kind == "embed":
        return fs.flagsparse_embedding(s["tokens"], s["table"], alpha=s["alpha"],
                                       ignore_index=s["ignore"])
    if kind == "grad":
        return fs.flagsparse_embedding_grad(
            s["tokens"], s["grad"], case["vocab"], alpha=s["alpha"], beta=case["beta"],
            ignore_index=s["ignore"], out=s["out"], out_dtype=DTYPES[case["out"]])
    route = fs.prepare_token_route(s["experts"], case["experts"])
    plan = {"indptr": route.indptr, "slots": route.slots}
    if kind == "there":
        return {"rows": fs.flagsparse_token_dispatch(s["x"], route), **plan}
    if kind == "trip":
        rows = fs.flagsparse_token_dispatch(s["x"], route)
        out = fs.flagsparse_token_combine(s["y"], route, s["weights"])
        return {"rows": rows, "out": out, **plan}
    grad_y, grad_weights = fs.flagsparse_token_combine_grad(s["grad_out"], s["y"], route,
                                                            s["weights"])
    grad_x = fs.flagsparse_token_dispatch_grad(s["grad_rows"], route)
    return {"grad_y": grad_y, "grad_weights": grad_weights, "grad_x": grad_x, **plan}


def _run_plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "embed":
        return _plain_embed(s)
    if kind == "grad":
        return _plain_grad(s)
    slots, indptr, order, held = _plain_plan(s["experts"], case["experts"])
    plan = {"indptr": indptr, "slots": slots}
    n, k, dim = case["n"], case["k"], case["dim"]
    if kind != "back":
        # row i of the sorted rows is the row of the token that assignment order[i] belongs to;
        # the rows of masked assignments stand last and are zero
        rows = s["x"][order // k]
        rows = torch.where((torch.arange(n * k, device="cuda") < held)[:, None], rows, 0)
        if kind == "there":
            return {"rows": rows, **plan}
    live = slots >= 0
    place = torch.where(live, slots, 0).long()
    w = torch.where(live, s["weights"].float(), 0.0)
    if kind == "trip":
        picked = s["y"][place].float()
        out = (picked * w[:, :, None]).sum(dim=1).to(s["y"].dtype)
        return {"rows": rows, "out": out, **plan}
    picked = s["y"][place].float()
    g = s["grad_out"].float()
    grad_w = torch.where(live, (picked * g[:, None, :]).sum(dim=2), 0.0).to(s["weights"].dtype)
    at = order.new_empty(n * k)
    at[order] = torch.arange(n * k, device="cuda")  # where each assignment stands, masked or not
    grad_y = torch.empty(n * k, dim, dtype=s["y"].dtype, device="cuda")
    grad_y[at] = (g[:, None, :] * w[:, :, None]).to(grad_y.dtype).reshape(n * k, dim)
    back = torch.where(live[:, :, None], s["grad_rows"][place].float(), 0.0)
    grad_x = back.sum(dim=1).to(s["grad_rows"].dtype)
    return {"grad_y": grad_y, "grad_weights": grad_w, "grad_x": grad_x, **plan}


def _plain_embed(s):
    tokens = s["tokens"].long()
    if s["ignore"] is None:
        return (s["table"][tokens].float() * s["alpha"]).to(s["table"].dtype)
    live = tokens != s["ignore"]
    rows = s["table"][torch.where(live, tokens, 0)].float() * s["alpha"]
    return torch.where(live[:, None], rows, 0.0).to(s["table"].dtype)


def _plain_grad(s):
    case = s["case"]
    tokens, grad = s["tokens"].long(), s["grad"].float()
    if s["ignore"] is not None:
        live = tokens != s["ignore"]
        tokens, grad = torch.where(live, tokens, 0), torch.where(live[:, None], grad, 0.0)
    total = torch.zeros(case["vocab"], case["dim"], device="cuda")
    total.index_add_(0, tokens, grad)
    total *= s["alpha"]
    if not case["beta"]:
        return total.to(DTYPES[case["out"]])
    total += case["beta"] * s["out"].float()
    return s["out"].copy_(total)


def _plain_plan(experts, n_experts):
    """Where each assignment stands among the rows sorted by expert (-1: masked, nowhere), where
    each expert's rows begin, the assignment of each row, and the number of rows held."""
    flat = experts.reshape(-1).long()
    key = torch.where(flat < 0, n_experts, flat)
    ordered, order = torch.sort(key, stable=True)
    edges = torch.arange(n_experts + 1, device="cuda")
    indptr = torch.searchsorted(ordered, edges).int()
    at = torch.empty_like(order)
    at[order] = torch.arange(flat.numel(), device="cuda")
    slots = torch.where(flat < 0, -1, at).int().reshape(experts.shape)
    return slots, indptr, order, indptr[-1]


# ------------------------------------------------------------------------------------------------
# the definition in 64 bits: products with the matrix that selects
# ------------------------------------------------------------------------------------------------


def _selection(rows, cols, values, shape):
    at = torch.stack([rows, cols])
    return torch.sparse_coo_tensor(at, values, shape, check_invariants=False)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in ("embed", "grad"):
        n = case["n"]
        live = torch.nonzero(s["tokens"] >= 0).flatten()
        cols = s["tokens"].long()[live]
        alpha = torch.full((live.numel(),), s["alpha"], dtype=torch.float64, device="cuda")
        if kind == "embed":
            out = torch.zeros(n, case["dim"], dtype=torch.float64, device="cuda")
            out[live] = s["table"].index_select(0, cols).double() * s["alpha"]
            return out
        select = _selection(cols, live, alpha, (case["vocab"], n))
        total = torch.sparse.mm(select, s["grad"].double())
        if case["beta"]:
            total += case["beta"] * s["out"].double()
        return total
    n, k, experts = case["n"], case["k"], case["experts"]
    flat = s["experts"].reshape(-1).long()
    hit = (flat[:, None] == torch.arange(experts, device="cuda")[None, :]).long()
    count = hit.sum(dim=0)
    first = count.cumsum(0) - count
    place = torch.where(flat >= 0, ((hit.cumsum(0) - hit + first) * hit).sum(dim=1), -1)
    del hit
    live = torch.nonzero(flat >= 0).flatten()
    where, who = place[live], live // k
    indptr = torch.cat([first, count.sum().reshape(1)]).int()
    plan = {"indptr": indptr, "slots": place.int().reshape(n, k)}
    w = s["weights"].double().reshape(-1)[live]
    if kind != "back":
        rows = torch.zeros(n * k, case["dim"], dtype=torch.float64, device="cuda")
        rows[where] = s["x"].double().index_select(0, who)
        if kind == "there":
            return {"rows": rows, **plan}
        out = torch.sparse.mm(_selection(who, where, w, (n, n * k)), s["y"].double())
        return {"rows": rows, "out": out, **plan}
    g = s["grad_out"].double()
    grad_y = torch.sparse.mm(_selection(where, who, w, (n * k, n)), g)
    grad_w = torch.zeros(n * k, dtype=torch.float64, device="cuda")
    grad_w[live] = torch.linalg.vecdot(s["y"].double()[where], g[who])
    grad_x = torch.sparse.mm(_selection(who, where, torch.ones_like(w), (n, n * k)),
                             s["grad_rows"].double())
    return {"grad_y": grad_y, "grad_weights": grad_w.reshape(n, k), "grad_x": grad_x, **plan}


# ------------------------------------------------------------------------------------------------
# what one pass has to read, write and compute
# ------------------------------------------------------------------------------------------------


def _distinct(case):
    """The expected number of different rows that the tokens name."""
    vocab = case["vocab"]
    n = case["n"] * (1.0 - case["drop"])
    r = torch.arange(1, vocab + 1, dtype=torch.float64)
    if case["draw"] == "even":
        p = torch.full_like(r, 1.0 / vocab)
    else:
        p = torch.log1p(1.0 / r) / math.log(vocab + 1.0)
    if case["draw"] == "padded":
        n *= 2.0 / 3.0
    return max(1.0, float((1.0 - torch.pow(1.0 - p, n)).sum()))


def work(case):
    n, dim, size = case["n"], case["dim"], SIZE[case["dtype"]]
    ids = 4 if case["index"] == "i32" else 8
    if case["kind"] == "embed":
        rows = _distinct(case)
        return {"bytes": (rows + n) * dim * size + n * ids, "flops": n * dim}
    kept = n * (1.0 - case["drop"])
    if case["kind"] == "grad":
        out = SIZE[case["out"]]
        rows = 2 * _distinct(case) if case["beta"] else case["vocab"]
        return {"bytes": kept * dim * size + rows * dim * out + n * ids, "flops": kept * dim}
    k = case["k"]
    kept = n * k * (1.0 - case["drop"])
    token, row, live = n * dim * size, n * k * dim * size, kept * dim * size
    weights = n * k * SIZE[case["weight"]]
    plan = n * k * (ids + 4)
    if case["kind"] == "there":
        return {"bytes": token + row + plan, "flops": 0}
    if case["kind"] == "trip":
        return {"bytes": token + row + live + token + weights + plan, "flops": 2 * kept * dim}
    moved = token + live + row + live + token
    return {"bytes": moved + 2 * weights + plan, "flops": 4 * kept * dim}
