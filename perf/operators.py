"""Operators of typed layers and of the training step's tail, as they are measured.

Four operators that a training or serving program over rows of several kinds (node types,
experts, partitions with weights of their own) calls next to each other:

``group``   rows ordered by the kind each row has, on the GPU: ``order`` (a stable counting sort;
            rows of no kind, id -1, come last) and ``ptr`` (where each kind's rows begin).
``linear``  ``y[i] = x[i] @ W[kind(i)]^T + b[kind(i)]``, kinds of ragged sizes, rows of no kind
            give zeros; ``train``: the same with the gradients of x, W and b.
``clip``    the global norm over many tensors and their scaling in place by
            ``min(1, max_norm / (norm + 1e-6))``.
``adam``    an Adam step whose gradients are clipped by their global norm as they are read.

``own = False`` computes them in plain torch, ``own = True`` calls the package.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
LR, BETA1, BETA2, EPS = 1e-3, 0.9, 0.999, 1e-8


def _package():
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "incagg-gnn_amd")
    if here not in sys.path:
        sys.path.insert(0, here)
    import torch_geometric_autoscale
    from torch_geometric_autoscale import nn, ops, optim
    return torch_geometric_autoscale, ops, nn, optim


# ------------------------------------------------------------------ cases
def listed():
    return [
        # the gradients of a 3-layer GCN (128 -> 256 -> 256 -> 40, batch norm) after its backward
        # pass: ten tensors, under 0.5 MB -- launches and latency count
        dict(name="clip-gcn-step", op="clip", shapes="gcn", dtype="float32", norm="2",
             max_norm=0.1),
        # the gradients of a large model with 16-bit weights and float32 norms and biases
        dict(name="clip-many-mixed", op="clip", shapes="many", tensors=300, elements=200_000_000,
             dtype="mixed", norm="2", max_norm=0.1),
        # the optimizer step of the 8 x 256 GCNII (100 features, 47 classes), two groups
        dict(name="adam-gcn2-step", op="adam", shapes="gcn2", max_norm=0.5),
        # the optimizer step of a model with a wide embedding and many blocks
        dict(name="adam-many", op="adam", shapes="many", tensors=120, elements=64_000_003,
             max_norm=0.5),
        # one request's rows sorted by kind
        dict(name="group-request", op="group", rows=517, groups=64, none=0.0),
        # every node of a 2.4 M node graph by its type
        dict(name="group-graph", op="group", rows=2_449_029, groups=16, none=0.02),
        # a few rows of a request, each with a kind of its own: the weights are read once
        dict(name="linear-request", op="linear", rows=12, groups=64, k=1024, n=1024,
             dtype="bfloat16", bias=True, form="ids", none=0.0),
        # the input layer of a partition batch with its halo rows: 128 k x 100 -> 256
        dict(name="linear-batch", op="linear", rows=128_064, groups=4, k=100, n=256,
             dtype="float32", bias=True, form="order", none=0.01),
        # all rows of a large batch through 16 experts, rows sorted beforehand
        dict(name="linear-experts", op="linear", rows=131_072, groups=16, k=1024, n=2048,
             dtype="bfloat16", bias=False, form="ptr", none=0.0),
        # a training step of a hidden layer over one partition batch
        dict(name="train-hidden", op="train", rows=16_326, groups=5, k=256, n=256,
             dtype="float32", bias=True, form="order", none=0.0),
        # a classifier with odd widths, some kinds without a row
        dict(name="train-odd", op="train", rows=23_297, groups=37, k=602, n=41,
             dtype="float16", bias=True, form="order", none=0.05),
        # a training step of an expert layer
        dict(name="train-experts", op="train", rows=49_152, groups=32, k=1024, n=1024,
             dtype="bfloat16", bias=True, form="ptr", none=0.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["clip", "adam", "group", "linear", "linear", "train", "train"])
    if op == "clip":
        dtype = rng.choice(["float32", "bfloat16", "float16", "mixed"])
        return dict(op=op, shapes="many", tensors=_log(rng, 1, 400),
                    elements=_log(rng, 1_000, 150_000_000), dtype=dtype,
                    norm=rng.choice(["2", "2", "1", "inf"]), max_norm=100.0 if dtype == "float16" else 0.1)
    if op == "adam":
        return dict(op=op, shapes="many", tensors=_log(rng, 1, 200),
                    elements=_log(rng, 1_000, 60_000_000), max_norm=rng.choice([0.25, 0.5, 1.0]))
    if op == "group":
        return dict(op=op, rows=_log(rng, 1, 2_400_000), groups=_log(rng, 1, 1024),
                    none=rng.choice([0.0, 0.0, 0.05]))
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    case = dict(op=op, rows=_log(rng, 1, 131_072 if op == "linear" else 49_152),
                groups=_log(rng, 1, 128), k=_log(rng, 8, 2048), n=_log(rng, 8, 2048), dtype=dtype,
                bias=rng.random() < 0.5, form=rng.choice(["order", "ptr", "ids"]),
                none=rng.choice([0.0, 0.0, 0.05]))
    if rng.random() < 0.5:        # half of the layers have widths in whole vectors
        case["k"], case["n"] = (max(8, v // 32 * 32) for v in (case["k"], case["n"]))
    budget = 2.0e11 if op == "linear" else 4.0e10      # rows * k * n
    if dtype == "float32":
        budget /= 4
    case["rows"] = max(1, min(case["rows"], int(budget / (case["k"] * case["n"]))))
    # (at most 2 GB of weights in float32)
    case["groups"] = max(1, min(case["groups"], int(5.0e8 / (case["k"] * case["n"]))))
    return case


# ------------------------------------------------------------------ inputs
def _tensor_shapes(case):
    if case["shapes"] == "gcn":
        return [(256, 128), (256,), (256,), (256,), (256, 256), (256,), (256,), (256,), (40, 256),
                (40,)]
    if case["shapes"] == "gcn2":
        return [(256, 256)] * 16 + [(256, 100), (256,), (47, 256), (47,)]
    # every third tensor is a short vector, the others share the elements unevenly
    count = case["tensors"]
    big = [i for i in range(count) if i % 3 != 2] or [0]
    weights = {i: 1.0 + (i * 7 % 11) for i in big}
    total = sum(weights.values())
    out = []
    for i in range(count):
        if i in weights:
            out.append((max(1, int(case["elements"] * weights[i] / total)),))
        else:
            out.append((257 + 13 * (i % 17),))
    return out


def _tensor_types(case, shapes):
    if case["op"] == "adam":
        return [torch.float32] * len(shapes)
    if case["dtype"] == "mixed":
        return [torch.float32 if i % 3 == 2 else torch.bfloat16 for i in range(len(shapes))]
    return [DTYPES[case["dtype"]]] * len(shapes)


def _kinds(case, gen):
    """A kind for every row: ragged shares, every eighth kind without a row."""
    groups, rows = case["groups"], case["rows"]
    share = -torch.log(torch.rand(groups, device="cuda", generator=gen).clamp_(min=1e-6))
    if groups > 8:
        share[::8] = 0
    ids = torch.multinomial(share.cpu(), rows, replacement=True,
                            generator=torch.Generator().manual_seed(int(gen.initial_seed())))
    ids = ids.to("cuda")
    if case["none"]:
        ids[torch.rand(rows, device="cuda", generator=gen) < case["none"]] = -1
    return ids


def _plain_group(ids, groups):
    key = torch.where(ids < 0, torch.full_like(ids, groups), ids)
    order = torch.sort(key, stable=True).indices
    count = torch.bincount(key, minlength=groups + 1)[:groups]
    ptr = torch.zeros(groups + 1, dtype=torch.int64, device=ids.device)
    ptr[1:] = torch.cumsum(count, 0)
    return order, ptr


def _flat(shapes, gen, scale, dtype=torch.float32, square=False):
    """Tensors of these shapes as views of one buffer, each of them starting at a multiple of 64
    elements (zeros between them), and the buffer."""
    starts, total = [], 0
    for s in shapes:
        starts.append(total)
        total += -(-math.prod(s) // 64) * 64
    buffer = torch.zeros(total, dtype=dtype, device="cuda")
    views = [buffer[at:at + math.prod(s)].view(s) for at, s in zip(starts, shapes)]
    for v in views:
        r = torch.randn(v.shape, device="cuda", generator=gen)
        v.copy_((r.square_() if square else r) * scale)
    return views, buffer


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    state = {"case": case}
    if case["op"] == "clip":
        # gradients live side by side, as data-parallel training keeps them
        shapes = _tensor_shapes(case)
        types = _tensor_types(case, shapes)
        scale = 30.0 if case["dtype"] == "float16" else 0.03      # (float16: a scaled loss)
        state["params"], state["flat"] = [], []
        for t in sorted(set(types), key=str):
            views, buffer = _flat([s for s, u in zip(shapes, types) if u == t], gen, scale, t)
            state["flat"].append(buffer)
            for v in views:
                state["params"].append(torch.nn.Parameter(torch.empty_like(v)))
                state["params"][-1].grad = v
        return state
    if case["op"] == "adam":
        shapes = _tensor_shapes(case)
        count = len(shapes)
        k = (2 * count + 2) // 3                   # two groups: decayed, not decayed
        params, state["p"] = _flat(shapes, gen, 0.1)
        grads, state["g"] = _flat(shapes, gen, 0.03)
        m, state["m"] = _flat(shapes, gen, 1e-3)
        v, state["v"] = _flat(shapes, gen, 1e-5, square=True)
        state["steps"] = torch.full((count,), 41.0, device="cuda")
        state["decayed"] = sum(-(-math.prod(s) // 64) * 64 for s in shapes[:k])
        if own:
            _, _, _, optim = _package()
            params = [p.requires_grad_() for p in params]
            groups = [dict(params=params[:k], weight_decay=5e-4),
                      dict(params=params[k:], weight_decay=0.0)]
            opt = optim.Adam([g for g in groups if g["params"]], lr=LR, betas=(BETA1, BETA2),
                             eps=EPS)
            for i, p in enumerate(params):
                p.grad = grads[i]
                opt.state[p].update(exp_avg=m[i], exp_avg_sq=v[i], step=state["steps"][i])
            state["opt"] = opt
        return state
    ids = _kinds(case, gen)
    if case["op"] == "group":
        state["ids"] = ids
        return state
    groups, k, n, t = case["groups"], case["k"], case["n"], DTYPES[case["dtype"]]
    order, ptr = _plain_group(ids, groups)
    if case["form"] == "ptr":           # the rows lie sorted already; those of no kind last
        ids, order = ids[order], torch.arange(case["rows"], device="cuda")
    state["x"] = randn(case["rows"], k).to(t)
    state["w"] = (randn(groups, n, k) / math.sqrt(k)).to(t)
    state["b"] = (randn(groups, n) * 0.1).to(t) if case["bias"] else None
    if case["op"] == "train":
        state["dy"] = (randn(case["rows"], n) * 0.05).to(t)
        for key in ("x", "w", "b"):
            if state[key] is not None:
                state[key].requires_grad_()
    state["ids"] = ids
    if case["form"] != "ids":           # a batch's kinds are known when the batch is built
        state["order"], state["bounds"] = order, ptr.tolist()
        if own:
            _, ops, _, _ = _package()
            state["groups"] = (ops.groups_from_ptr(ptr, case["rows"]) if case["form"] == "ptr"
                               else ops.group_rows(ids, groups))
    return state


# ------------------------------------------------------------------ one pass
def _plain_clip(state):
    case = state["case"]
    flat = state["flat"]
    if case["norm"] == "inf":
        total = torch.stack([g.float().abs().max() for g in flat]).max()
    elif case["norm"] == "1":
        total = torch.stack([g.float().abs().sum(dtype=torch.float64) for g in flat]).sum().float()
    else:
        total = torch.stack([g.float().square().sum(dtype=torch.float64)
                             for g in flat]).sum().sqrt().float()
    scale = torch.clamp(case["max_norm"] / (total + 1e-6), max=1.0)
    for g in flat:
        if g.dtype == torch.float32:
            g.mul_(scale)
        else:
            g.copy_(g.float() * scale)
    return [total] + flat


def _plain_adam(state):
    """(every tensor has made the same number of steps)"""
    p, g, m, v, steps = (state[key] for key in ("p", "g", "m", "v", "steps"))
    total = g.square().sum(dtype=torch.float64).sqrt().float()
    scale = torch.clamp(state["case"]["max_norm"] / (total + 1e-6), max=1.0)
    steps += 1
    c1 = (1.0 - BETA1 ** steps[0].double()).float()
    c2 = (1.0 - BETA2 ** steps[0].double()).sqrt().float()
    g = g * scale
    g[:state["decayed"]] += 5e-4 * p[:state["decayed"]]
    m.add_(g - m, alpha=1.0 - BETA1)
    v.mul_(BETA2).add_(g.square_(), alpha=1.0 - BETA2)
    p.sub_((LR / c1) * m / (v.sqrt() / c2 + EPS))
    return [total, p, m, v, steps]


def _plain_few(state):
    """A few rows: every row with a weight matrix of its own, all of them in one batched product."""
    ids, w, b = state["ids"], state["w"], state["b"]
    there = ids >= 0
    at = torch.where(there, ids, torch.zeros_like(ids))
    y = torch.bmm(w[at].float(), state["x"].float().unsqueeze(2)).squeeze(2)
    if b is not None:
        y = y + b[at].float()
    return [torch.where(there.unsqueeze(1), y, torch.zeros_like(y)).to(w.dtype)]


@torch.no_grad()
def _plain_layer(state):
    case = state["case"]
    train = case["op"] == "train"
    x, w, b = state["x"], state["w"], state["b"]
    if not train and case["rows"] <= 64:
        return _plain_few(state)
    if case["form"] == "ids":
        order, ptr = _plain_group(state["ids"], case["groups"])
        bounds = ptr.tolist()
    else:
        order, bounds = state["order"], state["bounds"]
    t = x.dtype
    y = torch.zeros(case["rows"], case["n"], device="cuda")
    if train:
        dy = state["dy"]
        dx = torch.zeros(case["rows"], case["k"], device="cuda")
        dw = torch.zeros(w.shape, device="cuda")
        db = torch.zeros(case["groups"], case["n"], device="cuda")
    for g in range(case["groups"]):
        lo, hi = bounds[g], bounds[g + 1]
        if lo == hi:
            continue
        rows = slice(lo, hi) if case["form"] == "ptr" else order[lo:hi]
        xg, wg = x[rows].float(), w[g].float()
        yg = xg @ wg.t()
        if b is not None:
            yg = yg + b[g].float()
        y[rows] = yg
        if train:
            dyg = dy[rows].float()
            dx[rows] = dyg @ wg
            torch.mm(dyg.t(), xg, out=dw[g])
            if b is not None:
                torch.sum(dyg, 0, out=db[g])
    if not train:
        return [y.to(t)]
    out = [y.to(t), dx.to(t), dw.to(t)]
    return out + [db.to(t)] if b is not None else out


def run(state):
    case = state["case"]
    if not own:
        if case["op"] == "clip":
            return _plain_clip(state)
        if case["op"] == "adam":
            return _plain_adam(state)
        if case["op"] == "group":
            order, ptr = _plain_group(state["ids"], case["groups"])
            return [order.int(), ptr.int()]
        return _plain_layer(state)
    _, ops, nn, optim = _package()
    if case["op"] == "clip":
        total = optim.clip_grad_norm_(state["params"], case["max_norm"],
                                      norm_type=float(case["norm"]))
        return [total] + state["flat"]
    if case["op"] == "adam":
        total = state["opt"].step(max_norm=case["max_norm"])
        return [total] + [state[key] for key in ("p", "m", "v", "steps")]
    if case["op"] == "group":
        groups = ops.group_rows(state["ids"], case["groups"])
        return [groups.order, groups.ptr]
    groups = state["groups"] if case["form"] != "ids" else ops.group_rows(state["ids"],
                                                                          case["groups"])
    x, w, b = state["x"], state["w"], state["b"]
    y = nn.grouped_linear(x, w, b, groups)
    if case["op"] == "linear":
        return [y]
    grads = torch.autograd.grad(y, [x, w] if b is None else [x, w, b], state["dy"])
    return [y.detach()] + list(grads)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["op"] in ("clip", "adam"):
        shapes = _tensor_shapes(case)
        sizes = [math.prod(s) for s in shapes]
        if case["op"] == "adam":       # p, g, m, v in; p, m, v out
            return {"bytes": 28 * sum(sizes), "flops": 18 * sum(sizes)}
        types = _tensor_types(case, shapes)
        stored = sum(n * t.itemsize for n, t in zip(sizes, types))
        return {"bytes": 2 * stored, "flops": 3 * sum(sizes)}
    rows, groups = case["rows"], case["groups"]
    if case["op"] == "group":
        return {"bytes": 12 * rows + 4 * groups, "flops": rows}
    k, n = case["k"], case["n"]
    size = DTYPES[case["dtype"]].itemsize
    used = min(rows, groups)
    product = 2 * rows * k * n
    if case["op"] == "linear":
        return {"bytes": size * (rows * (k + n) + used * k * n), "flops": product}
    return {"bytes": size * (2 * rows * (k + n) + used * k * n + groups * k * n),
            "flops": 3 * product}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    if case["op"] == "group":
        import numpy as np
        ids = prepare(case, seed)["ids"].cpu().numpy()
        kind = np.where(ids < 0, case["groups"], ids)
        ptr = np.searchsorted(np.sort(kind), np.arange(case["groups"] + 1))
        return [torch.from_numpy(np.argsort(kind, kind="stable").astype("int32")),
                torch.from_numpy(ptr.astype("int32"))]
    state = prepare(case, seed)
    if case["op"] == "clip":
        flat = [g.double() for g in state["flat"]]
        if case["norm"] == "2":
            total = torch.sqrt(sum(torch.dot(f, f) for f in flat))
        elif case["norm"] == "1":
            total = sum(torch.sum(torch.abs(f)) for f in flat)
        else:
            total = max(torch.max(torch.abs(f)) for f in flat)
        factor = min(1.0, case["max_norm"] / (float(total) + 1e-6))
        return [total] + [f * factor for f in flat]
    if case["op"] == "adam":
        p, g, m, v = (state[key].detach().double() for key in ("p", "g", "m", "v"))
        total = torch.sqrt(torch.dot(g, g))
        decay = torch.zeros_like(p)
        decay[:state["decayed"]] = 5e-4
        d = g * min(1.0, case["max_norm"] / (float(total) + 1e-6)) + decay * p
        m = BETA1 * m + (1 - BETA1) * d
        v = BETA2 * v + (1 - BETA2) * d ** 2
        step = state["steps"].double() + 1
        m_hat, v_hat = m / (1 - BETA1 ** float(step[0])), v / (1 - BETA2 ** float(step[0]))
        return [total, p - LR * m_hat / (torch.sqrt(v_hat) + EPS), m, v, step]
    ids, groups = state["ids"], case["groups"]
    x, w = state["x"].detach().double(), state["w"].detach()
    y = x.new_zeros(case["rows"], case["n"])
    train = case["op"] == "train"
    if train:
        dy = state["dy"].double()
        dx, dw = torch.zeros_like(x), torch.zeros(w.shape, dtype=torch.float64, device="cuda")
        db = x.new_zeros(groups, case["n"])
    for g in range(groups):
        mine = torch.nonzero(ids == g).view(-1)
        if mine.numel() == 0:
            continue
        wg, xg = w[g].double(), x.index_select(0, mine)
        bias = 0.0 if state["b"] is None else state["b"][g].detach().double()
        y.index_copy_(0, mine, torch.mm(xg, wg.t().contiguous()) + bias)
        if train:
            d = dy.index_select(0, mine)
            dx.index_copy_(0, mine, torch.mm(d, wg))
            dw[g] = torch.mm(d.t().contiguous(), xg)
            db[g] = torch.sum(d, 0)
    if not train:
        return [y]
    return [y, dx, dw, db] if state["b"] is not None else [y, dx, dw]
