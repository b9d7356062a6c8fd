"""The training operators of tcc_b200 beside the aggregation, as measurable cases:

* ``lookup``       rows of a learned node-embedding table, scaled;
* ``lookup_grad``  the gradient of that table, summed by sorted index;
* ``norm``         group norm over channels-last node features with an activation
                   (forward alone, or forward and backward);
* ``clip``         the global gradient norm over a model's tensors, and clipping.

``run`` computes each in plain torch operations, or, where ``own`` is true,
through the framework.  Sizes are those of the framework's own graphs: 1,048,576
nodes at width 128, 232,965 nodes (602 features, hidden 256), 2,449,029 nodes
(100 features, hidden 256, 47 classes) and its 200-node mini-batches.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
SKEW = 2.5  # index = rows * u^SKEW: low ids are hubs, as in an R-MAT graph


def _lookup(rows, width, n, ids="skew", table="f32", out="f32", index="i64", pad=False, scale=1.0):
    return dict(op="lookup", rows=rows, width=width, n=n, ids=ids, table=table, out=out, index=index, pad=pad,
                scale=scale)


def _norm(samples, steps, groups, per_group, act, x="f32", params="f32", train=True):
    return dict(op="norm", samples=samples, steps=steps, groups=groups, per_group=per_group, act=act, x=x,
                params=params, train=train)


def _clip(rows, width, layers, hidden, kinds, max_norm=1.0):
    return dict(op="clip", rows=rows, width=width, layers=layers, hidden=hidden, kinds=kinds, max_norm=max_norm)


def listed():
    return [
        # one node's embedding, read for an online answer: latency alone
        dict(_lookup(16384, 128, 1, ids="distinct", table="bf16"), name="lookup_one_node"),
        # input rows of a sampled block (distinct nodes, padded to a fixed size with -1) at the raw feature width
        dict(_lookup(232965, 602, 65537, ids="distinct", pad=True), name="lookup_block"),
        # endpoints of positive and negative edges for link prediction: hubs repeat
        dict(_lookup(2449029, 100, 2000003, index="i32", scale=10.0), name="lookup_edges"),
        # a mini-batch of 200 seed nodes trains a small table
        dict(_lookup(16384, 100, 200, ids="distinct"), op="lookup_grad", name="grad_seeds"),
        # link prediction on a million nodes: power-law repeats, the whole dense gradient written
        dict(_lookup(1048576, 128, 1 << 20, index="i32", scale=11.3137085), op="lookup_grad", name="grad_edges"),
        # 47 edge or node types shared by all: every row of the table is a very long sum
        dict(_lookup(47, 256, 400003, ids="uniform", table="bf16", out="bf16", pad=True), op="lookup_grad",
             name="grad_types"),
        # one mini-batch of hidden rows at inference
        dict(_norm(128, 1, 8, 32, "relu", x="bf16", params="bf16", train=False), name="norm_serve"),
        # a batch of small graphs of odd size, a norm over each, training
        dict(_norm(64, 517, 10, 10, "gelu"), name="norm_batch"),
        # one whole graph normalised over all of its nodes, training
        dict(_norm(1, 232965, 32, 8, "silu", x="bf16"), name="norm_graph"),
        # the hidden layer of full-graph training: each node by itself (the activation follows with the dropout)
        dict(_norm(2449029, 1, 8, 32, "none"), name="norm_hidden"),
        # the two weight matrices of the 2-layer model and the affine parameters of its norm
        dict(_clip(0, 0, 1, 256, "f32"), name="clip_gcn"),
        # a node-embedding table's gradient and a deep model's many small tensors of mixed type
        dict(_clip(2449029, 100, 20, 251, "mixed"), name="clip_table"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["lookup", "lookup_grad", "norm", "clip"])
    if op in ("lookup", "lookup_grad"):
        width = rng.choice([47, 64, 100, 128, 256, 602, _log(rng, 8, 640)])
        rows = _log(rng, 40, 2449029)
        n = min(_log(rng, 1, 2000003), 200_000_000 // width)
        if rows * width > 250_000_000:
            rows = 250_000_000 // width
        ids = rng.choice(["skew", "uniform", "distinct"])
        if ids == "distinct":
            n = min(n, rows)
        table = rng.choice(["f32", "f32", "f16", "bf16"])
        return dict(_lookup(rows, width, n, ids=ids, table=table, out=rng.choice([table, "f32"]),
                            index=rng.choice(["i32", "i64"]), pad=rng.random() < 0.4,
                            scale=rng.choice([1.0, 0.5, round(math.sqrt(width), 4)])), op=op)
    if op == "norm":
        groups = rng.choice([1, 2, 4, 8, 16, 32, rng.randint(3, 12)])
        per_group = rng.choice([4, 8, 16, 32, rng.randint(2, 40)])
        channels = groups * per_group
        most = 400_000_000 // channels
        kind = rng.choice(["rows", "graph", "batch"])
        if kind == "rows":
            samples, steps = min(_log(rng, 1, 2449029), most), 1
            per_group = max(per_group, 8)
        elif kind == "graph":
            samples, steps = rng.randint(1, 8), _log(rng, 100, 232965)
            steps = min(steps, most // samples)
        else:
            samples, steps = _log(rng, 2, 512), _log(rng, 8, 2048)
        train = rng.random() < 0.7
        act = rng.choice(["none", "silu", "gelu"] if train else ["none", "relu", "silu", "gelu"])
        x = rng.choice(["f32", "f16", "bf16"])
        return _norm(samples, steps, groups, per_group, act, x=x, params=rng.choice(["f32", x]), train=train)
    rows = rng.choice([0, _log(rng, 100, 1048576)])
    return _clip(rows, rng.choice([47, 100, 128]), rng.randint(1, 20), rng.choice([64, 256, rng.randint(5, 300)]),
                 rng.choice(["f32", "bf16", "mixed"]), max_norm=rng.choice([1.0, 0.25]))


# ---------------------------------------------------------------- inputs --

def _ids(case, gen):
    rows, n = case["rows"], case["n"]
    if case["ids"] == "distinct":
        idx = torch.randperm(rows, generator=gen, device="cuda")[:n]
    elif case["ids"] == "uniform":
        idx = torch.randint(rows, (n,), generator=gen, device="cuda")
    else:
        u = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)
        idx = (u.pow(SKEW) * rows).long().clamp_(max=rows - 1)
    if case["pad"] and n > 1:  # a block filled up to a fixed size
        idx[n - max(1, n // 20):] = -1
    return idx.to(torch.int32 if case["index"] == "i32" else torch.int64)


def _grad_shapes(case):
    """(shape, type) of each gradient: a table, then weight, bias and norm parameters of each layer."""
    kinds = ["f32", "bf16", "f16"] if case["kinds"] == "mixed" else [case["kinds"]]
    h, shapes = case["hidden"], []
    if case["rows"]:
        shapes.append(((case["rows"], case["width"]), kinds[0]))
    for i in range(case["layers"]):
        k = kinds[(i + 1) % len(kinds)]
        shapes += [((100, h) if i == 0 else (h, h), k), ((h,), k), ((h,), "f32")]
    return shapes + [((h, 47), kinds[0])]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    if case["op"] == "lookup":
        return dict(case=case, idx=_ids(case, gen), table=normal(case["rows"], case["width"]).to(DTYPES[case["table"]]))
    if case["op"] == "lookup_grad":
        return dict(case=case, idx=_ids(case, gen), grad=normal(case["n"], case["width"]).to(DTYPES[case["out"]]))
    if case["op"] == "norm":
        c, x_type, p_type = case["groups"] * case["per_group"], DTYPES[case["x"]], DTYPES[case["params"]]
        shape = (case["samples"], c) if case["steps"] == 1 else (case["samples"], case["steps"], c)
        # aggregated features: channels differ in level and in spread
        level, spread = 0.5 * normal(c), 0.25 + normal(c).abs()
        state = dict(case=case, x=normal(*shape).mul_(spread).add_(level).to(x_type),
                     weight=(1 + 0.1 * normal(c)).to(p_type), bias=(0.1 * normal(c)).to(p_type))
        if case["train"]:
            state["dy"] = normal(*shape).to(x_type)
        return state
    params = []
    for shape, kind in _grad_shapes(case):
        p = torch.zeros(shape, dtype=DTYPES[kind], device="cuda")
        p.grad = (0.01 * normal(*shape)).to(DTYPES[kind])
        params.append(p)
    return dict(case=case, params=params)


# ------------------------------------------------------------- the passes --

def run(state):
    case = state["case"]
    if case["op"] == "lookup":
        pad = -1 if case["pad"] else None
        if own:
            from tcc_b200.embedding import embedding
            return embedding(state["table"], state["idx"], scale=case["scale"], padding_idx=pad,
                             out_dtype=DTYPES[case["out"]])
        idx = state["idx"]
        out = state["table"][idx.clamp(min=0)].float() * case["scale"]
        if case["pad"]:
            out = out * (idx >= 0)[:, None]
        return out.to(DTYPES[case["out"]])
    if case["op"] == "lookup_grad":
        if own:
            from tcc_b200.embedding import embedding_backward
            return embedding_backward(state["grad"], state["idx"], case["rows"], scale=case["scale"],
                                      padding_idx=-1 if case["pad"] else None, dtype=DTYPES[case["table"]])
        idx, grad = state["idx"], state["grad"].float() * case["scale"]
        if case["pad"]:
            grad = grad * (idx >= 0)[:, None]
        total = torch.zeros((case["rows"], case["width"]), device=grad.device)
        return total.index_add_(0, idx.clamp(min=0), grad).to(DTYPES[case["table"]])
    if case["op"] == "norm":
        return _norm_own(state) if own else _norm_plain(state)
    params = state["params"]
    if own:
        from tcc_b200.clip import clip_grad_norm_
        norm = clip_grad_norm_(params, case["max_norm"])
        return [norm] + [p.grad for p in params]
    squares = [p.grad.double().square().sum() for p in params]
    norm = torch.stack(squares).sum().sqrt()
    factor = (case["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    [p.grad.copy_(p.grad.float() * factor) for p in params]
    return [norm.float()] + [p.grad for p in params]


def _norm_own(state):
    from tcc_b200.norm import group_norm, group_norm_backward, group_norm_forward
    case, x, weight, bias = state["case"], state["x"], state["weight"], state["bias"]
    if not case["train"]:
        return group_norm(x, case["groups"], weight, bias, eps=1e-5, act=case["act"])
    y, mean, rstd = group_norm_forward(x, case["groups"], weight, bias, eps=1e-5, act=case["act"])
    dx, dw, db = group_norm_backward(state["dy"], x, mean, rstd, case["groups"], weight, bias, act=case["act"])
    return y, dx, dw, db


def _norm_plain(state):
    case = state["case"]
    shape = (case["samples"], case["steps"], case["groups"], case["per_group"])
    x = state["x"].float().view(shape)
    w = state["weight"].float().view(shape[2:])
    b = state["bias"].float().view(shape[2:])
    # sums over many nodes in 64 bits
    wide = torch.float64 if case["steps"] * case["per_group"] > 4096 else torch.float32
    mean = x.mean((1, 3), keepdim=True, dtype=wide).float()
    x = x - mean
    rstd = ((x * x).mean((1, 3), keepdim=True, dtype=wide) + 1e-5).rsqrt().float()
    hat = x * rstd
    z = hat * w + b
    act = case["act"]
    if act == "relu":
        y = z * (z > 0)
    elif act == "silu":
        gate = 1 / (1 + torch.exp(-z))
        y = z * gate
    elif act == "gelu":
        below = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        y = z * below
    else:
        y = z
    y = y.to(state["x"].dtype).view(state["x"].shape)
    if not case["train"]:
        return y
    dz = state["dy"].float().view(shape)
    if act == "silu":
        dz = dz * (gate * (1 + z * (1 - gate)))
    elif act == "gelu":
        dz = dz * (below + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi)))
    db = dz.sum((0, 1), dtype=torch.float64)
    dw = (dz * hat).sum((0, 1), dtype=torch.float64)
    dh = dz * w
    dx = rstd * (dh - dh.mean((1, 3), keepdim=True, dtype=wide).float()
                 - hat * (dh * hat).mean((1, 3), keepdim=True, dtype=wide).float())
    p_type = state["weight"].dtype
    return y, dx.to(state["x"].dtype).view(state["x"].shape), dw.to(p_type).view(-1), db.to(p_type).view(-1)


# ------------------------------------------------------------------ floor --

def _distinct(case):
    """Expected number of table rows that n indices touch."""
    n = case["n"] - (max(1, case["n"] // 20) if case["pad"] and case["n"] > 1 else 0)
    rows = case["rows"]
    if case["ids"] == "distinct":
        return n
    if case["ids"] == "uniform":
        return -rows * math.expm1(n * math.log1p(-1 / rows)) if rows > 1 else 1
    edge = (np.arange(rows + 1) / rows) ** (1 / SKEW)
    return float(-np.expm1(n * np.log1p(-np.minimum(np.diff(edge), 1 - 1e-12))).sum())


def work(case):
    if case["op"] in ("lookup", "lookup_grad"):
        ids = case["n"] * (4 if case["index"] == "i32" else 8)
        moved = case["n"] * case["width"]
        if case["op"] == "lookup":  # each touched row in, every looked-up row out
            return dict(bytes=ids + _distinct(case) * case["width"] * BYTES[case["table"]]
                        + moved * BYTES[case["out"]], flops=moved)
        return dict(bytes=ids + moved * BYTES[case["out"]] + case["rows"] * case["width"] * BYTES[case["table"]],
                    flops=2 * moved)
    if case["op"] == "norm":
        c = case["groups"] * case["per_group"]
        n = case["samples"] * case["steps"] * c
        return dict(bytes=(4 if case["train"] else 2) * n * BYTES[case["x"]]
                    + (4 if case["train"] else 2) * c * BYTES[case["params"]],
                    flops=(25 if case["train"] else 8) * n)
    sizes = [(math.prod(s), k) for s, k in _grad_shapes(case)]
    return dict(bytes=4 + 2 * sum(n * BYTES[k] for n, k in sizes), flops=3 * sum(n for n, _ in sizes))


# ---------------------------------------------------------- in 64 bits --

def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "lookup":
        idx = state["idx"].long()
        wide = torch.cat([state["table"].double().mul_(case["scale"]),
                          torch.zeros((1, case["width"]), dtype=torch.float64, device=idx.device)])
        return wide.index_select(0, torch.where(idx < 0, case["rows"], idx))  # -1: the zero row
    if case["op"] == "lookup_grad":
        # runs of equal index after a sort: differences of one running sum
        order = torch.argsort(state["idx"], stable=True)
        keys, counts = torch.unique_consecutive(state["idx"].long()[order], return_counts=True)
        ends = counts.cumsum(0)
        total = torch.zeros((case["rows"], case["width"]), dtype=torch.float64, device=keys.device)
        at = state["grad"].double()[order].cumsum(0)[ends - 1]
        at[1:] = at[1:] - at[:-1].clone()
        real = keys >= 0
        total[keys[real]] = at[real] * case["scale"]
        return total
    if case["op"] == "norm":
        x = state["x"].double().requires_grad_(case["train"])
        w = state["weight"].double().requires_grad_(case["train"])
        b = state["bias"].double().requires_grad_(case["train"])
        grouped = x.view(case["samples"], case["steps"], case["groups"], case["per_group"])
        var, mean = torch.var_mean(grouped, dim=(1, 3), correction=0, keepdim=True)
        z = ((grouped - mean) / torch.sqrt(var + 1e-5)).reshape(x.shape) * w + b
        y = {"none": lambda v: v, "relu": torch.relu, "silu": lambda v: v * torch.sigmoid(v),
             "gelu": lambda v: v * torch.special.ndtr(v)}[case["act"]](z)
        if not case["train"]:
            return y
        grads = torch.autograd.grad(y, (x, w, b), state["dy"].double())
        return (y.detach(), *grads)
    grads = [p.grad.double() for p in state["params"]]
    norm = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(g) for g in grads]))
    factor = min(1.0, case["max_norm"] / (float(norm) + 1e-6))
    return [norm] + [g * factor for g in grads]
