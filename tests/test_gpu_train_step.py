"""Embedding lookup, aggregation, group norm, dropout epilogue and clipping
together, as a training step uses them, against 64-bit torch; and the trainer's
norm and clipping options."""
import numpy as np
import pytest
import torch

from gpu_util import csr_dev, rel_fro
from tcc_b200 import clip, gcn, minibatch, train_gcn
from tcc_b200 import embedding as E
from tcc_b200 import graphs as G
from tcc_b200 import norm as N

pytestmark = pytest.mark.gpu

# fp32-accurate tiles (1e-5 per aggregation, the SpMM tests' tolerance), two
# aggregations forward and two backward, three fp32 products in between
STEP_TOL = 1e-4


def _dense(g, dev):
    A = torch.zeros((g.rows, g.cols), dtype=torch.float64, device=dev)
    rows = torch.repeat_interleave(torch.arange(g.rows), torch.from_numpy(np.diff(g.rowptr.astype(np.int64))))
    A[rows.to(dev), torch.from_numpy(g.col.astype(np.int64)).to(dev)] = 1.0
    return A


def _reference_norm(x, groups, w, b):
    v = x.view(x.shape[0], groups, -1)
    v = (v - v.mean(2, keepdim=True)) / torch.sqrt(v.var(2, keepdim=True, correction=0) + 1e-5)
    return v.reshape(x.shape) * w + b


@pytest.mark.parametrize("table_type", [torch.float32, torch.bfloat16])
def test_full_graph_step(gpu, table_type):
    """Rows of a learned table -> A -> W1 -> group norm, silu -> A -> W2 -> loss; clip; step."""
    dev = gpu
    g = G.rmat(10, 8 << 10, seed=31)
    rp, col = csr_dev(g)
    rs, cs = (torch.from_numpy(v).to(dev) for v in G.gcn_scales(g))
    tg = gcn.TiledGraph(rp, col, g.rows, rs=rs, cs=cs, tc_threshold=65)
    gen = torch.Generator(device=dev).manual_seed(32)
    types, feats, hidden, classes = 61, 64, 48, 16
    kinds = torch.randint(types, (g.rows,), generator=gen, device=dev)  # a node's type
    table = torch.randn((types, feats), generator=gen, device=dev).to(table_type).requires_grad_(True)
    W1 = (torch.randn((feats, hidden), generator=gen, device=dev) / 8).requires_grad_(True)
    W2 = (torch.randn((hidden, classes), generator=gen, device=dev) / 7).requires_grad_(True)
    layer = N.GroupNorm(6, hidden, act="silu", device=dev)
    with torch.no_grad():
        layer.weight.mul_(1 + 0.2 * torch.randn(hidden, generator=gen, device=dev))
        layer.bias.add_(0.2 * torch.randn(hidden, generator=gen, device=dev))
    labels = torch.randint(classes, (200,), generator=gen, device=dev)
    labelled = torch.randperm(g.rows, generator=gen, device=dev)[:200]
    params = [table, W1, W2, layer.weight, layer.bias]

    x = E.embedding(table, kinds, scale=2.0, out_dtype=torch.float32)
    h = layer(gcn._Aggregate.apply(tg, x) @ W1)
    logits = gcn._Aggregate.apply(tg, h) @ W2
    loss = torch.nn.functional.cross_entropy(E.embedding(logits, labelled), labels)
    loss.backward()

    ref = [p.detach().double().requires_grad_(True) for p in params]
    A = rs.double()[:, None] * _dense(g, dev) * cs.double()[None, :]
    rh = torch.nn.functional.silu(_reference_norm(A @ (2.0 * ref[0][kinds]) @ ref[1], 6, ref[3], ref[4]))
    rl = torch.nn.functional.cross_entropy((A @ rh @ ref[2])[labelled], labels)
    rl.backward()
    assert abs(float(loss) - float(rl)) <= STEP_TOL * float(rl)
    for p, r in zip(params, ref):
        tol = STEP_TOL + (2.0 ** -8 if p.dtype == torch.bfloat16 else 0.0)
        assert p.grad.dtype == p.dtype
        assert rel_fro(p.grad.float().cpu().numpy(), r.grad.cpu().numpy()) <= tol
    grads = [p.grad.clone() for p in params]
    total = float(torch.stack([v.double().square().sum() for v in grads]).sum().sqrt())
    got = clip.clip_grad_norm_(params, 0.5 * total)
    assert abs(float(got) - total) <= 1e-6 * total
    for p, v in zip(params, grads):
        assert rel_fro(p.grad.float().cpu().numpy(), 0.5 * v.float().cpu().numpy()) <= \
            1e-5 + (2.0 ** -8 if p.dtype == torch.bfloat16 else 0.0)


def test_block_rows_from_a_learned_table(gpu):
    g = G.rmat(11, 12 << 11, seed=33)
    rp, col = csr_dev(g)
    gen = torch.Generator(device="cuda").manual_seed(34)
    seeds = torch.randperm(g.rows, device="cuda", generator=gen)[:200]
    blocks = minibatch.sample_blocks(rp, col, seeds, (5, 10), generator=gen)
    table = torch.randn((g.rows, 32), generator=gen, device="cuda").bfloat16().requires_grad_(True)
    x = minibatch.embedding_rows(table, blocks[0], scale=0.5)
    assert x.dtype == torch.float32 and torch.equal(x, table.detach().float()[blocks[0].src_ids] * 0.5)
    bcsr, _ = minibatch.block_tiles(blocks[0])
    y = gcn.T.bcsr_spmm(bcsr, x.detach(), tc_threshold=65)  # the aggregation takes the rows as they are
    assert y.shape == (blocks[0].num_dst, 32)
    x.sum().backward()
    want = torch.zeros_like(table.detach())
    want[blocks[0].src_ids] = 0.5  # a block's source ids are distinct
    assert torch.equal(table.grad, want)


@pytest.mark.parametrize("training,p", [(True, 0.5), (True, 0.0), (False, 0.5)])
def test_gcn_with_norm(gpu, training, p):
    g = G.rmat(9, 8 << 9, seed=35)
    rp, col = csr_dev(g)
    tg = gcn.TiledGraph(rp, col, g.rows, tc_threshold=65)
    torch.manual_seed(1)
    model = gcn.GCN(32, 40, 8, dropout=p, seed=3, norm_groups=5).to(gpu).train(training)
    x = torch.randn((g.rows, 32), device=gpu)
    out = model(tg, x)
    h = N.group_norm(tg.aggregate(x) @ model.conv1.weights, 5, model.norm.weight, model.norm.bias)
    want = tg.aggregate(gcn.relu_dropout(h, p, 3 * 1_000_003 + 1, training)) @ model.conv_final.weights
    assert rel_fro(out.detach().cpu().numpy(), want.detach().cpu().numpy()) <= 1e-5
    out.sum().backward()
    assert model.norm.weight.grad is not None and model.norm.bias.grad is not None


def test_trainer_with_norm_and_clipping(gpu, tmp_path):
    """The options reach the step: the clipped gradient's norm bounds what SGD-like
    updates see, a checkpoint carries the norm's parameters, and runs repeat."""
    cfg = train_gcn.config(shrink=10)
    cfg.update(dropout=0.0, norm_groups=8, clip_norm=1e-3)
    ck = str(tmp_path / "gcn.pt")
    whole = train_gcn.train(dict(cfg, epochs=4), gpu, 1, 0)
    first = train_gcn.train(dict(cfg, epochs=2, save=ck), gpu, 1, 0)
    rest = train_gcn.train(dict(cfg, epochs=4, resume=ck), gpu, 1, 0)
    got = first["losses"] + rest["losses"]
    assert len(got) == 4 and all(np.isfinite(got))
    assert max(abs(a - b) / b for a, b in zip(got, whole["losses"])) < 1e-4
    saved = torch.load(ck, map_location="cpu")
    assert set(saved["norm"]) == {"weight", "bias"} and saved["norm"]["weight"].shape == (cfg["hidden"],)
    plain = train_gcn.train(dict(cfg, epochs=1, norm_groups=0, clip_norm=None), gpu, 1, 0)
    assert abs(plain["losses"][0] - whole["losses"][0]) > 1e-6  # the norm changes the model


def test_functional_chain_in_a_captured_graph(gpu):
    """Lookup, norm, their gradients and clipping in one captured graph, replayed on new values."""
    gen = torch.Generator(device="cuda").manual_seed(36)
    table = torch.randn((3000, 64), generator=gen, device="cuda")
    idx = torch.randint(3000, (5000,), generator=gen, device="cuda")
    w, b = torch.ones(64, device="cuda"), torch.zeros(64, device="cuda")
    p = torch.zeros_like(table)
    p.grad = torch.zeros_like(table)

    def chain():
        x = E.embedding(table, idx, 1.5)
        y, mean, rstd = N.group_norm_forward(x, 8, w, b, act="silu")
        dx, dw, db = N.group_norm_backward(y, x, mean, rstd, 8, w, b, act="silu")
        p.grad.copy_(E.embedding_backward(dx, idx, 3000, 1.5))
        return y, dw, db, clip.clip_grad_norm_([p], 0.25)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        chain()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = chain()
    for seed in (37, 38):
        new = torch.Generator(device="cuda").manual_seed(seed)
        table.copy_(torch.randn((3000, 64), generator=new, device="cuda"))
        idx.copy_(torch.randint(3000, (5000,), generator=new, device="cuda"))
        graph.replay()
        got = [o.clone() for o in outs] + [p.grad.clone()]
        want = list(chain()) + [p.grad]
        assert all(torch.equal(a, v) for a, v in zip(got, want))  # every order of sums is fixed


COLD = """
import torch
from tcc_b200 import clip, embedding, norm
dev = "cuda"
idx = torch.randint(3000, (80000,), device=dev)
g = torch.randn(80000, 64, device=dev)
xs = [torch.randn(*s, device=dev) for s in ((2, 9000, 64), (500, 64), (5, 300, 64))]
w = torch.ones(64, device=dev)
p = torch.zeros(300000, device=dev)
p.grad = torch.randn(300000, device=dev)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    d = [embedding.embedding_backward(g[:n], idx[:n], 3000) for n in (500, 5000, 80000)]
    e = embedding.embedding(d[2], idx)
    y = [norm.group_norm_forward(x, 8, w, w, act="gelu") for x in xs]
    dx = [norm.group_norm_backward(x, x, m, r, 8, w, w, act="gelu") for x, (_, m, r) in zip(xs, y)]
    total = clip.clip_grad_norm_([p], 1.0)
graph.replay()
torch.cuda.synchronize()
for n, t in zip((500, 5000, 80000), d):
    assert torch.equal(t, embedding.embedding_backward(g[:n], idx[:n], 3000))
assert torch.equal(e, embedding.embedding(d[2], idx))
for x, (o, m, r), t in zip(xs, y, dx):
    assert torch.equal(o, norm.group_norm(x, 8, w, w, act="gelu"))
    assert all(torch.equal(a, b) for a, b in zip(t, norm.group_norm_backward(x, x, m, r, 8, w, w, act="gelu")))
assert abs(float(clip.grad_norm([p.grad])) - 1.0) < 1e-5 and float(total) > 1.0
print("done")
"""


def test_captured_before_any_other_call(gpu):
    """A process whose first calls of every form are captured into a graph."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", COLD], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "done" in r.stdout, r.stderr[-2000:]


@pytest.mark.parametrize("captured", [False, True])
def test_back_to_back_calls_give_what_they_give_alone(gpu, captured):
    """Kernels of one call overlap where they may; calls that follow each other, in scratch that the
    allocator hands on, do not see each other's: the same bits as with the device idle before each."""
    gen = torch.Generator(device=gpu).manual_seed(57)

    def rand(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=gen, device=gpu).to(dtype)

    jobs = []
    for n, rows, width, dtype in [(200003, 30011, 64, torch.float32), (5003, 70001, 100, torch.bfloat16),
                                  (90001, 47, 96, torch.float32), (3001, 9, 33, torch.float16)]:
        idx, grad = torch.randint(rows, (n,), generator=gen, device=gpu), rand(n, width, dtype=dtype)
        jobs.append(lambda idx=idx, grad=grad, rows=rows: (E.embedding_backward(grad, idx, rows),))
    for shape, groups, act, dtype in [((1, 20011, 96), 6, "silu", torch.bfloat16), ((3, 9001, 64), 4, "gelu", torch.float32),
                                      ((8, 517, 100), 10, "none", torch.float32), ((5003, 128), 8, "relu", torch.float16)]:
        x, dy, w, b = rand(*shape, dtype=dtype), rand(*shape, dtype=dtype), rand(shape[-1]), rand(shape[-1])

        def norm(x=x, dy=dy, w=w, b=b, groups=groups, act=act):
            y, mean, rstd = N.group_norm_forward(x, groups, w, b, act=act)
            return (y, mean, rstd, *N.group_norm_backward(dy, x, mean, rstd, groups, w, b, act=act))
        jobs.append(norm)
    for count in (40, 600):
        grads = [rand(3001 + 7 * i) for i in range(count)]

        def clipped(grads=grads):
            copies = [g.clone() for g in grads]
            norm = clip.grad_norm(copies)
            clip.clip_grads_with_norm_(copies, 1.5, norm)
            again = torch.nn.ParameterList([torch.nn.Parameter(c) for c in copies])
            for p, g in zip(again, grads):
                p.grad = g.clone()
            return (norm, *copies, clip.clip_grad_norm_(list(again), 2.5), *[p.grad for p in again])
        jobs.append(clipped)

    def alone(job):
        torch.cuda.synchronize()
        out = job()
        torch.cuda.synchronize()
        return out
    want = [alone(job) for job in jobs]

    def all_of(times):
        return [[job() for job in jobs] for _ in range(times)]
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = all_of(2)
        for _ in range(3):
            graph.replay()
    else:
        all_of(1)  # its memory is handed on
        got = all_of(4)
    torch.cuda.synchronize()
    for outs in got:
        for out, expect in zip(outs, want):
            assert all(torch.equal(o, e) for o, e in zip(out, expect))
