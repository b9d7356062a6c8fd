"""Embedding lookup with scaling and its sorted gradient (tcc_b200.embedding)
against 64-bit torch.

Tolerances, u = 2^-24 (fp32 rounding), u_t = eps/2 of the output type:
* lookup: one fp32 product, one rounding to the output type:
  |out - exact| <= (u + u_t) |exact|;
* gradient of a row with k terms: k - 1 fp32 additions in some order, the
  product with the scale, one rounding to the table's type:
  |out - exact| <= (k + 1) u |scale| sum|g| + u_t |exact|;
both plus one smallest subnormal of the output type."""
import pytest
import torch

from tcc_b200 import _lib as L
from tcc_b200 import embedding as E

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TINY = {F32: 2.0 ** -149, F16: 2.0 ** -24, BF16: 2.0 ** -133}


def _half_step(t):
    return torch.finfo(t).eps / 2


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _check_lookup(out, table, idx, scale, padding):
    real = (idx >= 0) & (idx < table.shape[0])
    if padding is not None:
        real &= idx != padding
    safe = torch.where(real, idx, 0).long()
    want = table.double()[safe] * scale if table.shape[0] else torch.zeros_like(out, dtype=torch.float64)
    want = torch.where(real[..., None], want, 0.0)
    tol = (U + _half_step(out.dtype)) * want.abs() + TINY[out.dtype]
    assert out.shape == want.shape
    assert bool(((out.double() - want).abs() <= tol).all())


def _check_grad(out, grad, idx, scale, padding):
    rows, width = out.shape
    flat, g = idx.reshape(-1).long(), grad.reshape(-1, width).double()
    real = (flat >= 0) & (flat < rows)
    if padding is not None:
        real &= flat != padding
    at = flat[real]
    want = torch.zeros((rows, width), dtype=torch.float64, device=out.device).index_add_(0, at, g[real]) * scale
    size = torch.zeros_like(want).index_add_(0, at, g[real].abs()) * abs(scale)
    terms = torch.bincount(at, minlength=rows)[:, None]
    tol = (terms + 1) * U * size + _half_step(out.dtype) * want.abs() + TINY[out.dtype]
    assert bool(((out.double() - want).abs() <= tol).all())
    assert bool((out[torch.bincount(at, minlength=rows) == 0] == 0).all())


def _ids(rows, n, kind, gen, dtype):
    if kind == "same":
        idx = torch.full((n,), rows // 2, device="cuda")
    elif kind == "skew":
        idx = (torch.rand(n, generator=gen, device="cuda").pow(4) * rows).long().clamp_(max=rows - 1)
    elif kind == "distinct":
        idx = torch.randperm(rows, generator=gen, device="cuda")[:n]
    else:
        idx = torch.randint(rows, (n,), generator=gen, device="cuda")
    return idx.to(dtype)


@pytest.mark.parametrize("types", [(F32, F32), (F16, F16), (BF16, F32)])
@pytest.mark.parametrize("width", [5, 7, 9, 13, 25, 33, 53, 89, 101, 127, 129, 257, 333, 523])
def test_lookup_odd_widths(gpu, types, width):
    gen = _gen(width)
    table = torch.randn((301, width), generator=gen, device="cuda").to(types[0])
    for n in (1, 37, 20011):
        idx = torch.randint(-1, 302, (n,), generator=gen, device="cuda")
        _check_lookup(E.embedding(table, idx, 1.7, padding_idx=-1, out_dtype=types[1]), table, idx, 1.7, -1)
    idx.fill_(-1)
    assert not E.embedding(table, idx, float("inf"), padding_idx=-1).any()
    wide = torch.randn((301, width + 4), generator=gen, device="cuda").to(types[0])
    for first in (1, 2):  # rows that begin anywhere
        view = wide[:, first:first + width]
        idx = torch.randint(301, (2003,), generator=gen, device="cuda")
        _check_lookup(E.embedding(view, idx, out_dtype=types[1]), view, idx, 1.0, None)


@pytest.mark.parametrize("types", [(F32, F32), (F16, F16), (F16, F32), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("width", [1, 2, 3, 47, 100, 128, 602, 2056])
def test_lookup_types_and_widths(gpu, types, width):
    gen = _gen(width)
    table = torch.randn((517, width), generator=gen, device="cuda").to(types[0])
    for n, it, scale in ((1, torch.int64, 1.0), (333, torch.int32, 0.3), (4097, torch.int64, -2.5)):
        idx = _ids(517, n, "uniform", gen, it)
        out = E.embedding(table, idx, scale=scale, out_dtype=types[1])
        assert out.dtype == types[1]
        _check_lookup(out, table, idx, scale, None)


@pytest.mark.parametrize("types", [(F32, F32), (F16, F16), (F16, F32), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("width", [1, 2, 3, 47, 100, 128, 602, 2056])
def test_gradient_types_and_widths(gpu, types, width):
    gen = _gen(width + 7)
    for rows, n, kind, it in ((300, 1, "uniform", torch.int64), (300, 2500, "skew", torch.int32),
                              (301, 9001, "uniform", torch.int64)):
        idx = _ids(rows, n, kind, gen, it)
        grad = torch.randn((n, width), generator=gen, device="cuda").to(types[1])
        out = E.embedding_backward(grad, idx, rows, scale=1.7, dtype=types[0])
        assert out.dtype == types[0]
        _check_grad(out, grad, idx, 1.7, None)


# row counts on both sides of a digit of the sort, index counts on both sides of
# its tiles, hubs, and one row that gets everything
@pytest.mark.parametrize("rows", [1, 2, 255, 256, 257, 2047, 2048, 2049, 65535, 65537, 300001])
@pytest.mark.parametrize("n,kind", [(1, "uniform"), (31, "skew"), (255, "distinct"), (1025, "uniform"),
                                    (2049, "skew"), (4096, "uniform"), (4097, "same"), (20000, "skew"),
                                    (100003, "uniform"), (100003, "same")])
def test_gradient_sizes(gpu, rows, n, kind):
    gen = _gen(rows * 7 + n)
    if kind == "distinct":
        n = min(n, rows)
    idx = _ids(rows, n, kind, gen, torch.int64)
    grad = torch.randn((n, 20), generator=gen, device="cuda")
    out = E.embedding_backward(grad, idx, rows)
    _check_grad(out, grad, idx, 1.0, None)


@pytest.mark.parametrize("n", [5, 700, 6000])
def test_padding_and_bad_indices(gpu, n):
    gen = _gen(n)
    table = torch.randn((50, 12), generator=gen, device="cuda")
    grad = torch.randn((n, 12), generator=gen, device="cuda")
    idx = torch.randint(50, (n,), generator=gen, device="cuda")
    idx[::3] = -1
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    _check_lookup(E.embedding(table, idx, 2.0, padding_idx=-1, bad=bad), table, idx, 2.0, -1)
    _check_grad(E.embedding_backward(grad, idx, 50, 2.0, padding_idx=-1, bad=bad), grad, idx, 2.0, -1)
    assert int(bad) == 0  # padding is not an error
    inside = idx.clamp(min=0)
    _check_lookup(E.embedding(table, inside, padding_idx=0, bad=bad), table, inside, 1.0, 0)
    _check_grad(E.embedding_backward(grad, inside, 50, padding_idx=0, bad=bad), grad, inside, 1.0, 0)
    assert int(bad) == 0
    for wrong in (50, -2, 1 << 40, -(1 << 62)):
        idx[1] = wrong
        for call in (lambda: _check_lookup(E.embedding(table, idx, padding_idx=-1, bad=bad), table, idx, 1.0, -1),
                     lambda: _check_grad(E.embedding_backward(grad, idx, 50, padding_idx=-1, bad=bad), grad, idx,
                                         1.0, -1)):
            bad.zero_()
            call()
            assert int(bad) == 1
    idx.fill_(-1)  # nothing but padding
    assert not E.embedding_backward(grad, idx, 50, padding_idx=-1).any()
    assert not E.embedding(table, idx, float("inf"), padding_idx=-1).any()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_offsets_and_shapes(gpu, dtype):
    gen = _gen(3)
    wide = torch.randn((90, 61), generator=gen, device="cuda").to(dtype)
    for first, width in ((0, 60), (1, 60), (3, 8), (4, 57), (5, 1)):
        table = wide[:, first:first + width]
        idx = torch.randint(90, (7, 5, 3), generator=gen, device="cuda")
        out = E.embedding(table, idx, 0.5)
        assert out.shape == (7, 5, 3, width)
        _check_lookup(out, table, idx, 0.5, None)
        # every other index, read through a strided view
        part = torch.randint(90, (400,), generator=gen, device="cuda", dtype=torch.int32)[::2]
        _check_lookup(E.embedding(table, part), table, part, 1.0, None)
        g = torch.randn((200, 61), generator=gen, device="cuda").to(dtype)[:, first:first + width]
        _check_grad(E.embedding_backward(g, part, 90), g, part, 1.0, None)
        ones = torch.ones((), device="cuda", dtype=dtype).expand(200, width)  # a broadcast gradient
        _check_grad(E.embedding_backward(ones, part, 90), ones, part, 1.0, None)
        t = torch.randn((width, 200), generator=gen, device="cuda").to(dtype).t()
        _check_grad(E.embedding_backward(t, part, 90), t, part, 1.0, None)


def test_gradient_leaves_columns_beyond_the_width(gpu):
    """The C call with a row stride wider than F: what lies between the rows stays."""
    gen = _gen(4)
    for n in (3, 5000):
        idx = torch.randint(40, (n,), generator=gen, device="cuda")
        grad = torch.randn((n, 10), generator=gen, device="cuda")
        out = torch.full((40, 16), 7.0, device="cuda")
        nbytes = L.lib().tcc_embedding_backward_scratch_bytes(n, 40, 10)
        scratch = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
        L.call("tcc_embedding_backward", grad.data_ptr(), L.F32, 10, idx.data_ptr(), L.I64, n, L.NO_PADDING, 1.0,
               out.data_ptr(), L.F32, 16, 40, 10, scratch.data_ptr(), nbytes, None,
               torch.cuda.current_stream().cuda_stream)
        _check_grad(out[:, :10], grad, idx, 1.0, None)
        assert bool((out[:, 10:] == 7.0).all())


@pytest.mark.parametrize("rows,width,dtype", [(300007, 100, F32), (13, 3, BF16), (60001, 5, F16), (1, 1, F32)])
@pytest.mark.parametrize("n", [1025, 9001, 40961, 65536, 65537])
def test_gradient_covers_every_row_and_no_more(gpu, rows, width, dtype, n):
    """Rows without an index are written wherever the zeroing beside the sort ends; what lies behind the table stays."""
    gen = _gen(rows + n)
    idx = torch.randint(rows, (n,), generator=gen, device="cuda")
    grad = torch.randn((n, width), generator=gen, device="cuda").to(dtype)
    out = torch.full((rows * width + 8,), float("nan"), device="cuda", dtype=dtype)
    out[rows * width:] = 7.0
    nbytes = L.lib().tcc_embedding_backward_scratch_bytes(n, rows, width)
    scratch = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    code = {F32: L.F32, F16: L.F16, BF16: L.BF16}[dtype]
    L.call("tcc_embedding_backward", grad.data_ptr(), code, width, idx.data_ptr(), L.I64, n, L.NO_PADDING, 1.0,
           out.data_ptr(), code, width, rows, width, scratch.data_ptr(), nbytes, None,
           torch.cuda.current_stream().cuda_stream)
    _check_grad(out[:rows * width].view(rows, width), grad, idx, 1.0, None)
    assert bool((out[rows * width:] == 7.0).all())


def test_empty(gpu):
    table = torch.randn((5, 4), device="cuda")
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    assert E.embedding(table, none).shape == (0, 4)
    assert not E.embedding_backward(torch.empty((0, 4), device="cuda"), none, 5).any()
    assert E.embedding_backward(torch.empty((0, 4), device="cuda"), none, 0).shape == (0, 4)
    some = torch.tensor([0, 1], device="cuda")
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert not E.embedding(torch.empty((0, 4), device="cuda"), some, bad=bad).any()
    assert int(bad) == 1
    assert E.embedding_backward(torch.ones((2, 4), device="cuda"), some, 0).shape == (0, 4)
    assert E.embedding(torch.empty((5, 0), device="cuda"), some).shape == (2, 0)


@pytest.mark.parametrize("n,kind", [(1500, "skew"), (50021, "skew"), (50021, "same")])
def test_gradient_is_the_same_bits_every_time(gpu, n, kind):
    gen = _gen(n)
    idx = _ids(4000, n, kind, gen, torch.int64)
    grad = torch.randn((n, 33), generator=gen, device="cuda")
    first = E.embedding_backward(grad, idx, 4000)
    for _ in range(5):
        assert torch.equal(E.embedding_backward(grad, idx, 4000), first)


def test_nonfinite_rows_stay_where_they_are(gpu):
    table = torch.randn((6, 8), device="cuda")
    table[2, 3], table[4] = float("nan"), float("inf")
    idx = torch.tensor([0, 2, 4, -1], device="cuda")
    out = E.embedding(table, idx, 2.0, padding_idx=-1)
    assert bool(out[1, 3].isnan()) and int(out.isnan().sum()) == 1
    assert bool(out[2].isinf().all()) and not out[3].any()
    grad = torch.ones((4, 8), device="cuda")
    grad[3] = float("nan")  # the padded row's gradient is not read into any sum
    grad[1, 0] = float("inf")
    dt = E.embedding_backward(grad, idx, 6, padding_idx=-1)
    assert not dt.isnan().any() and bool(dt[2, 0].isinf()) and int(dt.isinf().sum()) == 1


def test_offsets_past_32_bits(gpu):
    """A table, and a gradient, of more than 2^31 elements (5 GB)."""
    rows, width = 10_000_019, 256
    table = torch.zeros((rows, width), dtype=BF16, device="cuda")
    picks = torch.tensor([rows - 1, 0, 8_388_609, 8_388_607, rows - 1, 9_999_999], device="cuda")
    for k, r in enumerate(picks.tolist()):
        table[r] = k + 1.0
    out = E.embedding(table, picks)
    assert torch.equal(out[:, 7].float().cpu(), torch.tensor([5.0, 2.0, 3.0, 4.0, 5.0, 6.0]))
    grad = torch.arange(1, 7, device="cuda", dtype=BF16)[:, None].expand(6, width).contiguous()
    for repeat in (1, 1000):  # few indices, and many
        idx, g = picks.repeat(repeat), grad.repeat(repeat, 1)
        dt = E.embedding_backward(g, idx, rows)
        # the sums are whole numbers below 2^24, exact in fp32; bf16 keeps 8 bits of each
        sums = torch.tensor([2.0, 4.0, 3.0, 6.0, 6.0], device="cuda").mul(repeat).to(BF16)
        at = [0, 8_388_607, 8_388_609, 9_999_999, rows - 1]
        assert torch.equal(dt[at], sums[:, None].expand(5, width))
        assert float(dt.sum(dtype=torch.float64)) == float(sums.double().sum()) * width
        del dt


def test_autograd_and_differences(gpu):
    gen = _gen(11)
    table = torch.randn((40, 6), generator=gen, device="cuda", requires_grad=True)
    idx = torch.randint(40, (3, 50), generator=gen, device="cuda")
    idx[0, :5] = -1
    w = torch.randn((3, 50, 6), generator=gen, device="cuda")

    def f(t):
        return float((E.embedding(t, idx, 1.5, padding_idx=-1).double() * w.double()).sum())

    out = E.embedding(table, idx, 1.5, padding_idx=-1)
    (out * w).sum().backward()
    _check_grad(table.grad, w, idx, 1.5, -1)
    step = 2.0 ** -6  # linear: the difference is exact up to the roundings of f's rows
    for r, c in ((0, 0), (13, 5), (39, 2)):
        t = table.detach().clone()
        t[r, c] += step
        up = f(t)
        t[r, c] -= 2 * step
        slope = (up - f(t)) / (2 * step)
        terms = int((idx == r).sum())
        bound = terms * 8 * 1.5 * U * float(w.abs().max()) * (float(t.abs().max()) + 1) / step
        assert abs(slope - float(table.grad[r, c])) <= bound + 1e-12
    assert not E.embedding(table.detach(), idx, padding_idx=-1).requires_grad
    layer = E.NodeEmbedding(30, 10, scale=0.5, dtype=BF16, out_dtype=F32, device="cuda")
    y = layer(torch.arange(30, device="cuda"))
    assert y.dtype == F32
    y.sum().backward()
    assert layer.weight.grad.dtype == BF16 and bool((layer.weight.grad == 0.5).all())


def test_other_stream_and_captured_graph(gpu):
    gen = _gen(12)
    table = torch.randn((5000, 64), generator=gen, device="cuda")
    side = torch.cuda.Stream()
    for n in (64, 7000):
        idx = torch.randint(5000, (n,), generator=gen, device="cuda")
        grad = torch.randn((n, 64), generator=gen, device="cuda")
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            out, dt = E.embedding(table, idx), E.embedding_backward(grad, idx, 5000)
        torch.cuda.current_stream().wait_stream(side)
        _check_lookup(out, table, idx, 1.0, None)
        _check_grad(dt, grad, idx, 1.0, None)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, dt = E.embedding(table, idx), E.embedding_backward(grad, idx, 5000)
        for seed in (1, 2):
            idx.copy_(_ids(5000, n, "skew", _gen(seed), torch.int64))
            grad.copy_(torch.randn((n, 64), generator=_gen(seed + 9), device="cuda"))
            out.fill_(float("nan"))
            dt.fill_(float("nan"))
            graph.replay()
            _check_lookup(out, table, idx, 1.0, None)
            _check_grad(dt, grad, idx, 1.0, None)


def test_two_streams_at_once(gpu):
    gen = _gen(13)
    idx = [_ids(20000, 60000, "skew", gen, torch.int64) for _ in range(2)]
    grad = [torch.randn((60000, 32), generator=gen, device="cuda") for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[k].append(E.embedding_backward(grad[k], idx[k], 20000))
    torch.cuda.synchronize()
    for k in range(2):
        for o in outs[k]:
            _check_grad(o, grad[k], idx[k], 1.0, None)
            assert torch.equal(o, outs[k][0])
