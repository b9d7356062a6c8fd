"""Group norm with an activation (tcc_b200.norm) against its 64-bit formula.

Tolerances.  u = 2^-24, u_t = eps/2 of the output type, and D = 192, above the
length of any chain of fp32 operations behind one statistic at the sizes tested
(a thread's block of at most 32 values, its merges, the trees over a CTA and a
sample; each merge is a few operations).  With A = mean |x| of the group:
* h = (x - mean) * rstd is off by at most   eh = D u (A rstd + |h| + 1)
  (the error of the mean, at most D u A, over the deviation; rstd's relative
  error, at most D u (1 + A rstd) from its variance; the final operations);
* y: |w| eh + 4 u (|w h| + |b|), times the activation's slope (at most 1.13),
  plus 8 u |z| for the activation itself, plus u_t |y|;
* dz = dy act'(z): ed = |dy| (|w| eh * 0.8 + 16 u) (0.8 bounds |act''|);
* db: sum ed + D u sum |dz|;  dw: sum (ed |h| + |dz| eh) + D u sum |dz h|;
* dx: rstd (|w| ed + D u |dz w| + mean(|w| ed + D u |dz w|)
      + |h| mean(|w| (ed |h| + |dz| eh) + D u |dz w h|) + eh mean|dz w h|)
      + D u (1 + A rstd) |dx|, plus u_t |dx|.
The slope of relu jumps at 0: where |z| < 1e-3 the tests make dy zero."""
import math

import pytest
import torch

from tcc_b200 import _lib as L
from tcc_b200 import norm as N

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
D = 192
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TINY = {F32: 2.0 ** -149, F16: 2.0 ** -24, BF16: 2.0 ** -133}


def _half_step(t):
    return torch.finfo(t).eps / 2


def _act(act, z):
    phi = 0.5 * (1 + torch.erf(z / math.sqrt(2)))
    sig = torch.sigmoid(z)
    if act == "relu":
        return z.clamp(min=0), (z > 0).double()
    if act == "silu":
        return z * sig, sig * (1 + z * (1 - sig))
    if act == "gelu":
        return z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return z, torch.ones_like(z)


class Oracle:
    """The formula in 64 bits on x [N, S, G, Cg], and the bounds above."""

    def __init__(self, x, groups, w, b, eps, act):
        c = x.shape[-1]
        self.shape = x.shape
        self.x = x.double().reshape(x.shape[0], -1, groups, c // groups)
        self.w = (torch.ones(c, device=x.device) if w is None else w).double().view(groups, -1)
        self.b = (torch.zeros(c, device=x.device) if b is None else b).double().view(groups, -1)
        dims = (1, 3)
        self.mean = self.x.mean(dims, keepdim=True)
        var = (self.x - self.mean).square().mean(dims, keepdim=True)
        self.rstd = 1 / torch.sqrt(var + eps)
        self.h = (self.x - self.mean) * self.rstd
        self.z = self.h * self.w + self.b
        self.y, self.slope = _act(act, self.z)
        self.away = self.x.abs().mean(dims, keepdim=True) * self.rstd
        self.eh = D * U * (self.away + self.h.abs() + 1)

    def check_forward(self, y, mean=None, rstd=None):
        w, b = self.w.abs(), self.b.abs()
        tol = 1.13 * (w * self.eh + 4 * U * (w * self.h.abs() + b)) + 8 * U * self.z.abs() \
            + _half_step(y.dtype) * self.y.abs() + TINY[y.dtype]
        err = (y.double().view_as(self.y) - self.y).abs()
        assert bool((err <= tol).all()), float((err / tol).max())
        if mean is not None:
            a = self.x.abs().mean((1, 3))
            assert bool(((mean.double() - self.mean[:, 0, :, 0]).abs() <= D * U * a + TINY[F32]).all())
            r = self.rstd[:, 0, :, 0]
            assert bool(((rstd.double() - r).abs() <= D * U * (1 + a * r) * r).all())

    def check_backward(self, dy, dx, dw, db):
        dims = (1, 3)
        dy = dy.double().reshape(self.x.shape)
        dz, w, h = dy * self.slope, self.w.abs(), self.h.abs()
        ed = dy.abs() * (0.8 * w * self.eh + 16 * U)
        dh = dz * self.w
        if db is not None:
            want = dz.sum((0, 1))
            tol = (ed + D * U * dz.abs()).sum((0, 1)) + _half_step(db.dtype) * want.abs() + TINY[db.dtype]
            err = (db.double().view_as(want) - want).abs()
            assert bool((err <= tol).all()), float((err / tol).max())
        if dw is not None:
            want = (dz * self.h).sum((0, 1))
            tol = (ed * h + dz.abs() * self.eh + D * U * (dz * self.h).abs()).sum((0, 1)) \
                + _half_step(dw.dtype) * want.abs() + TINY[dw.dtype]
            err = (dw.double().view_as(want) - want).abs()
            assert bool((err <= tol).all()), float((err / tol).max())
        if dx is not None:
            m1, m2 = dh.mean(dims, keepdim=True), (dh * self.h).mean(dims, keepdim=True)
            want = self.rstd * (dh - m1 - self.h * m2)
            e1 = w * ed + D * U * dh.abs()
            e2 = w * (ed * h + dz.abs() * self.eh) + D * U * (dh * self.h).abs()
            tol = self.rstd * (e1 + e1.mean(dims, keepdim=True) + h * e2.mean(dims, keepdim=True)
                               + self.eh * (dh * self.h).abs().mean(dims, keepdim=True)) \
                + D * U * (1 + self.away) * want.abs() + _half_step(dx.dtype) * want.abs() + TINY[dx.dtype]
            err = (dx.double().reshape(want.shape) - want).abs()
            assert bool((err <= tol).all()), float((err / tol).max())


def _inputs(shape, dtype, p_dtype, seed, level=0.5):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*s):
        return torch.randn(s, generator=gen, device="cuda")

    c = shape[-1]
    x = (normal(*shape) * (0.25 + normal(c).abs()) + level * normal(c)).to(dtype)
    w, b = (1 + 0.3 * normal(c)).to(p_dtype), (0.3 * normal(c)).to(p_dtype)
    return x, w, b, normal(*shape).to(dtype)


def _both(x, groups, w, b, dy, act, eps=1e-5):
    o = Oracle(x, groups, w, b, eps, act)
    if act == "relu":
        dy = torch.where((o.z.abs() < 1e-3).view(dy.shape), torch.zeros_like(dy), dy)
    y, mean, rstd = N.group_norm_forward(x, groups, w, b, eps, act)
    o.check_forward(y, mean, rstd)
    assert torch.equal(N.group_norm(x, groups, w, b, eps, act), y)
    dx, dw, db = N.group_norm_backward(dy, x, mean, rstd, groups, w, b, act)
    assert (dw is None) == (w is None) and (db is None) == (b is None)
    o.check_backward(dy, dx, dw, db)


# rows by themselves: group widths from one value on, odd ones, wider than a warp holds
@pytest.mark.parametrize("groups,per", [(1, 4), (8, 32), (32, 8), (4, 64), (5, 10), (3, 7), (47, 3), (2, 128),
                                        (1, 256), (6, 100), (1, 602), (2, 1000), (300, 4), (100, 2), (1, 2500)])
@pytest.mark.parametrize("rows", [1, 2, 77, 1500])
def test_rows(gpu, groups, per, rows):
    x, w, b, dy = _inputs((rows, groups * per), F32, F32, groups * 100 + per + rows)
    _both(x, groups, w, b, dy, "silu")


# samples over many rows: one value to many a group, one row more or less than a chunk
@pytest.mark.parametrize("groups,per", [(1, 4), (8, 32), (32, 8), (10, 10), (3, 7), (1, 47), (2, 300), (1, 1100),
                                        (300, 4), (1, 1)])
@pytest.mark.parametrize("n,steps", [(1, 8), (3, 33), (5, 257), (2, 5001), (700, 3)])
def test_samples(gpu, groups, per, n, steps):
    if n * steps * groups * per > 12_000_000:
        pytest.skip("large")
    x, w, b, dy = _inputs((n, steps, groups * per), F32, F32, groups * 100 + per + n)
    _both(x, groups, w, b, dy, "gelu")


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu"])
@pytest.mark.parametrize("dtype,p_dtype", [(F32, F32), (F16, F16), (F16, F32), (BF16, BF16), (BF16, F32), (F32, BF16)])
@pytest.mark.parametrize("shape,groups", [((65, 256), 8), ((2, 130, 48), 4), ((3, 5, 7, 30), 5), ((33, 21), 7)])
def test_types_and_activations(gpu, act, dtype, p_dtype, shape, groups):
    x, w, b, dy = _inputs(shape, dtype, p_dtype, len(shape))
    _both(x, groups, w, b, dy, act)


@pytest.mark.parametrize("shape", [(50, 64), (4, 40, 64)])
@pytest.mark.parametrize("w_on,b_on", [(False, False), (True, False), (False, True)])
def test_without_parameters(gpu, shape, w_on, b_on):
    x, w, b, dy = _inputs(shape, F32, F32, 5)
    _both(x, 8, w if w_on else None, b if b_on else None, dy, "silu")


@pytest.mark.parametrize("shape", [(300, 64), (2, 3000, 64)])
def test_large_mean(gpu, shape):
    """A mean 300 times the deviation: sums of squares would lose the variance."""
    x, w, b, dy = _inputs(shape, F32, F32, 6, level=300.0)
    x = x + 500.0
    _both(x, 8, w, b, dy, "none")


@pytest.mark.parametrize("shape", [(9, 64), (2, 300, 64)])
def test_constant_group_and_outlier(gpu, shape):
    x, w, b, dy = _inputs(shape, F32, F32, 7)
    flat = x.view(-1, 64)
    flat[:, :8] = 3.0     # a group without variance: h is 0, y is act(bias)
    flat[0, 8] = 1e4      # one value far from its group
    y = N.group_norm(x, 8, w, b)
    assert bool(((y.view(-1, 64)[:, :8] - b[:8]).abs() <= 1e-4).all())
    Oracle(x, 8, w, b, 1e-5, "none").check_forward(y)
    _both(x[..., 8:].contiguous(), 7, w[8:].contiguous(), b[8:].contiguous(), dy[..., 8:].contiguous(), "none")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_and_offsets(gpu, dtype):
    for shape, groups in (((37, 70), 5), ((3, 41, 70), 5)):
        x, w, b, dy = _inputs(shape, dtype, F32, 8)
        for first, c in ((0, 70), (0, 40), (1, 60), (2, 40), (30, 40), (5, 5)):
            part = (..., slice(first, first + c))
            _both(x[part], groups, w[first:first + c], b[first:first + c], dy[part], "silu")
        # rows in another order: a copy is made
        t = x.transpose(0, 1) if len(shape) == 3 else x.t().contiguous().t()
        _both(t, groups, w, b, dy.transpose(0, 1) if len(shape) == 3 else dy, "silu")
        ones = torch.ones((), device="cuda", dtype=dtype).expand(shape)
        _both(x, groups, w, b, ones, "silu")


def test_empty(gpu):
    for shape in ((0, 16), (3, 0, 16)):
        x = torch.empty(shape, device="cuda")
        w = torch.ones(16, device="cuda")
        y, mean, rstd = N.group_norm_forward(x, 4, w, w)
        assert y.shape == shape and mean.shape == (shape[0], 4)
        dx, dw, db = N.group_norm_backward(x, x, mean, rstd, 4, w, w)
        assert dx.shape == shape and not dw.any() and not db.any()


def test_nan_and_infinity_stay_in_their_group(gpu):
    for shape in ((20, 32), (4, 50, 32)):
        x, w, b, _ = _inputs(shape, F32, F32, 9)
        clean = N.group_norm(x, 4, w, b, act="relu")
        hurt = x.clone()
        hurt[1, ..., 3] = float("nan")
        hurt[2, ..., 30] = float("inf")
        y = N.group_norm(hurt, 4, w, b, act="relu")
        assert bool(y[1, ..., :8].isnan().all()) and bool(y[2, ..., 30].isnan().all())
        rest = torch.ones_like(x, dtype=torch.bool)
        rest[1, ..., :8] = False
        rest[2, ..., 24:] = False
        assert torch.equal(y[rest], clean[rest])


def test_same_bits_every_time(gpu):
    for shape in ((9000, 64), (2, 9000, 64)):
        x, w, b, dy = _inputs(shape, F32, F32, 10)
        first = None
        for _ in range(4):
            y, mean, rstd = N.group_norm_forward(x, 8, w, b, act="gelu")
            got = (y, mean, rstd, *N.group_norm_backward(dy, x, mean, rstd, 8, w, b, act="gelu"))
            first = first or got
            assert all(torch.equal(p, q) for p, q in zip(got, first))


@pytest.mark.parametrize("shape", [(12, 24), (3, 11, 24)])
@pytest.mark.parametrize("act", ["none", "silu", "gelu"])
def test_autograd_and_differences(gpu, shape, act):
    """Gradients against central differences of the 64-bit formula: the step's
    error is of the order of step^2 times a third derivative; 1e-4 of the scale
    covers it at a step of 1e-4, and the fp32 gradient is far closer."""
    x, w, b, dy = _inputs(shape, F32, F32, 11)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    N.group_norm(leaves[0], 4, leaves[1], leaves[2], 1e-5, act).backward(dy)

    def f(values):
        return float((Oracle(values[0], 4, values[1], values[2], 1e-5, act).y.view(shape) * dy.double()).sum())

    gen = torch.Generator().manual_seed(1)
    for k, leaf in enumerate(leaves):
        for i in torch.randint(leaf.numel(), (6,), generator=gen).tolist():
            at = [t.double() for t in (x, w, b)]
            lo, hi = [], []
            for sign, out in ((1, hi), (-1, lo)):
                moved = [t.clone() for t in at]
                moved[k].view(-1)[i] += sign * 1e-4
                out.append(f(moved))
            slope = (hi[0] - lo[0]) / 2e-4
            scale = float(leaf.grad.abs().max()) + 1.0
            assert abs(slope - float(leaf.grad.view(-1)[i])) <= 1e-4 * scale
    # only the parameters need gradients
    w2 = w.clone().requires_grad_(True)
    N.group_norm(x, 4, w2, b, 1e-5, act).backward(dy)
    assert torch.equal(w2.grad, leaves[1].grad)
    layer = N.GroupNorm(4, 24, act=act, device="cuda")
    assert torch.equal(layer(x), N.group_norm(x, 4, torch.ones_like(w), torch.zeros_like(b), 1e-5, act))


def test_other_stream_and_captured_graph(gpu):
    for shape in ((2000, 128), (3, 900, 128)):
        x, w, b, dy = _inputs(shape, F32, F32, 12)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            y, mean, rstd = N.group_norm_forward(x, 8, w, b, act="silu")
            grads = N.group_norm_backward(dy, x, mean, rstd, 8, w, b, act="silu")
        torch.cuda.current_stream().wait_stream(side)
        o = Oracle(x, 8, w, b, 1e-5, "silu")
        o.check_forward(y, mean, rstd)
        o.check_backward(dy, *grads)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y, mean, rstd = N.group_norm_forward(x, 8, w, b, act="silu")
            grads = N.group_norm_backward(dy, x, mean, rstd, 8, w, b, act="silu")
        for seed in (21, 22):
            x2, _, _, dy2 = _inputs(shape, F32, F32, seed)
            x.copy_(x2)
            dy.copy_(dy2)
            for t in (y, mean, rstd, *grads):
                t.fill_(float("nan"))
            graph.replay()
            o = Oracle(x, 8, w, b, 1e-5, "silu")
            o.check_forward(y, mean, rstd)
            o.check_backward(dy, *grads)


def test_offsets_past_32_bits(gpu):
    """More than 2^31 values (4.3 GB in bf16): equal rows give equal outputs everywhere."""
    rows, c = 8_400_001, 256
    line = torch.randn(c, device="cuda").to(BF16)
    x = line.expand(rows, c).contiguous()
    y, mean, rstd = N.group_norm_forward(x, 8)
    assert bool((y[::70001] == y[0]).all()) and torch.equal(y[rows - 1], y[0])
    Oracle(x[rows - 3:], 8, None, None, 1e-5, "none").check_forward(y[rows - 3:])
    del y
    dx, _, _ = N.group_norm_backward(x, x, mean, rstd, 8)
    assert torch.equal(dx[rows - 1], dx[0]) and bool((dx[::70001] == dx[0]).all())
    del dx
    whole = N.group_norm(x.view(1, rows, c), 8)
    assert torch.equal(whole[0, rows - 1], whole[0, 0]) and bool((whole[0, ::70001] == whole[0, 0]).all())


def _call(name, *args):
    L.call(name, *args, torch.cuda.current_stream().cuda_stream)


@pytest.mark.parametrize("shape,groups", [((500, 1, 64), 8), ((300, 5, 24), 6), ((7, 130, 40), 4), ((2, 6000, 64), 8)])
def test_outputs_in_the_place_of_inputs(gpu, shape, groups):
    """The C calls with y = x and dx = dy (every form), and with rows further apart than C."""
    n, steps, c = shape
    for pad in (0, 8):
        x, w, b, dy = _inputs((n, steps, c + pad), F32, F32, 14)
        o = Oracle(x[..., :c].contiguous(), groups, w[:c], b[:c], 1e-5, "silu")
        mean, rstd = torch.empty((2, n, groups), device="cuda").unbind(0)
        size = L.lib().tcc_group_norm_scratch_bytes(n, steps, c, groups, 1)
        size = max(size, L.lib().tcc_group_norm_scratch_bytes(n, steps, c, groups, 0), 256)
        scratch = torch.empty(size, dtype=torch.uint8, device="cuda")
        y, dx, beside = x.clone(), dy.clone(), [t[..., c:].clone() for t in (x, dy)]
        _call("tcc_group_norm_forward", y.data_ptr(), L.F32, c + pad, w.data_ptr(), b.data_ptr(), L.F32, y.data_ptr(),
              c + pad, mean.data_ptr(), rstd.data_ptr(), n, steps, c, groups, 1e-5, 2, scratch.data_ptr(), size)
        o.check_forward(y[..., :c].contiguous(), mean, rstd)
        dw, db = torch.empty_like(w[:c]), torch.empty_like(b[:c])
        _call("tcc_group_norm_backward", dx.data_ptr(), c + pad, x.data_ptr(), c + pad, L.F32, w.data_ptr(),
              b.data_ptr(), L.F32, mean.data_ptr(), rstd.data_ptr(), dx.data_ptr(), c + pad, dw.data_ptr(),
              db.data_ptr(), n, steps, c, groups, 2, scratch.data_ptr(), size)
        o.check_backward(dy[..., :c].contiguous(), dx[..., :c].contiguous(), dw, db)
        assert torch.equal(y[..., c:], beside[0]) and torch.equal(dx[..., c:], beside[1])


@pytest.mark.parametrize("shape,groups", [((500, 1, 64), 8), ((7, 130, 40), 4), ((2, 6000, 64), 8)])
def test_parts_of_the_backward(gpu, shape, groups):
    """Only dx, only one parameter's gradient: the same bits as all at once."""
    n, steps, c = shape
    x, w, b, dy = _inputs(shape, F32, F32, 15)
    _, mean, rstd = N.group_norm_forward(x, groups, w, b, act="gelu")
    dx, dw, db = N.group_norm_backward(dy, x, mean, rstd, groups, w, b, act="gelu")
    none_dx, dw2, db2 = N.group_norm_backward(dy, x, mean, rstd, groups, w, b, act="gelu", need_dx=False)
    assert none_dx is None and torch.equal(dw, dw2) and torch.equal(db, db2)
    size = L.lib().tcc_group_norm_scratch_bytes(n, steps, c, groups, 1)
    scratch = torch.empty(max(size, 256), dtype=torch.uint8, device="cuda")
    for want in ((dx, None, None), (None, dw, None), (dx, None, db)):
        got = [None if t is None else torch.empty_like(t) for t in want]
        ptr = [None if t is None else t.data_ptr() for t in got]
        _call("tcc_group_norm_backward", dy.data_ptr(), c, x.data_ptr(), c, L.F32, w.data_ptr(), b.data_ptr(), L.F32,
              mean.data_ptr(), rstd.data_ptr(), ptr[0], c, ptr[1], ptr[2], n, steps, c, groups, 3, scratch.data_ptr(),
              size)
        for t, v in zip(got, want):
            assert t is None or torch.equal(t, v)


@pytest.mark.parametrize("n,steps,c,groups", [(5000, 4, 64, 8), (3000, 40, 24, 3), (40, 2000, 64, 8), (1200, 1, 2048, 1)])
def test_many_samples(gpu, n, steps, c, groups):
    """More samples than CTAs run at once, in every form."""
    shape = (n, c) if steps == 1 else (n, steps, c)
    x, w, b, dy = _inputs(shape, F32, F32, 16)
    _both(x, groups, w, b, dy, "silu")
