"""Group norm over more than 2^31 values (4.3 GB in bf16), every form forward and backward, against
the 64-bit formula: samples from both ends and from both sides of 2^31, and the sums over all.
Bounds of test_gpu_group_norm."""
import pytest
import torch

from tcc_b200 import norm as N
from test_gpu_group_norm import BF16, D, F32, TINY, U, Oracle, _half_step

pytestmark = pytest.mark.gpu


def _picks(count, at):
    return torch.tensor(sorted({0, 1, at - 1, at, at + 1, count // 2, count - 2, count - 1}), device="cuda")


# rows form, resident form, split form of many samples
@pytest.mark.parametrize("n,steps,c,groups", [(8_400_001, 1, 256, 8), (65_001, 130, 256, 8), (1_050_001, 1, 2048, 1)])
def test_many_samples(gpu, n, steps, c, groups):
    gen = torch.Generator(device="cuda").manual_seed(n)
    x = torch.empty((n, steps, c), device="cuda", dtype=BF16).normal_(generator=gen)
    dy = torch.empty((n, steps, c), device="cuda", dtype=BF16).normal_(generator=gen)
    w, b = (1 + 0.3 * torch.randn(c, generator=gen, device="cuda") for _ in range(2))
    y, mean, rstd = N.group_norm_forward(x, groups, w, b)
    picks = _picks(n, 2 ** 31 // (steps * c))
    o = Oracle(x[picks], groups, w, b, 1e-5, "none")
    o.check_forward(y[picks].contiguous(), mean[picks], rstd[picks])
    del y
    dx, dw, db = N.group_norm_backward(dy, x, mean, rstd, groups, w, b)
    o.check_backward(dy[picks], dx[picks].contiguous(), None, None)
    del dx
    # the parameters' gradients: 64-bit sums, with the kernels' fp32 statistics, over a part at a time
    want_w, want_b, size_w, size_b = (torch.zeros(c, device="cuda", dtype=torch.float64) for _ in range(4))
    for at in range(0, n, 32768 // steps):
        part = slice(at, min(n, at + 32768 // steps))
        m, r = (t[part].double()[:, None, :, None] for t in (mean, rstd))
        shape = (m.shape[0], steps, groups, c // groups)
        d = dy[part].double().view(shape)
        dh = d * ((x[part].double().view(shape) - m) * r)
        want_w += dh.sum((0, 1)).view(-1)
        size_w += dh.abs().sum((0, 1)).view(-1)
        want_b += d.sum((0, 1)).view(-1)
        size_b += d.abs().sum((0, 1)).view(-1)
    # h is a difference and a product: 2 u of |x| + |mean| beside the sums' D u
    assert bool(((db.double() - want_b).abs() <= D * U * size_b).all())
    assert bool(((dw.double() - want_w).abs() <= (D + 8) * U * size_w).all())


def test_one_sample(gpu):
    """Rows are one line or its negative, so that the statistics over all 8.4 M are known exactly."""
    rows, c, groups = 8_400_001, 256, 8
    gen = torch.Generator(device="cuda").manual_seed(1)
    line, slope = ((0.7 + torch.randn(c, generator=gen, device="cuda")).to(BF16) for _ in range(2))
    s, t = (torch.rand(rows, generator=gen, device="cuda") < p for p in (0.6, 0.3))  # rows of the negative

    def signed(v, minus):
        out = v.expand(1, rows, c).contiguous()
        out[0, minus] = -v
        return out
    x, dy = signed(line, s), signed(slope, t)
    ns, nt, nst = (1 - 2 * float(m.double().mean()) for m in (s, t, s ^ t))
    a, g = line.double().view(groups, -1), slope.double().view(groups, -1)
    mean = ns * a.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt((a * a).mean(1, keepdim=True) - mean * mean + 1e-5)
    away = a.abs().mean(1, keepdim=True) * rstd
    # means over the sample of dz, of dz h
    m1 = nt * g.mean(1, keepdim=True)
    m2 = rstd * (nst * (a * g).mean(1, keepdim=True) - mean * nt * g.mean(1, keepdim=True))
    h_most = (a.abs() + mean.abs()) * rstd

    y, got_mean, got_rstd = N.group_norm_forward(x, groups)
    assert bool(((got_mean.double().view(-1, 1) - mean).abs() <= D * U * a.abs().mean(1, keepdim=True)).all())
    assert bool(((got_rstd.double().view(-1, 1) / rstd - 1).abs() <= D * U * (1 + away)).all())
    picks = _picks(rows, 2 ** 31 // c)
    xs, ds = x[0, picks].double().view(-1, groups, c // groups), dy[0, picks].double().view(-1, groups, c // groups)
    h = (xs - mean) * rstd
    eh = D * U * (away + h.abs() + 1)
    err = (y[0, picks].double().view_as(h) - h).abs()
    assert bool((err <= eh + 12 * U * h.abs() + _half_step(BF16) * h.abs() + TINY[BF16]).all())
    del y
    w, b = torch.ones(c, device="cuda"), torch.zeros(c, device="cuda")
    dx, dw, db = N.group_norm_backward(dy, x, got_mean, got_rstd, groups, w, b)
    want = rstd * (ds - m1 - h * m2)
    eh_most = D * U * (away + h_most + 1)
    e1 = D * U * g.abs()
    e2 = g.abs() * eh_most + D * U * g.abs() * h_most
    tol = rstd * (e1 + e1.mean(1, keepdim=True) + h.abs() * e2.mean(1, keepdim=True)
                  + eh * (g.abs() * h_most).mean(1, keepdim=True)) \
        + D * U * (1 + away) * want.abs() + _half_step(BF16) * want.abs() + TINY[BF16]
    assert bool(((dx[0, picks].double().view_as(want) - want).abs() <= tol).all())
    want_b = rows * nt * g
    assert bool(((db.double().view_as(g) - want_b).abs() <= D * U * rows * g.abs() + TINY[F32]).all())
    want_w = rows * rstd * g * (nst * a - nt * mean)
    assert bool(((dw.double().view_as(g) - want_w).abs() <= rows * (g.abs() * eh_most + D * U * g.abs() * h_most)).all())
