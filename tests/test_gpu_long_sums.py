"""Long sums of the training operators against their exact values.

The values are constants that round the same way at every step of a long chain of fp32
additions: c = 1 + 2^-14 - 2^-23 added to a sum in [1024, 2048), whose unit is 2^-13, becomes
1 and loses 2^-14, that is 1024 u (u = 2^-24).  A chain of 2,000 such additions is off by
some 500 u; the operators' chains, 192 operations at most, stay below 192 u."""
import pytest
import torch

from tcc_b200 import embedding as E
from tcc_b200 import norm as N
from test_gpu_group_norm import D, F32, U, Oracle

pytestmark = pytest.mark.gpu

C_DOWN = 1 + 2.0 ** -14 - 2.0 ** -23


def test_split_form_sums(gpu):
    """2,027 rows to each of 444 CTAs, 255 channels: a thread a channel."""
    shape = (1, 900_001, 255)
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(shape, generator=gen, device="cuda")
    w, b = (1 + 0.3 * torch.randn(255, generator=gen, device="cuda") for _ in range(2))
    _, mean, rstd = N.group_norm_forward(x, 1, w, b)
    dy = torch.full(shape, C_DOWN, device="cuda")
    dx, dw, db = N.group_norm_backward(dy, x, mean, rstd, 1, w, b)
    want = shape[1] * float(dy[0, 0, 0])
    assert float((db.double() - want).abs().max()) <= (D + 1) * U * want
    o = Oracle(x, 1, w, b, 1e-5, "none")
    o.check_backward(dy, dx, dw, db)


def test_resident_form_sums(gpu):
    """2,100 samples to each of 1,184 CTAs."""
    n, steps, c = 1184 * 2100 + 1, 33, 8
    x = torch.randn((n, steps, c), device="cuda")
    w, b = torch.ones(c, device="cuda"), torch.zeros(c, device="cuda")
    _, mean, rstd = N.group_norm_forward(x, 1, w, b)
    dy = torch.full((n, steps, c), C_DOWN, device="cuda")
    _, _, db = N.group_norm_backward(dy, x, mean, rstd, 1, w, b, need_dx=False)
    want = n * steps * float(dy[0, 0, 0])
    assert float((db.double() - want).abs().max()) <= (D + 1) * U * want
    dx, dw, db2 = N.group_norm_backward(dy, x, mean, rstd, 1, w, b)
    assert torch.equal(db, db2)
    h = (x.double() - mean.double()[..., None]) * rstd.double()[..., None]
    want = (h * C_DOWN).sum((0, 1))
    size = (h.abs() * C_DOWN).sum((0, 1))
    assert bool(((dw.double() - want).abs() <= D * U * size).all())


def test_rows_form_sums(gpu):
    """4,000 rows to a thread, in two levels of 64; three values a row."""
    n, c = 592 * 64 * 4000 + 5, 3
    x = torch.zeros((n, c), device="cuda")
    stats = torch.zeros((n, 1), device="cuda")
    dy = torch.full((n, c), C_DOWN, device="cuda")
    w, b = torch.ones(c, device="cuda"), torch.zeros(c, device="cuda")
    _, _, db = N.group_norm_backward(dy, x, stats, stats, 1, w, b, need_dx=False)
    want = n * float(dy[0, 0])
    assert float((db.double() - want).abs().max()) <= (D + 1) * U * want


def test_split_form_moments(gpu):
    """Rows of one sign and the other in turn, 32,000 to each of 444 CTAs: every block of
    four adds 4 + 2^-10 to the sum of squares, which from 16,384 on loses the 2^-10."""
    steps, c = 444 * 32_000, 129
    a = 1 + 2.0 ** -13
    x = torch.full((1, steps, c), a, device="cuda")
    x[:, 1::2] = -a
    _, mean, rstd = N.group_norm_forward(x, 1, eps=0.0)
    assert abs(float(mean)) <= D * U * a
    assert abs(float(rstd) * a - 1) <= D * U * 2  # |x| is the deviation: A rstd = 1


@pytest.mark.parametrize("width", [1024, 257])
def test_run_of_one_row(gpu, width):
    """1.2 M gradient rows of one table row: 2,344 ranges of 512 to be joined, one thread a column.
    A range's own sum is exact but for the 2^-23 of each value."""
    n = 1_200_000
    idx = torch.full((n,), 3, device="cuda")
    grad = torch.full((n, width), 1 + 2.0 ** -14 - 2.0 ** -23, device="cuda")
    out = E.embedding_backward(grad, idx, 7)
    want = n * float(grad[0, 0])
    assert float((out[3].double() - want).abs().max()) <= (D + 1) * U * want
    assert not out[:3].any() and not out[4:].any()
