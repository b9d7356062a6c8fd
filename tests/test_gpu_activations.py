"""The activations behind the group norm alone, over a sweep of z against 64 bits.

With a weight of zero the bias is z exactly, so y = act(bias), and with dy = 1 and one row
dbias = act'(bias), each a single term.  u = 2^-24; the hardware's exponential and reciprocal
are off by 4 u and 2 u, every other operation by u of its result.

sigmoid s: exponential 4 u, sum and product 1 u each, reciprocal 2 u, and |z| u from the rounded
exponent: (10 + |z|) u of itself, 1 - s absolutely as much.
Phi of fp32 features: at most 6 u from coefficients, t and Horner's steps, reciprocal 2 u,
exponential 4 u, products 2 u, below 16 u; the rounded exponent, 1.5 z^2 u; the fit,
1.5 (1 + z^4) u: all of Phi(-|z|).  Phi(z) of z > 0 is one subtraction more.
Phi of 16-bit features: 4.2e-7, of which 0.75e-7 from the approximation, 1.6e-7 from fp32's
roundings (the published form emulated with correctly rounded operations is off by 2.3e-7),
0.6e-7 and 1.2e-7 from reciprocal and exponential.
Values below 2^-126 are flushed to zero, times |z| < 2^7."""
import math

import pytest
import torch

from tcc_b200 import norm as N

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
FLUSH = 2.0 ** -119
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _sweep(count):
    """Values of both signs up to 100, most between 2^-20 and 16; infinite and zero ones apart."""
    small = torch.logspace(-20, 4, count // 4, base=2.0, dtype=torch.float64)
    wide = torch.linspace(0, 100, count // 4, dtype=torch.float64)
    z = torch.cat([small, wide])
    return torch.cat([z, -z]).float().cuda()


def _exact(act, z):
    """(y, y', their error bounds for fp32 features, for 16-bit features before the rounding of y)."""
    a = z.abs()
    if act == "silu":
        s, rest = torch.sigmoid(z), torch.sigmoid(-z)
        y, d = z * s, s + z * s * rest
        es = (10 + a) * U * s
        fine = coarse = (a * es + U * y.abs(), es * (1 + a * rest) + a * s * (es + U) + 3 * U * d.abs())
    else:
        tail, phi = 0.5 * torch.erfc(a / math.sqrt(2)), torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        cdf = 0.5 * torch.erfc(-z / math.sqrt(2))
        y, d = z * cdf, cdf + z * phi
        e_cdf = U * ((16 + 1.5 * z ** 2 + 1.5 * (1 + z ** 4)) * tail + 2 * (z > 0))
        e_phi = a * phi * (8 + 1.5 * z * z) * U
        fine = (a * e_cdf + U * y.abs(), e_cdf + e_phi + U * d.abs())
        coarse = (a * 4.2e-7 + U * y.abs(), 4.2e-7 + e_phi + U * d.abs())
    return y, d, fine, coarse


def _run(z, act, dtype, per, steps):
    """y and act'(z) of each channel; `per` channels to a group."""
    c = z.numel() // per * per
    z = z[:c]
    gen = torch.Generator(device="cuda").manual_seed(c)
    x = torch.randn((1, steps, c), generator=gen, device="cuda").to(dtype)
    dy = torch.zeros((1, steps, c), device="cuda", dtype=dtype)
    dy[:, steps // 2] = 1
    w = torch.zeros(c, device="cuda")
    y, mean, rstd = N.group_norm_forward(x, c // per, w, z, act=act)
    assert torch.equal(y.nan_to_num(7.0), y[:, :1].expand_as(y).nan_to_num(7.0))
    _, _, db = N.group_norm_backward(dy, x, mean, rstd, c // per, w, z, act=act, need_dx=False)
    return z.double(), y[0, 0].double(), db.double()


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
# rows form in packs and value by value, several rows; resident form; split form
@pytest.mark.parametrize("count,per,steps", [(1 << 18, 8, 1), (1 << 18, 7, 1), (1 << 16, 2, 3), (1 << 9, 8, 50),
                                             (1 << 14, 16, 40)])
def test_sweep(gpu, act, dtype, count, per, steps):
    z, y, db = _run(_sweep(count), act, dtype, per, steps)
    want, slope, fine, coarse = _exact(act, z)
    e_y, e_d = fine if dtype == F32 else coarse
    half = 0.0 if dtype == F32 else torch.finfo(dtype).eps / 2
    tiny = FLUSH if dtype != F16 else 2.0 ** -24
    err = (y - want).abs()
    assert bool((err <= e_y + half * want.abs() + tiny).all()), float((err / (e_y + half * want.abs() + tiny)).max())
    err = (db - slope).abs()
    assert bool((err <= e_d + FLUSH).all()), float((err / (e_d + FLUSH)).max())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_ends(gpu, dtype):
    """Zero, the largest values and infinity: what torch gives."""
    z = torch.tensor([0.0, -0.0, 1e30, 3e38, float("inf"), float("nan"), 150.0, 40.0], device="cuda")
    for act, f in (("silu", torch.nn.functional.silu), ("gelu", torch.nn.functional.gelu)):
        _, y, _ = _run(z, act, dtype, 1, 1)
        assert torch.equal(y.float().nan_to_num(7.0), f(z).to(dtype).float().nan_to_num(7.0)), (act, y)
        _, y, _ = _run(torch.tensor([-1e30, -3e38, -150.0, -200.0], device="cuda"), act, dtype, 1, 1)
        assert not y.any()
