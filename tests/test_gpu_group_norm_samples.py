"""Group norm of many samples with wide groups (tcc_b200.norm): the backward keeps the
parameters' sums per CTA, not per sample.  Formula and bounds of test_gpu_group_norm."""
import pytest
import torch

from tcc_b200 import _lib as L
from tcc_b200 import norm as N
from test_gpu_group_norm import BF16, F16, F32, _both, _call, _inputs

pytestmark = pytest.mark.gpu


# groups in parts of several CTAs, one whole group, some and many groups to a CTA; sums by
# threads and by warps; each also with a last sample, a last part and a last CTA that are not full
@pytest.mark.parametrize("n,steps,c,groups,dtype", [
    (2001, 1, 2048, 1, F32), (1001, 2, 1030, 1, F32), (400, 40, 1025, 5, F32), (1001, 33, 1040, 260, F32),
    (903, 34, 1032, 86, F32), (1003, 33, 4096, 16, BF16), (700, 3, 5000, 2, F16), (901, 1, 2051, 7, BF16),
    (445, 35, 2100, 1050, F16), (1780, 1, 602, 1, F32), (1, 33, 65600, 1025, F32)])
def test_wide_groups(gpu, n, steps, c, groups, dtype):
    x, w, b, dy = _inputs((n, steps, c), dtype, F32, n + c)
    for act in ("none", "gelu"):
        _both(x, groups, w, b, dy, act)
    _both(x, groups, None, b, dy, "silu")


@pytest.mark.parametrize("n,steps,c,groups", [(1790, 255, 512, 8), (1781, 251, 520, 4), (1781, 2003, 64, 4)])
def test_long_samples(gpu, n, steps, c, groups):
    """Several rows of threads to a sample that does not stay on chip."""
    x, w, b, dy = _inputs((n, steps, c), F32, F32, 3)
    _both(x, groups, w, b, dy, "none")


def test_parts_of_the_backward(gpu):
    """Only dx, only one parameter's gradient: the same bits as all at once, every time."""
    n, steps, c, groups = 1501, 1, 2052, 2
    x, w, b, dy = _inputs((n, steps, c), F32, F32, 15)
    _, mean, rstd = N.group_norm_forward(x, groups, w, b, act="gelu")
    dx, dw, db = N.group_norm_backward(dy, x, mean, rstd, groups, w, b, act="gelu")
    for again in (N.group_norm_backward(dy, x, mean, rstd, groups, w, b, act="gelu") for _ in range(3)):
        assert all(torch.equal(p, q) for p, q in zip(again, (dx, dw, db)))
    none_dx, dw2, db2 = N.group_norm_backward(dy, x, mean, rstd, groups, w, b, act="gelu", need_dx=False)
    assert none_dx is None and torch.equal(dw, dw2) and torch.equal(db, db2)
    size = L.lib().tcc_group_norm_scratch_bytes(n, steps, c, groups, 1)
    scratch = torch.full((size + 256,), 77, dtype=torch.uint8, device="cuda")
    for want in ((dx, None, None), (None, dw, None), (dx, None, db)):
        got = [None if t is None else torch.empty_like(t) for t in want]
        ptr = [None if t is None else t.data_ptr() for t in got]
        _call("tcc_group_norm_backward", dy.data_ptr(), c, x.data_ptr(), c, L.F32, w.data_ptr(), b.data_ptr(), L.F32,
              mean.data_ptr(), rstd.data_ptr(), ptr[0], c, ptr[1], ptr[2], n, steps, c, groups, 3, scratch.data_ptr(),
              size)
        for t, v in zip(got, want):
            assert t is None or torch.equal(t, v)
        assert bool((scratch[size:] == 77).all())


def test_memory_of_a_backward(gpu):
    """512 channels in one group, 400,000 nodes: the call takes its outputs and a few MB."""
    n, c = 400_000, 512
    x = torch.randn((n, c), device="cuda").to(BF16)
    w, b = torch.ones(c, device="cuda"), torch.zeros(c, device="cuda")
    _, mean, rstd = N.group_norm_forward(x, 1, w, b)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    dx, dw, db = N.group_norm_backward(x, x, mean, rstd, 1, w, b)
    extra = torch.cuda.max_memory_allocated() - before - dx.numel() * 2
    assert extra < 64 << 20, extra


@pytest.mark.parametrize("n,steps,c,groups,dtype", [(2, 32, 1 << 20, 1 << 20, F32), (1, 17, 1 << 20, 1 << 20, BF16),
                                                    (1, 32, 524280, 524280, F32)])
def test_a_million_groups(gpu, n, steps, c, groups, dtype):
    """Every channel by itself, as many as a call takes: more groups than the row form's grid."""
    x, w, b, dy = _inputs((n, steps, c), dtype, F32, 5)
    _both(x, groups, w, b, dy, "none")
