"""Refusals of the training operators' entry points, before any GPU call (CPU only)."""
import ctypes as C

import pytest
import torch

from tcc_b200 import _lib as L
from tcc_b200 import clip, embedding, norm


@pytest.fixture(scope="module")
def lib():
    from tcc_b200 import build
    build.build()
    return L.lib()


P = 0x10000  # an aligned address that no refused call reads


def test_embedding_refusals(lib):
    good = dict(table=P, tt=L.F32, ldt=8, rows=10, idx=P, it=L.I64, n=4, pad=L.NO_PADDING, scale=1.0, out=P, ot=L.F32,
                ldo=8, F=8)

    def forward(**kw):
        return lib.tcc_embedding_forward(*{**good, **kw}.values(), None, None)

    def backward(scratch=P, nbytes=1 << 30, **kw):
        a = {**good, **kw}
        return lib.tcc_embedding_backward(a["out"], a["ot"], a["ldo"], a["idx"], a["it"], a["n"], a["pad"], a["scale"],
                                          a["table"], a["tt"], a["ldt"], a["rows"], a["F"], scratch, nbytes, None, None)

    for bad in (dict(tt=3), dict(ot=7), dict(tt=L.F32, ot=L.BF16), dict(tt=L.F16, ot=L.BF16), dict(it=2), dict(F=0),
                dict(F=(1 << 20) + 1, ldt=1 << 21, ldo=1 << 21), dict(ldt=7), dict(ldo=7), dict(n=1 << 31),
                dict(rows=1 << 31), dict(idx=None), dict(out=None), dict(table=None), dict(table=P + 2),
                dict(idx=P + 4), dict(out=P + 1)):
        assert forward(**bad) == 1, bad
        assert backward(**bad) == 1, bad
        assert lib.tcc_last_error().startswith(b"tcc_embedding_backward")
    assert forward(n=0) == 0  # nothing to do
    assert backward(rows=0) == 0
    assert backward(n=5000, scratch=None) == 1
    assert backward(n=5000, scratch=P + 16) == 1
    assert backward(n=5000, nbytes=8) == 6  # TCC_ERR_CAPACITY
    assert lib.tcc_embedding_backward_scratch_bytes(200, 1 << 20, 64) == 0  # few indices: none
    assert lib.tcc_embedding_backward_scratch_bytes(1 << 20, 1 << 20, 64) > 8 << 20


def test_group_norm_refusals(lib):
    fwd = dict(x=P, type=L.F32, ldx=32, w=P, b=P, pt=L.F32, y=P, ldy=32, mean=P, rstd=P, N=4, S=50, C=32, G=4, eps=1e-5,
               act=0, scratch=P, nbytes=1 << 30)

    def forward(**kw):
        return lib.tcc_group_norm_forward(*{**fwd, **kw}.values(), None)

    bwd = dict(dy=P, lddy=32, x=P, ldx=32, type=L.F32, w=P, b=P, pt=L.F32, mean=P, rstd=P, dx=P, lddx=32, dw=P, db=P,
               N=4, S=50, C=32, G=4, act=0, scratch=P, nbytes=1 << 30)

    def backward(**kw):
        return lib.tcc_group_norm_backward(*{**bwd, **kw}.values(), None)

    both = (dict(type=5), dict(pt=-1), dict(act=4), dict(act=-1), dict(G=0), dict(C=0), dict(G=5), dict(x=None),
            dict(x=P + 2), dict(ldx=31), dict(N=1 << 31), dict(S=1 << 31), dict(w=P + 2), dict(b=P + 1),
            dict(S=1 << 20, scratch=None), dict(S=1 << 20, scratch=P + 8), dict(C=(1 << 20) + 4, ldx=1 << 21, ldy=1 << 21))
    for bad in both + (dict(y=None), dict(ldy=31), dict(eps=-1.0), dict(mean=None), dict(rstd=None)):
        assert forward(**bad) == 1, bad
    for bad in both[:-1] + (dict(dy=None), dict(lddy=31), dict(lddx=31), dict(mean=None), dict(rstd=None),
                            dict(dw=P + 2), dict(db=P + 2)):
        assert backward(**bad) == 1, bad
    assert forward(S=1 << 20, nbytes=16) == 6 and backward(S=1 << 20, nbytes=16) == 6
    assert forward(N=0) == 0 and forward(S=0) == 0
    # rows by themselves and samples that stay on chip, forward: none; backward: no more for more samples
    assert lib.tcc_group_norm_scratch_bytes(1000, 1, 256, 8, 0) == 0
    assert lib.tcc_group_norm_scratch_bytes(64, 517, 100, 10, 0) == 0
    for steps in (1, 4):
        few, many = (lib.tcc_group_norm_scratch_bytes(n, steps, 256, 8, 1) for n in (10_000, 10_000_000))
        assert few == many < 8 << 20


def test_clip_refusals(lib):
    def table(*rows):
        t = (L.Tensor * max(len(rows), 1))()
        for i, (data, n, kind) in enumerate(rows):
            t[i].data, t[i].n, t[i].type = data, n, kind
        return C.cast(t, C.c_void_p), len(rows), t

    def clip_call(rows, max_norm=1.0, eps=1e-6, out=P, scratch=P, nbytes=1 << 20):
        p, n, keep = table(*rows)
        return lib.tcc_clip_grad_norm(p, n, max_norm, eps, out, scratch, nbytes, None)

    one = (P, 100, L.F32)
    for bad in ([(P, 100, 9)], [(None, 100, L.F32)], [(P + 2, 100, L.F32)], [(P + 1, 100, L.BF16)],
                [(P, 1 << 47, L.F32)]):
        assert clip_call(bad) == 1
    assert clip_call([one, (P + 396, 10, L.F32)]) == 1 and b"share memory" in lib.tcc_last_error()
    assert clip_call([(P + 396, 10, L.F32), one]) == 1
    assert clip_call([one, one]) == 1
    large = (P, 1 << 20, L.F32)
    for kw in (dict(max_norm=-1.0), dict(max_norm=float("nan")), dict(eps=-1.0), dict(out=None), dict(scratch=None),
               dict(scratch=P + 8)):
        assert clip_call([large], **kw) == 1, kw
    assert clip_call([large], nbytes=8) == 6
    assert lib.tcc_clip_grad_norm(None, 2, 1.0, 1e-6, P, P, 1 << 20, None) == 1
    p, n, keep = table(one)
    assert lib.tcc_grad_norm(p, n, None, P, 1 << 20, None) == 1
    assert lib.tcc_clip_grads_with_norm(p, n, None, 1.0, 1e-6, None) == 1
    assert C.sizeof(L.Tensor) == 24 and L.Tensor.type.offset == 16


def test_python_refusals():
    t, i = torch.zeros(4, 6), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="CUDA"):
        embedding.embedding(t, i)
    with pytest.raises(TypeError):
        embedding.embedding(t.double(), i)
    with pytest.raises(ValueError, match="CUDA"):
        embedding.embedding_backward(torch.zeros(3, 6), i, 4)
    with pytest.raises(ValueError, match="CUDA"):
        norm.group_norm(t, 2)
    with pytest.raises(TypeError):
        norm.group_norm(t.double(), 2)
    with pytest.raises(ValueError, match="act"):
        norm.GroupNorm(2, 6, act="tanh")
    with pytest.raises(ValueError, match="divide"):
        norm.GroupNorm(4, 6)
    with pytest.raises(ValueError, match="CUDA"):
        clip.grad_norm([t])
    with pytest.raises(TypeError):
        clip.grad_norm([t.double()])
    assert float(clip.grad_norm([])) == 0.0


def test_calls_run_on_the_tensors_device(monkeypatch):
    """With another device current, the call runs inside a guard for the tensors' device,
    on that device's current stream; no guard where it is current (fakes, no GPU)."""
    from tcc_b200 import _args
    log = []

    class Guard:
        def __init__(self, device):
            log.append(("guard", device.index))

        def __enter__(self):
            log.append("in")

        def __exit__(self, *exc):
            log.append("out")

    monkeypatch.setattr(torch.cuda, "device", Guard)
    monkeypatch.setattr(_args, "_current_device", lambda: 0)
    monkeypatch.setattr(_args, "_raw_stream", lambda index: 100 + index)
    monkeypatch.setitem(_args._bound, "fake", lambda *args: log.append(args) or 0)
    _args.launch(torch.device("cuda", 1), "fake", 7)
    assert log == [("guard", 1), "in", (7, 101), "out"]
    log.clear()
    _args.launch(torch.device("cuda", 0), "fake", 8)
    assert log == [(8, 100)]
    monkeypatch.setitem(_args._bound, "fake", lambda *args: 1)
    with pytest.raises(L.TccError):
        _args.launch(torch.device("cuda", 1), "fake")


def test_rows_of_strides():
    from tcc_b200._args import rows_of
    t = torch.zeros(6, 5, 8)
    assert rows_of(t, 8) == (t, 8)
    part = t[..., 2:6]
    same, ld = rows_of(part, 4)
    assert same is part and ld == 8
    for other in (t.transpose(0, 1)[..., :4], t[:, ::2, :4][..., ::2], torch.zeros(4).expand(3, 5, 4), t[:, :3, :4]):
        copy, ld = rows_of(other, other.shape[-1])
        assert copy.is_contiguous() and ld == other.shape[-1] and torch.equal(copy, other)
    one = t[:1, :1, ::2]  # a single row: only its values' stride counts
    copy, ld = rows_of(t[:1, 1:2, :4], 4)
    assert ld == 4
    assert rows_of(one, 4)[0].is_contiguous()


@pytest.mark.parametrize("steps", [1, 2, 40])
@pytest.mark.parametrize("channels,groups", [(257, 1), (512, 1), (602, 1), (1024, 1), (1024, 2), (2048, 2), (2048, 1),
                                             (1040, 260)])
def test_norm_scratch_is_small_beside_the_input(lib, steps, channels, groups):
    """Wide groups of few rows: no row of parameter gradients per sample, whatever form the widths and
    pointers of a call lead to (512 channels of 2.4 M nodes took 10 GB)."""
    samples = 2_449_029
    for backward in (0, 1):
        got = lib.tcc_group_norm_scratch_bytes(samples, steps, channels, groups, backward)
        statistics = samples * groups * 8  # a mean and a deviation, or two sums, each
        # those, the parts of groups that CTAs of 256 values each see, and sums that do not grow with the samples
        parts = samples * groups * -(-channels // groups // 256) * 12
        assert got <= statistics + parts + (64 << 20), (got, backward)
