"""Global gradient norm and clipping (tcc_b200.clip) against 64-bit torch.

Tolerances: a pack of at most 8 squares in fp32 (8 u, u = 2^-24), 64-bit sums
(nothing at these sizes), half of it after the root, one rounding of the norm:
|norm - exact| <= 6 u exact.  The factor adds the sum with eps, the division and
the product: relative 6 u + 3 u, then one rounding to the gradient's type."""
import pytest
import torch

from tcc_b200 import clip as K

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TINY = {F32: 2.0 ** -149, F16: 2.0 ** -24, BF16: 2.0 ** -133}


def _exact(grads):
    return float(torch.stack([g.double().square().sum() for g in grads]).sum().sqrt())


def _params(shapes, dtypes, seed, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for i, s in enumerate(shapes):
        p = torch.zeros(s, dtype=dtypes[i % len(dtypes)], device="cuda")
        p.grad = (torch.randn(s, generator=gen, device="cuda") * scale).to(p.dtype)
        out.append(p)
    return out


def _check_clip(params, max_norm, call=None):
    before = [p.grad.clone() for p in params]
    norm = _exact(before)
    got = K.clip_grad_norm_(params, max_norm) if call is None else call()
    assert got.shape == () and got.dtype == F32
    assert abs(float(got) - norm) <= 6 * U * norm + TINY[F32]
    f = min(1.0, max_norm / (norm + 1e-6))
    for p, g in zip(params, before):
        want = g.double() * f
        if f == 1.0:
            assert torch.equal(p.grad, g)
        else:
            tol = (9 * U + torch.finfo(g.dtype).eps / 2) * want.abs() + TINY[g.dtype]
            assert bool(((p.grad.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("dtypes", [(F32,), (BF16,), (F16,), (F32, BF16, F16)])
@pytest.mark.parametrize("shapes", [[(1,)], [(5,), (3,)], [(100, 256), (256, 47)], [(8192,), (8193,), (16385,), (7,)],
                                    [(1000, 300), (), (0,), (4, 0, 3), (17, 5, 3)], [(3_000_017,)]])
def test_sizes_and_types(gpu, dtypes, shapes):
    _check_clip(_params(shapes, dtypes, 1), 1.0)
    _check_clip(_params(shapes, dtypes, 2), 1e9)  # above the norm: nothing changes
    _check_clip(_params(shapes, dtypes, 3), 0.0)
    grads = [p.grad for p in _params(shapes, dtypes, 4)]
    assert abs(float(K.grad_norm(grads)) - _exact(grads)) <= 6 * U * _exact(grads)


# one table of tensors to a launch, the next size of table, several launches
@pytest.mark.parametrize("count", [32, 33, 128, 129, 480, 481, 1500])
def test_many_tensors(gpu, count):
    shapes = [((i * 37) % 211,) for i in range(count)]
    _check_clip(_params(shapes, (F32, BF16), count), 2.0)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_alignment_and_orders(gpu, dtype):
    gen = torch.Generator(device="cuda").manual_seed(5)
    base = torch.randn(40000, generator=gen, device="cuda").to(dtype)
    keep = base.clone()
    spans = [(0, 1), (1, 2), (3, 9), (13, 8), (24, 1000), (1025, 9000), (10027, 16400), (26431, 3)]
    params = []
    for at, n in spans:
        p = torch.zeros(n, dtype=dtype, device="cuda")
        p.grad = base[at:at + n]
        params.append(p)
    _check_clip(params, 0.5)
    used = torch.zeros(40000, dtype=torch.bool, device="cuda")
    for at, n in spans:
        used[at:at + n] = True
    assert torch.equal(base[~used], keep[~used])  # nothing beside the tensors is touched
    p = torch.zeros((30, 20, 10), dtype=dtype, device="cuda").permute(2, 0, 1)
    p.grad = torch.randn((30, 20, 10), generator=gen, device="cuda").to(dtype).permute(2, 0, 1)
    _check_clip([p], 1.0)


@pytest.mark.parametrize("value", [1e-30, 1e-20, 1e15, 1e25, 3e37])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_squares_beyond_the_range_of_fp32(gpu, value, dtype):
    grads = [torch.full((10,), value, device="cuda").to(dtype), torch.full((3,), value, device="cuda").to(dtype)]
    want = _exact(grads)
    assert abs(float(K.grad_norm(grads)) - want) <= 6 * U * want


def test_nonfinite(gpu):
    for bad in (float("nan"), float("inf"), -float("inf")):
        ps = _params([(1000,), (10,)], (F32,), 6)
        ps[0].grad[999] = bad
        before = [p.grad.clone() for p in ps]
        with pytest.raises(RuntimeError, match="finite"):
            K.clip_grad_norm_(ps, 1.0, error_if_nonfinite=True)
        assert all(torch.equal(p.grad.nan_to_num(7), g.nan_to_num(7)) for p, g in zip(ps, before))
        norm = float(K.clip_grad_norm_(ps, 1.0))
        assert norm != norm if bad != bad else norm == float("inf")
        if bad != bad:
            assert bool(ps[1].grad.isnan().all())
        else:
            assert not ps[1].grad.any() and bool(ps[0].grad[999].isnan())
    ps = _params([(100,)], (F32,), 7)
    _check_clip(ps, 1.0, lambda: K.clip_grad_norm_(ps, 1.0, error_if_nonfinite=True))


def test_without_gradients_and_given_norm(gpu):
    assert float(K.clip_grad_norm_([torch.zeros(3, device="cuda")], 1.0)) == 0.0
    assert float(K.grad_norm([])) == 0.0
    p = torch.zeros(0, device="cuda")
    p.grad = torch.zeros(0, device="cuda")
    assert float(K.clip_grad_norm_(p, 1.0)) == 0.0
    ps = _params([(50,), (7, 3)], (F32,), 8)
    ps.insert(1, torch.zeros(4, device="cuda"))  # no gradient: passed over
    real = [ps[0], ps[2]]
    _check_clip(real, 1.0, lambda: K.clip_grad_norm_(iter(ps), 1.0))
    # parts of the parameters on several ranks: the norm is combined by the caller
    grads = [p.grad.clone() for p in real]
    total = torch.full((), 10.0, device="cuda")
    K.clip_grads_with_norm_([p.grad for p in real], 2.5, total)
    for p, g in zip(real, grads):
        assert bool(((p.grad - g * 0.25).abs() <= 1e-6 * g.abs()).all())


def test_refusals(gpu):
    g = torch.zeros(64, device="cuda")
    a, b = torch.zeros(40, device="cuda"), torch.zeros(40, device="cuda")
    a.grad, b.grad = g[:40], g[24:]
    with pytest.raises(RuntimeError, match="share memory"):
        K.clip_grad_norm_([a, b], 1.0)
    assert float(K.grad_norm([a.grad, b.grad])) == 0.0  # reading both is fine
    with pytest.raises(ValueError, match="block of memory"):
        K.grad_norm([torch.zeros((4, 8), device="cuda")[:, :5]])
    with pytest.raises(ValueError, match="block of memory"):
        K.grad_norm([torch.zeros((), device="cuda").expand(5)])
    with pytest.raises(TypeError):
        K.grad_norm([torch.zeros(4, dtype=torch.float64, device="cuda")])
    with pytest.raises(ValueError):
        K.grad_norm([torch.zeros(4)])
    with pytest.raises(ValueError):
        K.grad_norm([torch.zeros((4, 4), device="cuda").to_sparse()])
    with pytest.raises(RuntimeError, match="max_norm"):
        K.clip_grad_norm_([_params([(3,)], (F32,), 1)[0]], -1.0)
    with pytest.raises(RuntimeError, match="max_norm"):
        K.clip_grad_norm_([_params([(3,)], (F32,), 1)[0]], float("nan"))
    with pytest.raises(ValueError):
        K.clip_grads_with_norm_([g], 1.0, torch.ones((), dtype=torch.float64, device="cuda"))


def test_same_bits_and_version(gpu):
    ps = _params([(100003,), (77,)], (F32, BF16), 9)
    grads = [p.grad for p in ps]
    first = K.grad_norm(grads)
    for _ in range(4):
        assert torch.equal(K.grad_norm(grads), first)
    before = grads[0]._version
    K.clip_grad_norm_(ps, 1.0)
    assert grads[0]._version > before  # a graph that saved the gradient notices


def test_other_stream_and_captured_graph(gpu):
    ps = _params([(1000, 100), (33,)], (F32, BF16), 10)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _check_clip(ps, 1.0)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = K.clip_grad_norm_(ps, 1.0)

    def replay():
        graph.replay()
        return norm

    for seed in (1, 2):
        for p, q in zip(ps, _params([(1000, 100), (33,)], (F32, BF16), seed)):
            p.grad.copy_(q.grad)
        _check_clip(ps, 1.0, replay)


def test_offsets_past_32_bits(gpu):
    """One gradient of more than 2^32 elements (8.6 GB in bf16), scaled to its far end."""
    n = (1 << 32) + 4097
    p = torch.empty(n, dtype=BF16, device="cuda")
    p.grad = torch.zeros(n, dtype=BF16, device="cuda")
    p.grad[0], p.grad[1 << 31], p.grad[n - 1] = 3.0, 4.0, 12.0
    assert float(K.clip_grad_norm_(p, 6.5)) == 13.0
    assert [float(p.grad[i]) for i in (0, 1 << 31, n - 1)] == [1.5, 2.0, 6.0]


@pytest.mark.parametrize("shapes", [[(50,)], [(300, 300), (7,)]])
def test_zero_gradients(gpu, shapes):
    for max_norm, eps in ((1.0, 1e-6), (0.0, 1e-6), (0.0, 0.0), (1.0, 0.0)):
        ps = _params(shapes, (F32,), 1, scale=0.0)
        assert float(K.clip_grad_norm_(ps, max_norm, eps=eps)) == 0.0
        assert not any(p.grad.any() or p.grad.isnan().any() for p in ps)


def test_limit_of_the_one_launch_form(gpu):
    """One byte range and one tensor more than what one launch takes."""
    for shapes in ([(49152,)], [(49152,), (1,)], [(1536,)] * 32, [(1489,)] * 33):
        _check_clip(_params(shapes, (F32,), 11), 1.0)


def test_inference_tensors(gpu):
    with torch.inference_mode():
        g = torch.full((100,), 2.0, device="cuda")
    total = torch.full((), 20.0, device="cuda")
    K.clip_grads_with_norm_([g], 5.0, total)
    assert bool(((g - 0.5).abs() < 1e-6).all())
