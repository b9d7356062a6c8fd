"""What autograd sees of the training operators (CPU only: the launches are left out)."""
import pytest
import torch
from torch.autograd import forward_ad

from tcc_b200 import _lib as L
from tcc_b200 import embedding, gcn, minibatch, norm


@pytest.fixture
def no_launch(monkeypatch):
    """The operators on CPU tensors: types are checked, nothing is computed."""
    for module in (embedding, norm):
        monkeypatch.setattr(module, "type_code", lambda t, name: L.F32)
        monkeypatch.setattr(module, "launch", lambda *args: None)
    monkeypatch.setattr(norm, "_scratch_bytes", lambda *args: 0)


IDX = torch.tensor([2, 0, 1])
CALLS = [lambda t: embedding.embedding(t, IDX), lambda t: norm.group_norm(t, 2),
         lambda t: norm.group_norm(torch.ones(4, 6), 2, weight=t[0]),
         lambda t: norm.group_norm(torch.ones(4, 6), 2, bias=t[0]), norm.GroupNorm(3, 6)]


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("grad_mode", [False, True])
def test_forward_mode_is_refused(no_launch, call, requires_grad, grad_mode):
    """A dual tensor never gives an output without a tangent, which would read as a derivative of zero."""
    t = torch.randn(4, 6, requires_grad=requires_grad)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad_mode):
        with pytest.raises((RuntimeError, NotImplementedError), match="(?i)forward"):
            call(forward_ad.make_dual(t, torch.ones(4, 6)))
        assert forward_ad.unpack_dual(call(torch.randn(4, 6))).tangent is None  # one without: as outside
    with torch.no_grad():
        assert not call(t).requires_grad


@pytest.mark.parametrize("call", CALLS)
def test_reverse_mode_takes_the_functions_path(no_launch, call):
    assert call(torch.randn(4, 6, requires_grad=True)).requires_grad
    assert isinstance(call, norm.GroupNorm) or not call(torch.randn(4, 6)).requires_grad


@pytest.mark.parametrize("call", CALLS[:2])
def test_functional_transforms_are_refused(no_launch, call):
    t = torch.randn(4, 6)
    with pytest.raises(RuntimeError):
        torch.func.jvp(call, (t,), (torch.ones(4, 6),))
    with pytest.raises(RuntimeError):
        torch.func.vmap(call)(torch.randn(2, 4, 6))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: call(t).sum())(t)


@pytest.mark.parametrize("act", ["none", "relu", "silu"])
def test_hidden_activation_calls_the_module(monkeypatch, act):
    """Hooks of the norm run, and its own activation counts, in every mode; what they see is the
    same in all (plain torch in the kernels' places)."""
    acts = {"none": lambda z: z, "relu": torch.relu, "silu": torch.nn.functional.silu}

    def plain(x, groups, weight=None, bias=None, eps=1e-5, act="none"):
        return acts[act](torch.nn.functional.group_norm(x, groups, weight, bias, eps))
    monkeypatch.setattr(norm, "group_norm", plain)
    if hasattr(gcn, "group_norm"):
        monkeypatch.setattr(gcn, "group_norm", plain)
    monkeypatch.setattr(gcn.ReluDropout, "apply", lambda x, p, seed: torch.relu(x) * 2)  # drops nothing here
    layer, seen = norm.GroupNorm(2, 6, act=act), []
    with torch.no_grad():
        layer.weight.copy_(torch.linspace(-1, 2, 6))
        layer.bias.copy_(torch.linspace(-0.5, 0.5, 6))
    layer.register_forward_hook(lambda module, args, out: seen.append(out.detach()))
    x = torch.randn(5, 6)
    want = plain(x, 2, layer.weight, layer.bias, act=act)
    for training, p in ((True, 0.5), (True, 0.0), (False, 0.5), (False, 0.0)):
        out = gcn.hidden_activation(x, p, 3, training, layer)
        assert torch.equal(out, torch.relu(want) * (2 if training and p else 1))
    assert len(seen) == 4 and all(torch.equal(s, want) for s in seen)


def test_every_lookup_can_report_a_bad_index(no_launch, monkeypatch):
    """The module and the block's rows hand `bad` on to the call."""
    flags = []
    monkeypatch.setattr(embedding, "launch", lambda device, name, *args: flags.append(args[-1]))
    bad = torch.zeros(1, dtype=torch.int32)
    layer = embedding.NodeEmbedding(4, 6)
    block = minibatch.Block(dst_ids=IDX, src_ids=IDX, edge_dst=IDX, edge_src=IDX)
    for call in (lambda **kw: layer(IDX, **kw), lambda **kw: minibatch.embedding_rows(layer.weight, block, **kw)):
        call()
        call(bad=bad)
    assert flags == [None, bad.data_ptr()] * 2


def test_padding_beyond_64_bits_is_refused(no_launch):
    """-2^64 + 3 would be taken for 3."""
    t = torch.zeros(4, 6)
    for wrong in (-(1 << 64) + 3, (1 << 64) - 1, 1 << 63, -(1 << 63)):
        for call in (lambda: embedding.embedding(t, IDX, padding_idx=wrong),
                     lambda: embedding.embedding_backward(t[:3], IDX, 4, padding_idx=wrong),
                     lambda: embedding.embedding(t[:, :0], IDX, padding_idx=wrong)):
            with pytest.raises(ValueError, match="padding_idx"):
                call()
