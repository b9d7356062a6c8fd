"""What the trainer and the modules check of their inputs (GPU)."""
import pytest
import torch

from tcc_b200 import embedding as E
from tcc_b200 import train_gcn

pytestmark = pytest.mark.gpu


def _small(**kw):
    cfg = train_gcn.config(shrink=10)
    cfg.update(dropout=0.0, epochs=1)
    cfg.update(kw)
    return cfg


@pytest.mark.parametrize("order", [True, False])
def test_trainer_refuses_a_labelled_row_outside_the_graph(gpu, monkeypatch, order):
    build = train_gcn.build

    def broken(*args):
        r = build(*args)
        r["lab_idx"] = r["lab_idx"].clone()
        r["lab_idx"][0] = r["r1"] - r["r0"]  # one past the last row: the lookup reads nothing there
        return r
    monkeypatch.setattr(train_gcn, "build", broken)
    with pytest.raises(IndexError, match="labelled row"):
        train_gcn.train(_small(), gpu, 1, 0, order)


def test_module_reports_a_bad_index(gpu):
    layer = E.NodeEmbedding(30, 10, padding_idx=-1, device="cuda")
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    idx = torch.tensor([3, -1, 29], device="cuda")
    layer(idx, bad)
    assert int(bad) == 0
    idx[2] = 30
    assert not layer(idx, bad)[2].any() and int(bad) == 1


def test_resume_with_other_groups_is_refused(gpu, tmp_path):
    ck = str(tmp_path / "gcn.pt")
    train_gcn.train(_small(norm_groups=8, save=ck), gpu, 1, 0)
    for groups in (4, 0):
        with pytest.raises(ValueError, match="norm-groups"):
            train_gcn.train(_small(norm_groups=groups, epochs=2, resume=ck), gpu, 1, 0)
    assert len(train_gcn.train(_small(norm_groups=8, epochs=2, resume=ck), gpu, 1, 0)["losses"]) == 1


@pytest.mark.parametrize("clip", [None, 1e-3])
def test_the_optimiser_sees_clipped_gradients(gpu, monkeypatch, clip):
    """The norm of all gradients at Adam's step, with and without the option at the same model; the
    tiny limit is far below the gradients' own norm."""
    seen = []
    step = torch.optim.Adam.step

    def record(self, *args, **kw):
        grads = [p.grad.double() for group in self.param_groups for p in group["params"]]
        seen.append(float(torch.stack([g.square().sum() for g in grads]).sum().sqrt()))
        return step(self, *args, **kw)
    monkeypatch.setattr(torch.optim.Adam, "step", record)
    train_gcn.train(_small(norm_groups=8, clip_norm=clip, epochs=3), gpu, 1, 0)
    assert len(seen) == 3
    if clip is None:
        assert min(seen) > 2e-3
    else:  # eps beside a norm above 2e-3, the factor's roundings and that of every product
        assert all(abs(n / clip - 1) <= 1e-6 / 2e-3 + 4 * 2.0 ** -24 for n in seen)
