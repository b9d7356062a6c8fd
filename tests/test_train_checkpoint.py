"""What a run checks of the checkpoint it resumes (CPU only)."""
import pytest

from tcc_b200 import train_gcn


def _ck(groups, config=True):
    ck = {"epoch": 2}
    if groups:
        ck["norm"] = {}
    if config:
        ck["config"] = dict(train_gcn.config(10), norm_groups=groups)
    return ck


@pytest.mark.parametrize("saved,now", [(8, 4), (8, 0), (0, 8), (4, None), (None, 4), (1, 2)])
def test_other_groups_are_refused(saved, now):
    with pytest.raises(ValueError, match="norm-groups"):
        train_gcn.check_norm_groups(_ck(saved), dict(norm_groups=now))


@pytest.mark.parametrize("saved,now", [(8, 8), (0, 0), (None, 0), (0, None)])
def test_the_same_groups_are_taken(saved, now):
    train_gcn.check_norm_groups(_ck(saved), dict(norm_groups=now))
    train_gcn.check_norm_groups(_ck(saved), dict(norm_groups=now) if now else {})
    train_gcn.check_norm_groups(_ck(saved, config=False), dict(norm_groups=now))  # a checkpoint without its options


def test_a_checkpoint_from_before_the_option():
    ck = _ck(None)
    del ck["config"]["norm_groups"]
    train_gcn.check_norm_groups(ck, dict(norm_groups=0))
    with pytest.raises(ValueError):
        train_gcn.check_norm_groups(ck, dict(norm_groups=8))
