"""Every index outside a table is reported (tcc_b200.embedding), whatever its value and the call's sizes."""
import pytest
import torch

from tcc_b200 import embedding as E

pytestmark = pytest.mark.gpu

LOWEST = -(1 << 63)


def _calls(rows, width, idx, **kw):
    table = torch.randn((rows, width), device="cuda")
    grad = torch.randn((idx.numel(), width), device="cuda")
    return [lambda bad: E.embedding(table, idx, bad=bad, **kw),
            lambda bad: E.embedding_backward(grad, idx, rows, bad=bad, **kw)]


@pytest.mark.parametrize("n", [3, 1500, 70_001])  # owner form, cluster sort, tiles' sort
@pytest.mark.parametrize("padding", [None, -1, LOWEST + 1])
def test_the_lowest_index_is_no_padding(gpu, n, padding):
    idx = torch.randint(40, (n,), device="cuda")
    idx[2] = LOWEST
    for call in _calls(40, 8, idx, padding_idx=padding):
        bad = torch.zeros(1, dtype=torch.int32, device="cuda")
        call(bad)
        assert int(bad) == 1
    idx[2] = 5 if padding is None else padding
    for call in _calls(40, 8, idx, padding_idx=padding):
        bad = torch.zeros(1, dtype=torch.int32, device="cuda")
        call(bad)
        assert int(bad) == 0


@pytest.mark.parametrize("rows,width", [(0, 4), (0, 0), (5, 0)])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_tables_without_values(gpu, rows, width, dtype):
    for values, padding, want in (([rows], None, 1), ([-1, -1], -1, 0), ([-1, -1], None, 1), ([-1, rows], -1, 1),
                                  ([], None, 0)):
        idx = torch.tensor(values, dtype=dtype, device="cuda")
        for call in _calls(rows, width, idx, padding_idx=padding):
            bad = torch.zeros(2, dtype=torch.int32, device="cuda")
            call(bad)
            assert bad.tolist() == [want, 0], (values, padding)
    kept = torch.ones(1, dtype=torch.int32, device="cuda")  # a flag that is set stays set
    for call in _calls(rows, width, torch.empty(0, dtype=dtype, device="cuda")):
        call(kept)
        assert int(kept) == 1
