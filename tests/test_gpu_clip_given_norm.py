"""Clipping by a norm that the caller gives (tcc_b200.clip): it need not be the tensors' own."""
import math

import pytest
import torch

from tcc_b200 import clip as K

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sizes", [(50,), (7, 3), (100_003,)])
@pytest.mark.parametrize("total,max_norm,eps", [(0.0, 0.0, 1e-6), (0.0, 0.25, 1.0), (0.0, 1.0, 1e-6), (4.0, 1.0, 0.0),
                                                (math.inf, 1.0, 1e-6), (math.nan, 1.0, 1e-6), (0.0, 0.0, 0.0)])
def test_the_formula_holds_for_any_norm(gpu, sizes, total, max_norm, eps):
    """Every element times max_norm / (norm + eps) where that is below 1; a NaN norm spreads."""
    grads = [torch.linspace(-2, 3, n, device="cuda") for n in sizes]
    before = [g.clone() for g in grads]
    K.clip_grads_with_norm_(grads, max_norm, torch.tensor(total, device="cuda"), eps)
    bottom = total + eps
    factor = math.inf if bottom == 0 else max_norm / bottom
    for g, b in zip(grads, before):
        if math.isnan(total):
            assert bool(g.isnan().all())
        elif factor >= 1:  # 0 / 0 among them
            assert torch.equal(g, b)
        else:  # the factor's sum and quotient, and the product: 3 roundings of half a unit
            assert bool(((g.double() - b.double() * factor).abs() <= 3 * 2.0 ** -24 * b.double().abs() * factor).all())
