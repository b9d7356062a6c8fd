"""Group norm over channels-last node features, with the activation that follows.

The hidden-layer epilogue beside ``gcn.relu_dropout``: x is [N, C] (every node by
itself) or [N, ..., C] (every sample over all of its rows: a graph, a padded
batch of graphs); the C channels form groups of neighbours that share a mean and
a variance.  The reference's models have no normalisation
(train/tcgnn_conv_release.py:196-268, train/ = TAC_training_backend/train/).
"""
from __future__ import annotations

import functools
import math

import torch

from . import _lib as L
from ._args import launch, rows_of, scratch_for, tracked, type_code


def _parameter(p, name: str, channels: int, x: torch.Tensor):
    if p.dim() != 1 or p.shape[0] != channels:
        raise ValueError(f"{name} must have shape ({channels},)")
    if p.device != x.device:
        raise ValueError(f"{name} must be on x's device")
    return p if p.is_contiguous() else p.contiguous()


def _parameters(weight, bias, channels: int, x: torch.Tensor):
    """(weight, bias, their type) contiguous; checks shape, type and device."""
    code = L.F32
    if weight is not None:
        code = type_code(weight, "weight")
        weight = _parameter(weight, "weight", channels, x)
    if bias is not None:
        code = type_code(bias, "bias")
        bias = _parameter(bias, "bias", channels, x)
        if weight is not None and weight.dtype != bias.dtype:
            raise TypeError("weight and bias must have one type")
    return weight, bias, code


def _sizes(x: torch.Tensor, num_groups: int):
    shape = x.shape
    if len(shape) < 2:
        raise ValueError("x must be [N, ..., C]")
    channels = shape[-1]
    if num_groups < 1 or channels < 1 or channels % num_groups:
        raise ValueError("num_groups must divide a positive number of channels")
    return shape[0], 1 if len(shape) == 2 else math.prod(shape[1:-1]), channels


def _statistics(s, name: str, n: int, num_groups: int, x: torch.Tensor) -> None:
    if s.shape != (n, num_groups) or s.dtype != torch.float32 or s.device != x.device or not s.is_contiguous():
        raise ValueError(f"{name} must be a contiguous float32 [N, num_groups] tensor on x's device")


def _activation(act: str) -> int:
    code = L.ACTIVATIONS.get(act)
    if code is None:
        raise ValueError(f"act must be one of {', '.join(L.ACTIVATIONS)}")
    return code


def _ptr(t):
    return None if t is None else t.data_ptr()


def _empty(x):
    """A contiguous tensor of x's shape, type and device."""
    return torch.empty_like(x) if x.is_contiguous() else torch.empty(x.shape, dtype=x.dtype, device=x.device)


@functools.lru_cache(maxsize=256)
def _scratch_bytes(n: int, steps: int, channels: int, num_groups: int, backward: int) -> int:
    return L.lib().tcc_group_norm_scratch_bytes(n, steps, channels, num_groups, backward)


def _forward(x, num_groups, weight, bias, eps, act, stats):
    code, act = type_code(x, "x"), _activation(act)
    n, steps, channels = _sizes(x, num_groups)
    weight, bias, p_code = _parameters(weight, bias, channels, x)
    y = _empty(x)
    mean = rstd = None
    if stats:
        mean, rstd = torch.empty((2, n, num_groups), dtype=torch.float32, device=x.device).unbind(0)
    if n and steps:
        x, ld = rows_of(x, channels)
        nbytes = _scratch_bytes(n, steps, channels, num_groups, 0)
        hold, scratch = scratch_for(nbytes, x.device)
        launch(x.device, "tcc_group_norm_forward", x.data_ptr(), code, ld, _ptr(weight), _ptr(bias), p_code,
               y.data_ptr(), channels, _ptr(mean), _ptr(rstd), n, steps, channels, num_groups, eps, act,
               scratch, nbytes)
    elif stats:  # samples without rows have no statistics
        mean.zero_()
        rstd.zero_()
    return y, mean, rstd


def group_norm_forward(x: torch.Tensor, num_groups: int, weight: torch.Tensor | None = None,
                       bias: torch.Tensor | None = None, eps: float = 1e-5, act: str = "none"):
    """(y, mean, rstd): ``group_norm`` and the fp32 [N, num_groups] statistics its backward reads.
    Not differentiable: the pass by itself."""
    return _forward(x, num_groups, weight, bias, eps, act, True)


def group_norm_backward(dy: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor,
                        num_groups: int, weight: torch.Tensor | None = None,
                        bias: torch.Tensor | None = None, act: str = "none", need_dx: bool = True):
    """(dx, dweight, dbias) of ``group_norm`` for the output gradient dy, from the
    forward's x, mean and rstd.  None for a parameter that is None, and for dx
    without ``need_dx``.  Not differentiable itself."""
    code, act = type_code(x, "x"), _activation(act)
    n, steps, channels = _sizes(x, num_groups)
    if dy.shape != x.shape or dy.dtype != x.dtype or dy.device != x.device:
        raise ValueError("dy must have x's shape, type and device")
    _statistics(mean, "mean", n, num_groups, x)
    _statistics(rstd, "rstd", n, num_groups, x)
    weight, bias, p_code = _parameters(weight, bias, channels, x)
    dx = _empty(x) if need_dx else None
    dweight = None if weight is None else torch.empty_like(weight)
    dbias = None if bias is None else torch.empty_like(bias)
    x, ldx = rows_of(x, channels)
    dy, lddy = rows_of(dy, channels)
    nbytes = _scratch_bytes(n, steps, channels, num_groups, 1)
    hold, scratch = scratch_for(nbytes, x.device)
    launch(x.device, "tcc_group_norm_backward", dy.data_ptr(), lddy, x.data_ptr(), ldx, code, _ptr(weight),
           _ptr(bias), p_code, mean.data_ptr(), rstd.data_ptr(), _ptr(dx), channels, _ptr(dweight),
           _ptr(dbias), n, steps, channels, num_groups, act, scratch, nbytes)
    return dx, dweight, dbias


class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, num_groups, weight, bias, eps, act):
        y, mean, rstd = group_norm_forward(x, num_groups, weight, bias, eps, act)
        ctx.save_for_backward(x, weight, bias, mean, rstd)
        ctx.args = (num_groups, act)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, bias, mean, rstd = ctx.saved_tensors
        num_groups, act = ctx.args
        dx, dw, db = group_norm_backward(dy, x, mean, rstd, num_groups, weight, bias, act,
                                         need_dx=ctx.needs_input_grad[0])
        return dx, None, dw, db, None, None


def group_norm(x: torch.Tensor, num_groups: int, weight: torch.Tensor | None = None,
               bias: torch.Tensor | None = None, eps: float = 1e-5, act: str = "none") -> torch.Tensor:
    """act(group norm of x * weight + bias), differentiable in x, weight and bias (in reverse mode).

    x: [N, C] or [N, ..., C], float32, float16 or bfloat16; statistics per sample
    and group in fp32 with the population variance.  weight, bias: [C] of one
    type (x's or another), or None.  act: "none", "relu", "silu" or "gelu"."""
    if tracked(x, weight, bias):
        return _GroupNorm.apply(x, num_groups, weight, bias, eps, act)
    return _forward(x, num_groups, weight, bias, eps, act, False)[0]


class GroupNorm(torch.nn.Module):
    """``group_norm`` with learned weight and bias per channel."""

    def __init__(self, num_groups: int, channels: int, eps: float = 1e-5, act: str = "none", dtype=None,
                 device=None):
        super().__init__()
        if num_groups < 1 or channels % num_groups:
            raise ValueError("num_groups must divide the number of channels")
        _activation(act)
        self.num_groups, self.eps, self.act = num_groups, eps, act
        self.weight = torch.nn.Parameter(torch.ones(channels, dtype=dtype, device=device))
        self.bias = torch.nn.Parameter(torch.zeros(channels, dtype=dtype, device=device))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return group_norm(x, self.num_groups, self.weight, self.bias, self.eps, self.act)
