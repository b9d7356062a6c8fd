"""Argument handling shared by the training operators' Python entry points
(:mod:`embedding`, :mod:`norm`, :mod:`clip`)."""
from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import _lib as L

TYPES = {torch.float32: L.F32, torch.float16: L.F16, torch.bfloat16: L.BF16}


def type_code(t: torch.Tensor, name: str) -> int:
    """TCC_F32 / F16 / BF16 of a CUDA tensor; raises for anything else."""
    code = TYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"{name} must be float32, float16 or bfloat16, not {t.dtype}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    return code


def tracked(*tensors) -> bool:
    """Whether autograd has to see a call with these inputs (None for one left out): one requires a
    gradient, or carries a tangent (forward mode, which the operators' functions refuse with an error;
    past them its derivative would be lost in silence)."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    # outside dual_level, 0.3 us a tensor less than asking each
    return forward_ad._current_level >= 0 and any(
        t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


_bound = {}
# The current stream's handle without building a Stream object: 0.1 us in place
# of 2, of the 9 to 13 that a call takes on the host.
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice


def launch(device: torch.device, name: str, *args) -> None:
    """The C call with ``device`` current, on its current stream (the last argument)."""
    call = _bound.get(name)
    if call is None:
        call = _bound[name] = getattr(L.lib(), name)
    index = device.index
    if index == _current_device():
        status = call(*args, _raw_stream(index))
    else:
        with torch.cuda.device(device):
            status = call(*args, _raw_stream(index))
    if status:
        L.check(status, name)


def rows_of(t: torch.Tensor, width: int):
    """(tensor, row stride) of ``t`` seen as rows of ``width`` contiguous values;
    a contiguous copy where its strides have no such form."""
    if t.is_contiguous():
        return t, width
    if t.shape[-1] == 1 or t.stride(-1) == 1:
        dims = [d for d in range(t.dim() - 1) if t.shape[d] > 1]
        if not dims:
            return t, width
        ld = t.stride(dims[-1])
        if ld >= width and all(t.stride(a) == t.stride(b) * t.shape[b] for a, b in zip(dims, dims[1:])):
            return t, ld
    return t.contiguous(), width


def scratch_for(nbytes: int, device: torch.device):
    """(tensor that holds it, address) of ``nbytes`` of scratch; (None, None) for none."""
    if nbytes == 0:
        return None, None
    s = torch.empty(nbytes, dtype=torch.uint8, device=device)
    return s, s.data_ptr()
