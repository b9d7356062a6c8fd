"""The global norm of a model's gradients, and clipping by it.

The reference steps its optimiser on unclipped gradients
(TAC_training_backend/train/tcgnn_conv_release.py); ``train_gcn`` clips with
``--clip-norm``.  The norm stays on the GPU: nothing synchronises, and the calls
can be captured in a CUDA graph.
"""
from __future__ import annotations

import functools
from array import array

import torch

from . import _lib as L
from ._args import TYPES, launch, scratch_for


def _dense(t: torch.Tensor) -> bool:
    """Whether the elements of a tensor that is not contiguous fill one block of memory all the same."""
    want = 1
    for size, stride in sorted(((s, st) for s, st in zip(t.shape, t.stride()) if s > 1), key=lambda p: p[1]):
        if stride != want:
            return False
        want *= size
    return True


def _table(tensors):
    """(tcc_tensor array of the tensors, its length, their device, their bytes)."""
    index, words, nbytes = None, [], 0
    for t in tensors:
        code = TYPES.get(t.dtype)
        if code is None:
            raise TypeError(f"gradients must be float32, float16 or bfloat16, not {t.dtype}")
        where = t.get_device()
        if where < 0 or t.layout is not torch.strided:
            raise ValueError("gradients must be dense CUDA tensors")
        if where != index:
            if index is not None:
                raise ValueError("gradients must be on one device")
            index = where
        if not (t.is_contiguous() or _dense(t)):
            raise ValueError("a gradient's elements must fill one block of memory (no gaps, no broadcast)")
        n = t.numel()
        nbytes += n << 2 if code == L.F32 else n << 1
        words += (t.data_ptr(), n, code)  # data, n, type and reserved
    return array("Q", words), len(words) // 3, None if index is None else torch.device("cuda", index), nbytes


@functools.cache
def _scratch_bytes() -> int:
    return L.lib().tcc_grad_norm_scratch_bytes()


def _list(tensors) -> list:
    return [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)


def _written(tensors) -> None:
    """The tensors were changed in place: a graph that saved one notices."""
    try:
        torch.autograd.graph.increment_version(tensors)
    except RuntimeError:  # inference tensors have no version
        torch.autograd.graph.increment_version([t for t in tensors if not t.is_inference()])


def grad_norm(tensors) -> torch.Tensor:
    """The 2-norm of all elements of the tensors (one, or an iterable), a float32 scalar on
    their device; 64-bit sums in a fixed order.  Without tensors a CPU zero.  No derivative
    flows through it."""
    words, count, device, _ = _table(_list(tensors))
    if count == 0:
        return torch.zeros(())
    norm = torch.empty((), dtype=torch.float32, device=device)
    nbytes = _scratch_bytes()
    hold, scratch = scratch_for(nbytes, device)
    launch(device, "tcc_grad_norm", words.buffer_info()[0], count, norm.data_ptr(), scratch, nbytes)
    return norm


def clip_grads_with_norm_(tensors, max_norm: float, total_norm: torch.Tensor, eps: float = 1e-6) -> None:
    """Scale the tensors in place by max_norm / (total_norm + eps) where that is below 1.
    total_norm: a float32 scalar on their device (e.g. combined over the ranks that each
    hold a part of the parameters: the root of the sum of their squared norms)."""
    tensors = _list(tensors)
    words, count, device, _ = _table(tensors)
    if count == 0:
        return
    if total_norm.dtype != torch.float32 or total_norm.numel() != 1 or total_norm.device != device:
        raise ValueError("total_norm must be a float32 scalar on the gradients' device")
    launch(device, "tcc_clip_grads_with_norm", words.buffer_info()[0], count, total_norm.data_ptr(), max_norm, eps)
    _written(tensors)


def clip_grad_norm_(parameters, max_norm: float, eps: float = 1e-6, error_if_nonfinite: bool = False) -> torch.Tensor:
    """Clip the gradients of the parameters (one, or an iterable; those without a
    gradient are passed over) in place to a global 2-norm of max_norm, and return
    the norm they had, a float32 scalar.  Gradients of different types may mix;
    two that share memory are refused.  ``error_if_nonfinite`` waits for the norm
    and raises where it is NaN or infinite, before anything is scaled."""
    grads = [g for g in (p.grad for p in _list(parameters)) if g is not None]
    if error_if_nonfinite:
        norm = grad_norm(grads)
        if not bool(torch.isfinite(norm)):
            raise RuntimeError("the gradients' norm is not finite, so they cannot be clipped")
        if grads:
            clip_grads_with_norm_(grads, max_norm, norm, eps)
        return norm
    words, count, device, total = _table(grads)
    if count == 0:
        return torch.zeros(())
    norm = torch.empty((), dtype=torch.float32, device=device)
    small = count <= L.CLIP_SMALL_TENSORS and total <= L.CLIP_SMALL_BYTES
    nbytes = 0 if small else _scratch_bytes()
    hold, scratch = scratch_for(nbytes, device)
    launch(device, "tcc_clip_grad_norm", words.buffer_info()[0], count, max_norm, eps, norm.data_ptr(), scratch,
           nbytes)
    _written(grads)
    return norm
