"""The global norm of many gradient tensors, and clipping, in two HIP passes.

    norm = clip_grad_norm(model.parameters(), 1.0)        # in place, before optimizer.step()

(No counterpart in the reference, whose training loops call torch's.)
"""
from __future__ import annotations

import math
from typing import Iterable

import torch

from . import kernels

NORM_CODES = {2.0: 2, 1.0: 1, math.inf: 0}


def _norm_code(norm_type) -> int:
    code = NORM_CODES.get(float(norm_type))
    if code is None:
        raise ValueError(f"norm_type must be 1, 2 or infinity, got {norm_type!r}")
    return code


def _dense(t) -> bool:
    """Whether the elements fill one stretch of memory, each once, in any order of the dimensions."""
    if t.is_contiguous():
        return True
    span = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if stride != span:
            return False
        span *= size
    return True


def _check_tensors(grads, name):
    device = grads[0].device
    for t in grads:
        if t.device != device or not t.is_cuda:
            kernels.require_gpu(t, name)
            raise RuntimeError(f"{name} are on {device} and {t.device}: one GPU is needed")
        if t.dtype not in kernels.DTYPE_CODES:
            kernels.dtype_code(t.dtype)
        if t.layout != torch.strided:
            raise ValueError(f"{name} must be dense tensors, got {t.layout}")
    return device


def clip_gradients(grads: Iterable[torch.Tensor], max_norm: float, *, norm_type: float = 2.0, eps: float = 1e-6,
                   out: Iterable[torch.Tensor] | None = None, error_if_nonfinite: bool = False) -> torch.Tensor:
    """Scales ``grads`` by min(1, max_norm / (norm + eps)) and returns their global norm, a float32 scalar on
    their device.

    The norm is over all elements of all tensors (``norm_type`` 1, 2 or infinity) in 64 bits; types may
    be mixed.  In place, or into the tensors of ``out`` (one of the same shape and type for each).  Nothing waits for the
    GPU unless ``error_if_nonfinite`` asks whether the norm is finite, before anything is scaled.
    """
    grads = list(grads)
    code = _norm_code(norm_type)
    max_norm, eps = float(max_norm), float(eps)
    if not max_norm >= 0.0 or not eps >= 0.0:
        raise ValueError(f"max_norm and eps must not be negative, got {max_norm} and {eps}")
    if out is not None:
        out = list(out)
        if len(out) != len(grads):
            raise ValueError(f"{len(grads)} gradients and {len(out)} outputs")
    if not grads:
        return torch.zeros(())
    device = _check_tensors(grads, "gradients")
    if out is not None:
        if _check_tensors(out, "outputs") != device:
            raise RuntimeError(f"gradients are on {device}, outputs on {out[0].device}")
        for g, o in zip(grads, out):
            if g.shape != o.shape or g.dtype != o.dtype:
                raise ValueError(f"an output of {tuple(o.shape)} {o.dtype} for a gradient of {tuple(g.shape)} {g.dtype}")
    if error_if_nonfinite:
        total = grad_norm(grads, norm_type=norm_type)
        if not math.isfinite(float(total)):
            raise RuntimeError(f"The total norm of the gradients is {float(total)}: it cannot be clipped")
    # elements are taken in memory order: a tensor with gaps goes through a packed copy
    with torch.no_grad():
        into = grads if out is None else out
        src, dst, copies = [], [], []
        for g, o in zip(grads, into):
            if _dense(g) and (o is g or o.stride() == g.stride()):
                src.append(g)
                dst.append(o)
                continue
            if o is g and any(s == 0 and n > 1 for s, n in zip(g.stride(), g.shape)):
                raise ValueError("a gradient whose elements share memory cannot be scaled in place")
            packed = g.contiguous() if _dense(o) and o.is_contiguous() else g.clone(memory_format=torch.contiguous_format)
            src.append(packed)
            if o.is_contiguous():
                dst.append(o)
            else:
                dst.append(packed)
                copies.append((o, packed))
        norm = kernels.clip_gradients(src, dst, code, max_norm, eps, device)
        for o, packed in copies:
            o.copy_(packed)
    return norm


def grad_norm(grads: Iterable[torch.Tensor], *, norm_type: float = 2.0) -> torch.Tensor:
    """The global norm of the tensors, a float32 scalar on their device; nothing is scaled."""
    grads = list(grads)
    code = _norm_code(norm_type)
    if not grads:
        return torch.zeros(())
    device = _check_tensors(grads, "gradients")
    with torch.no_grad():
        return kernels.clip_gradients([g if _dense(g) else g.contiguous() for g in grads], None, code, 0.0, 0.0, device)


def clip_grad_norm(parameters: torch.Tensor | Iterable[torch.Tensor], max_norm: float, *, norm_type: float = 2.0,
                   eps: float = 1e-6, error_if_nonfinite: bool = False) -> torch.Tensor:
    """clip_gradients of the parameters' ``.grad`` in place; parameters without one are left out."""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    return clip_gradients([p.grad for p in parameters if p.grad is not None], max_norm, norm_type=norm_type, eps=eps,
                          error_if_nonfinite=error_if_nonfinite)


__all__ = ["clip_grad_norm", "clip_gradients", "grad_norm"]
