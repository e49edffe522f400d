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


def _refuse(tensors, name):
    """Says what is wrong with the first tensor that is."""
    device = tensors[0].device
    for t in tensors:
        if t.layout != torch.strided:
            raise ValueError(f"{name} must be dense tensors, got {t.layout}")
        kernels.require_gpu(t, name)
        kernels.dtype_code(t.dtype)
        if t.device != device:
            raise RuntimeError(f"{name} are on {device} and {t.device}: one GPU is needed")


def _facts(tensors, name):
    """(addresses, element counts, type codes) of tensors on one GPU; None for the tensors' own order if every
    one is contiguous, else the list of those that are."""
    codes = kernels.DTYPE_CODES
    try:
        index = tensors[0].get_device()
        if index < 0 or any([t.get_device() != index for t in tensors]):
            _refuse(tensors, name)
        types = [codes[t.dtype] for t in tensors]
        plain = [t.is_contiguous() for t in tensors]
        return [t.data_ptr() for t in tensors], [t.numel() for t in tensors], types, None if all(plain) else plain
    except (KeyError, RuntimeError):
        _refuse(tensors, name)
        raise


def clip_gradients(grads: Iterable[torch.Tensor], max_norm: float, *, norm_type: float = 2.0, eps: float = 1e-6,
                   out: Iterable[torch.Tensor] | None = None, error_if_nonfinite: bool = False) -> torch.Tensor:
    """Scales ``grads`` by min(1, max_norm / (norm + eps)) and returns their global norm, a float32 scalar on
    their device.

    The norm is over all elements of all tensors (``norm_type`` 1, 2 or infinity) in 64 bits; types may
    be mixed.  In place, or into the tensors of ``out`` (for each gradient one of its type, and of its shape
    or, all being contiguous, its number of elements).  Nothing waits for the GPU unless
    ``error_if_nonfinite`` asks whether the norm is finite, before anything is scaled.
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
    at, sizes, codes, plain = _facts(grads, "gradients")
    device = grads[0].device
    into, copies = at, []
    if out is not None:
        into, out_sizes, out_codes, out_plain = _facts(out, "outputs")
        if out[0].device != device:
            raise RuntimeError(f"gradients are on {device}, outputs on {out[0].device}")
        plain = plain or out_plain
        if codes != out_codes or sizes != out_sizes or (plain and [g.shape for g in grads] != [o.shape for o in out]):
            for g, o in zip(grads, out):
                if g.numel() != o.numel() or g.dtype != o.dtype or (plain and g.shape != o.shape):
                    raise ValueError(f"an output of {tuple(o.shape)} {o.dtype} for a gradient of {tuple(g.shape)} {g.dtype}")
    if error_if_nonfinite:
        total = grad_norm(grads, norm_type=norm_type)
        if not math.isfinite(float(total)):
            raise RuntimeError(f"The total norm of the gradients is {float(total)}: it cannot be clipped")
    if plain is not None:
        # elements are taken in memory order: a tensor with gaps goes through a packed copy
        at, into = list(at), list(into)
        with torch.no_grad():
            for i, (g, o) in enumerate(zip(grads, grads if out is None else out)):
                if _dense(g) and o.stride() == g.stride():
                    continue
                if o is g and any(s == 0 and n > 1 for s, n in zip(g.stride(), g.shape)):
                    raise ValueError("a gradient whose elements share memory cannot be scaled in place")
                packed = g.clone(memory_format=torch.contiguous_format)
                at[i] = into[i] = packed.data_ptr()
                copies.append((o, packed))
    norm = kernels.clip_gradients(at, into, sizes, codes, code, max_norm, eps, device)
    with torch.no_grad():
        for o, packed in copies:
            o.copy_(packed)
    return norm


def grad_norm(grads: Iterable[torch.Tensor], *, norm_type: float = 2.0) -> torch.Tensor:
    """The global norm of the tensors, a float32 scalar on their device; nothing is scaled."""
    grads = list(grads)
    code = _norm_code(norm_type)
    if not grads:
        return torch.zeros(())
    at, sizes, codes, plain = _facts(grads, "gradients")
    if plain is not None:
        with torch.no_grad():
            grads = [g if _dense(g) else g.contiguous() for g in grads]
        at = [g.data_ptr() for g in grads]
    return kernels.clip_gradients(at, None, sizes, codes, code, 0.0, 0.0, grads[0].device)


def clip_grad_norm(parameters: torch.Tensor | Iterable[torch.Tensor], max_norm: float, *, norm_type: float = 2.0,
                   eps: float = 1e-6, error_if_nonfinite: bool = False) -> torch.Tensor:
    """clip_gradients of the parameters' ``.grad`` in place; parameters without one are left out."""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    return clip_gradients([p.grad for p in parameters if p.grad is not None], max_norm, norm_type=norm_type, eps=eps,
                          error_if_nonfinite=error_if_nonfinite)


__all__ = ["clip_grad_norm", "clip_gradients", "grad_norm"]
