"""Rotary positions of queries and keys in one HIP kernel, forward and backward.

    cos, sin = rotary_tables(max_positions, rot)          # once
    q, k = rotary(q, k, cos, sin, positions=positions)    # batch x seq x heads x head

(No counterpart in the reference.)
"""
from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable

from . import _lib, kernels


def rotary_tables(length: int, rot: int, *, base: float = 10000.0, scaling: str | None = None, factor: float = 1.0,
                  original_length: int | None = None, beta_fast: float = 32.0, beta_slow: float = 1.0,
                  device="cuda") -> tuple[torch.Tensor, torch.Tensor]:
    """(cos, sin), ``length`` x ``rot`` / 2 in fp32, of position p times base^(-2 j / rot), from 64 bits.

    ``scaling`` for contexts ``factor`` times as long as a model was trained on: "linear" (frequencies
    divided by the factor), "ntk" (base times factor^(rot / (rot - 2))) or "by_parts" (pairs that turn
    more than ``beta_fast`` times over ``original_length`` kept, those that turn less than ``beta_slow``
    times divided, a linear blend between, tables times 0.1 ln(factor) + 1).
    """
    if scaling not in _lib.ROTARY_SCALINGS:
        raise ValueError(f"scaling must be one of {list(_lib.ROTARY_SCALINGS)}, got {scaling!r}")
    if int(length) != length or length < 0 or int(rot) != rot:
        raise ValueError("length and rot must be integers, length not negative")
    if not all(math.isfinite(v) for v in (base, factor, beta_fast, beta_slow)):
        raise ValueError("base, factor and the betas must be finite")
    if scaling == "by_parts" and original_length is None:
        raise ValueError("scaling by parts needs original_length")
    device = torch.device(device)
    if device.type != "cuda":
        raise RuntimeError(f"stacr_amd: rotary tables are made on a ROCm GPU (got device {device})")
    return kernels.rotary_tables(int(length), int(rot), base, scaling, factor, original_length or 0, beta_fast, beta_slow,
                                 device)


def _check_rotary(q, k, cos, sin, positions, layout) -> None:
    # the usual case in few steps: a call on single tokens is bound by the host
    shape, dtype, index, table = q.shape, q.dtype, q.get_device(), cos.shape
    if (len(shape) == 4 and index >= 0 and layout in _lib.ROTARY_LAYOUTS and dtype in kernels.DTYPE_CODES and
            k is not None and k.dtype is dtype and k.dim() == 4 and k.get_device() == index and
            k.shape[:2] == shape[:2] and k.shape[3] == shape[3] and len(table) == 2 and table == sin.shape and
            cos.dtype is torch.float32 and sin.dtype is torch.float32 and 2 <= 2 * table[1] <= shape[3] and
            cos.get_device() == index and sin.get_device() == index and positions is not None and
            positions.dtype is torch.int64 and positions.shape == shape[:2] and positions.get_device() == index):
        return
    if layout not in _lib.ROTARY_LAYOUTS:
        raise ValueError(f"layout must be one of {list(_lib.ROTARY_LAYOUTS)}, got {layout!r}")
    kernels.require_gpu(q, "queries")
    kernels.dtype_code(dtype)
    if len(shape) != 4:
        raise ValueError(f"queries are batch x seq x heads x head, got {q.dim()} dimensions")
    if k is not None:
        if k.dim() != 4 or k.shape[:2] != shape[:2] or k.shape[3] != shape[3]:
            raise ValueError(f"keys {tuple(k.shape)} do not match queries {tuple(shape)}")
        if k.dtype != dtype:
            raise TypeError(f"keys are {k.dtype}, queries {dtype}")
    if len(table) != 2 or table != sin.shape:
        raise ValueError(f"cos and sin must be two (positions, rot / 2) tables, got {tuple(table)} and "
                         f"{tuple(sin.shape)}")
    if cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise TypeError("cos and sin must be float32")
    if not 2 <= 2 * table[1] <= shape[3]:
        raise ValueError(f"tables of {table[1]} pairs do not fit heads of {shape[3]} features")
    if positions is not None:
        if positions.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"positions must be int32 or int64, got {positions.dtype}")
        if positions.shape not in (shape[1:2], shape[:2]):
            raise ValueError(f"positions must be (seq,) or (batch, seq), got {tuple(positions.shape)}")
    for t in (k, cos, sin, positions):
        if t is not None and t.get_device() != index:
            raise RuntimeError(f"rotary: tensors on {t.device} and {q.device}")


class RotaryFunction(torch.autograd.Function):
    """Linear in q and k: nothing of them is kept, the backward is the turn by the negative angles."""

    @staticmethod
    def forward(ctx, q, k, cos, sin, positions, offset, layout):
        ctx.save_for_backward(cos, sin, positions)
        ctx.offset, ctx.layout = offset, layout
        qo, ko = kernels.rotary(q, k, cos, sin, positions, offset, layout)
        return qo if k is None else (qo, ko)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk=None):
        cos, sin, positions = ctx.saved_tensors
        dq, dk = kernels.rotary(dq, dk, cos, sin, positions, ctx.offset, ctx.layout, inverse=True)
        return dq, dk, None, None, None, None, None


def rotary(q: torch.Tensor, k: torch.Tensor | None, cos: torch.Tensor, sin: torch.Tensor, *,
           positions: torch.Tensor | None = None, offset: int = 0, layout: str = "half", inplace: bool = False):
    """(q, k) turned by their positions' angles; q alone (and returned alone) with ``k`` None.

    q, k: batch x seq x heads x head with any strides of the first three (views of a fused projection
    and transposed tensors are taken as they are); k may have fewer heads.  The first 2 * cos.shape[1]
    features of each head are turned, the rest copied.  ``layout`` "half" pairs (j, j + rot / 2),
    "interleaved" (2 j, 2 j + 1).  ``positions`` (seq,) or (batch, seq), or None for ``offset`` + index;
    a position outside the tables gives NaN.  ``inplace`` overwrites q and k (no gradient through it).
    """
    _check_rotary(q, k, cos, sin, positions, layout)
    if positions is None and (offset < 0 or offset + q.shape[1] > cos.shape[0]):
        raise ValueError(f"positions {offset} .. {offset + q.shape[1]} are outside tables of {cos.shape[0]}")
    cos, sin = cos.contiguous(), sin.contiguous()
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        if inplace:
            raise ValueError("rotary in place has no gradient: pass inplace=False or use it under torch.no_grad()")
        return RotaryFunction.apply(q, k, cos, sin, positions, int(offset), layout)
    if inplace:
        for name, t in (("queries", q), ("keys", k)):
            if t is not None and ((t.stride(3) != 1 and t.shape[3] > 1) or _overlaps(t)):
                raise ValueError(f"rotary in place needs {name} with contiguous features that do not share memory")
    qo, ko = kernels.rotary(q, k, cos, sin, positions, offset, layout, inplace=inplace)
    return qo if k is None else (qo, ko)


def _overlaps(t) -> bool:
    """Whether two elements of a strided tensor may share memory (a dimension's stride is within the span of
    the smaller ones)."""
    span = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if stride < span:
            return True
        span = stride * (size - 1) + span
    return False


__all__ = ["RotaryFunction", "rotary", "rotary_tables"]
