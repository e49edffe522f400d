"""The gated feed-forward block h = act(x Wg^T + bg) * (x Wu^T + bu) and its gradients in HIP kernels.

``gated_feed_forward`` is the exact operator: one kernel forms both projections, the activation and the
product.
(No counterpart in the reference, whose layers wrap the projections one by one.)
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib, kernels

ACTIVATIONS = tuple(_lib.ACTIVATION_CODES)


def _check_gated(x, w_gate, w_up, b_gate, b_up, activation) -> None:
    if activation not in _lib.ACTIVATION_CODES:
        raise ValueError(f"activation must be one of {list(ACTIVATIONS)}, got {activation!r}")
    kernels.require_gpu(x, "input")
    shape = w_gate.shape
    if len(shape) != 2 or shape != w_up.shape or 0 in shape:
        raise ValueError(f"w_gate and w_up must be two (ff, d) matrices of one shape, got {tuple(shape)} and "
                         f"{tuple(w_up.shape)}")
    if x.dim() < 1 or x.shape[-1] != shape[1]:
        raise ValueError(f"Expected last input dimension {shape[1]}, got {tuple(x.shape)}")
    dtype, index = x.dtype, x.get_device()
    for name, t in (("w_gate", w_gate), ("w_up", w_up), ("b_gate", b_gate), ("b_up", b_up)):
        if t is None:
            continue
        if t.get_device() != index:
            raise RuntimeError(f"{name} is on {t.device}, the input on {x.device}")
        if t.dtype != dtype:
            raise TypeError(f"{name} is {t.dtype}, the input {dtype}: one type throughout")
        if name[0] == "b" and t.shape != shape[:1]:
            raise ValueError(f"{name} must have {shape[0]} values, got shape {tuple(t.shape)}")


def _contiguous(t):
    return None if t is None else t.contiguous()


class GatedFeedForwardFunction(torch.autograd.Function):
    """Saved tensors: the input, both weights, the biases (all of them the caller's own) and, unless the
    backward is to compute them again, the pre-activations."""

    @staticmethod
    def forward(ctx, x, w_gate, w_up, b_gate, b_up, activation, recompute):
        x2d = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
        h = kernels.gated_forward(x2d, w_gate, w_up, _contiguous(b_gate), _contiguous(b_up), activation,
                                  None if recompute else "full")
        kept = (None,) * 4
        if not recompute:
            h, kept = h
        ctx.save_for_backward(x, w_gate, w_up, b_gate, b_up, *kept)
        ctx.activation = activation
        return h if x.dim() == 2 else h.view(*x.shape[:-1], h.shape[1])

    @staticmethod
    @once_differentiable
    def backward(ctx, dh):
        x, w_gate, w_up, b_gate, b_up, *kept = ctx.saved_tensors
        need = ctx.needs_input_grad
        if x.dim() != 2:
            dh, x2d = dh.reshape(-1, dh.shape[-1]), x.reshape(-1, x.shape[-1])
        else:
            x2d = x
        dx, dwg, dwu, dbg, dbu, _ = kernels.gated_backward(
            dh, x2d, w_gate, w_up, _contiguous(b_gate), _contiguous(b_up), ctx.activation,
            None if kept[0] is None else kept, (need[0], need[1] or need[2], need[3], need[4]))
        if dx is not None and x.dim() != 2:
            dx = dx.view(x.shape)
        return dx, dwg if need[1] else None, dwu if need[2] else None, dbg, dbu, None, None


def gated_feed_forward(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, b_gate: torch.Tensor | None = None,
                       b_up: torch.Tensor | None = None, *, activation: str = "silu",
                       recompute: bool = False) -> torch.Tensor:
    """act(x w_gate^T + b_gate) * (x w_up^T + b_up) over the last dimension of ``x``, differentiable.

    Weights as nn.Linear keeps them, (ff, d); one of float32, bfloat16, float16 throughout (under
    autocast everything is cast to its type first).  ``activation``: "silu", "gelu", "gelu_tanh", "relu"
    or "sigmoid".  Sums in fp32, one rounding at the end; the backward rounds dg and du to the type
    between its products.

    For the backward the two pre-activations are kept, in 24 bits each (fp32: 32), which costs what eager
    16-bit training keeps of this block (g, act(g) and u).  ``recompute=True`` keeps nothing but the input
    and forms them again in the backward: the same gradients up to the 24 bits' rounding, at a third more work.
    """
    if torch.is_autocast_enabled(x.device.type):
        dtype = torch.get_autocast_dtype(x.device.type)
        x, w_gate, w_up, b_gate, b_up = (None if t is None else t.to(dtype) for t in (x, w_gate, w_up, b_gate, b_up))
    _check_gated(x, w_gate, w_up, b_gate, b_up, activation)
    if torch.is_grad_enabled() and (x.requires_grad or w_gate.requires_grad or w_up.requires_grad or
                                    (b_gate is not None and b_gate.requires_grad) or
                                    (b_up is not None and b_up.requires_grad)):
        return GatedFeedForwardFunction.apply(x, w_gate, w_up, b_gate, b_up, activation, recompute)
    if x.dim() == 2:
        return kernels.gated_forward(x, w_gate, w_up, _contiguous(b_gate), _contiguous(b_up), activation)
    h = kernels.gated_forward(x.reshape(-1, x.shape[-1]), w_gate, w_up, _contiguous(b_gate), _contiguous(b_up),
                              activation)
    return h.view(*x.shape[:-1], h.shape[1])


__all__ = ["ACTIVATIONS", "GatedFeedForwardFunction", "gated_feed_forward"]
