"""The gated feed-forward block h = act(x Wg^T + bg) * (x Wu^T + bu) and its gradients in HIP kernels.

``gated_feed_forward`` is the exact operator: one kernel forms both projections, the activation and the
product, and nothing but the input is kept for the backward, which forms the pre-activations again.
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
    """Saved tensors: the input, both weights and the biases (all of them the caller's own)."""

    @staticmethod
    def forward(ctx, x, w_gate, w_up, b_gate, b_up, activation):
        ctx.save_for_backward(x, w_gate, w_up, b_gate, b_up)
        ctx.activation = activation
        h = kernels.gated_forward(x.reshape(-1, x.shape[-1]), w_gate, w_up, _contiguous(b_gate), _contiguous(b_up),
                                  activation)
        return h.view(*x.shape[:-1], h.shape[1])

    @staticmethod
    @once_differentiable
    def backward(ctx, dh):
        x, w_gate, w_up, b_gate, b_up = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dwg, dwu, dbg, dbu, _ = kernels.gated_backward(
            dh.reshape(-1, dh.shape[-1]), x.reshape(-1, x.shape[-1]), w_gate, w_up, _contiguous(b_gate),
            _contiguous(b_up), ctx.activation, needs=(need[0], need[1] or need[2], need[3], need[4]))
        return (dx.view(x.shape) if dx is not None else None, dwg if need[1] else None, dwu if need[2] else None, dbg,
                dbu, None)


def gated_feed_forward(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, b_gate: torch.Tensor | None = None,
                       b_up: torch.Tensor | None = None, *, activation: str = "silu") -> torch.Tensor:
    """act(x w_gate^T + b_gate) * (x w_up^T + b_up) over the last dimension of ``x``, differentiable.

    Weights as nn.Linear keeps them, (ff, d); one of float32, bfloat16, float16 throughout (under
    autocast everything is cast to its type first).  ``activation``: "silu", "gelu", "gelu_tanh", "relu"
    or "sigmoid".  Sums in fp32, one rounding at the end; the backward rounds dg and du to the type
    between its products.
    """
    if torch.is_autocast_enabled(x.device.type):
        dtype = torch.get_autocast_dtype(x.device.type)
        x, w_gate, w_up, b_gate, b_up = (None if t is None else t.to(dtype) for t in (x, w_gate, w_up, b_gate, b_up))
    _check_gated(x, w_gate, w_up, b_gate, b_up, activation)
    if torch.is_grad_enabled() and (x.requires_grad or w_gate.requires_grad or w_up.requires_grad or
                                    (b_gate is not None and b_gate.requires_grad) or
                                    (b_up is not None and b_up.requires_grad)):
        return GatedFeedForwardFunction.apply(x, w_gate, w_up, b_gate, b_up, activation)
    if x.dim() == 2:
        return kernels.gated_forward(x, w_gate, w_up, _contiguous(b_gate), _contiguous(b_up), activation)
    h = kernels.gated_forward(x.reshape(-1, x.shape[-1]), w_gate, w_up, _contiguous(b_gate), _contiguous(b_up),
                              activation)
    return h.view(*x.shape[:-1], h.shape[1])


__all__ = ["ACTIVATIONS", "GatedFeedForwardFunction", "gated_feed_forward"]
