"""The gated feed-forward block h = act(x Wg^T + bg) * (x Wu^T + bu) and its gradients in HIP kernels.

``gated_feed_forward`` is the exact operator: one kernel forms both projections, the activation and the
product.  ``STACRGatedFeedForward`` is the block with its input compressed as STACRLinear compresses it: one
save serves both projections, whose weight gradients come from one call on [dg | du].
(No counterpart in the reference, whose layers wrap the projections one by one.)
"""
from __future__ import annotations

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _lib, kernels
from .layers import STACRLinear, _save_factors

ACTIVATIONS = tuple(_lib.ACTIVATION_CODES)


def _check_gated(x, w_gate, w_up, b_gate, b_up, activation) -> None:
    # the usual case in few steps: a call on a single token is bound by the host
    dtype, index, shape = x.dtype, x.get_device(), w_gate.shape
    if (b_gate is None and b_up is None and index >= 0 and activation in _lib.ACTIVATION_CODES and len(shape) == 2 and
            shape == w_up.shape and shape[0] and x.shape[-1:] == shape[1:] and w_gate.dtype is dtype and
            w_up.dtype is dtype and w_gate.get_device() == index and w_up.get_device() == index and shape[1]):
        return
    if activation not in _lib.ACTIVATION_CODES:
        raise ValueError(f"activation must be one of {list(ACTIVATIONS)}, got {activation!r}")
    kernels.require_gpu(x, "input")
    if len(shape) != 2 or shape != w_up.shape or 0 in shape:
        raise ValueError(f"w_gate and w_up must be two (ff, d) matrices of one shape, got {tuple(shape)} and "
                         f"{tuple(w_up.shape)}")
    if x.shape[-1:] != shape[1:]:
        raise ValueError(f"Expected last input dimension {shape[1]}, got {tuple(x.shape)}")
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
        h, kept = (h, None) if recompute else h
        ctx.save_for_backward(x, w_gate, w_up, b_gate, b_up, kept)
        ctx.activation = activation
        return h if x.dim() == 2 else h.view(*x.shape[:-1], h.shape[1])

    @staticmethod
    @once_differentiable
    def backward(ctx, dh):
        x, w_gate, w_up, b_gate, b_up, kept = ctx.saved_tensors
        need = ctx.needs_input_grad
        if x.dim() != 2:
            dh, x2d = dh.reshape(-1, dh.shape[-1]), x.reshape(-1, x.shape[-1])
        else:
            x2d = x
        dx, dwg, dwu, dbg, dbu, _ = kernels.gated_backward(
            dh, x2d, w_gate, w_up, _contiguous(b_gate), _contiguous(b_up), ctx.activation,
            kept, (need[0], need[1] or need[2], need[3], need[4]))
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
    if torch.is_autocast_enabled("cuda"):
        dtype = torch.get_autocast_dtype("cuda")
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


class STACRGatedFunction(torch.autograd.Function):
    """Exact forward and input gradient; weight gradients from the input's saved factors.

    Saved tensors: both weights and biases, coefficients, basis, the residual's indices, values and scale,
    and the two pre-activations in the type (the input itself is not kept, so they cannot be formed again).
    """

    @staticmethod
    def forward(ctx, x, w_gate, w_up, b_gate, b_up, basis, budget, bits, chunk_rows, mode, block_size, sample_ratio,
                activation):
        x2d = x.reshape(-1, x.shape[-1])
        h, kept = kernels.gated_forward(x2d, w_gate, w_up, _contiguous(b_gate), _contiguous(b_up), activation, "type")
        if mode == "none":
            mode, budget = "chunk_topk", 0.0
        coeff, idx, data, scale, census, bits, _ = _save_factors(x2d, basis.to(x.dtype), mode, float(budget), int(bits),
                                                                 int(chunk_rows), int(block_size), float(sample_ratio))
        ctx.save_for_backward(w_gate, w_up, b_gate, b_up, coeff, basis.to(x.dtype), idx, data, scale, kept)
        # the save's entry census (an intermediate, outside the saved tensors): the weight gradient need not count
        ctx.census = census if idx is not None else None
        ctx.bits, ctx.shape, ctx.activation = bits if idx is not None else 0, x.shape, activation
        return h.view(*x.shape[:-1], h.shape[1])

    @staticmethod
    @once_differentiable
    def backward(ctx, dh):
        w_gate, w_up, b_gate, b_up, coeff, q, idx, data, scale, kept = ctx.saved_tensors
        need = ctx.needs_input_grad
        weights = need[1] or need[2]
        with torch.autocast(device_type=dh.device.type, enabled=False):
            dx, _, _, dbg, dbu, dgu = kernels.gated_backward(
                dh.reshape(-1, dh.shape[-1]), None, w_gate, w_up, _contiguous(b_gate), _contiguous(b_up), ctx.activation,
                kept, (need[0], False, need[3], need[4]), slopes=weights)
            dwg = dwu = None
            if weights:
                residual = (idx, data, scale) if idx is not None and idx.numel() else None
                dw, _ = kernels.weight_grad(dgu, coeff, q, residual, ctx.bits, False, w_gate.dtype, census=ctx.census)
                ff, pad = w_gate.shape[0], dgu.shape[1] // 2
                dwg, dwu = dw[:ff] if need[1] else None, dw[pad:pad + ff] if need[2] else None
        return (dx.view(ctx.shape) if dx is not None else None, dwg, dwu, dbg, dbu) + (None,) * 8


class STACRGatedFeedForward(nn.Module):
    """act(gate(x)) * up(x) of two projections of one input, whose saved copy is compressed once for both.

    ``gate`` holds the gate projection's parameters and the basis with its schedule (a STACRLinear: set_step on
    a model reaches it); the up projection's are ``up_weight`` and ``up_bias``.  Options as STACRLinear's.
    Eval, no-grad and frozen-weight calls run gated_feed_forward, as do inputs without rows.
    """

    def __init__(self, gate: STACRLinear, up_weight: nn.Parameter, up_bias: nn.Parameter | None, *,
                 activation: str = "silu"):
        super().__init__()
        if activation not in _lib.ACTIVATION_CODES:
            raise ValueError(f"activation must be one of {list(ACTIVATIONS)}, got {activation!r}")
        if gate.transposed:
            raise ValueError("the gate projection must keep its weight as (out, in)")
        if up_weight.shape != gate.weight.shape or up_weight.dtype != gate.weight.dtype:
            raise ValueError(f"gate and up weights differ: {tuple(gate.weight.shape)} {gate.weight.dtype} and "
                             f"{tuple(up_weight.shape)} {up_weight.dtype}")
        if up_bias is not None and up_bias.shape != up_weight.shape[:1]:
            raise ValueError("bias shape must match the output feature count")
        self.gate, self.up_weight, self.up_bias, self.activation = gate, up_weight, up_bias, activation
        self.in_features, self.out_features = gate.in_features, gate.out_features

    @classmethod
    def from_linears(cls, gate: nn.Linear, up: nn.Linear, *, activation: str = "silu", **options) -> "STACRGatedFeedForward":
        """The block of two nn.Linear layers, whose parameters it takes over."""
        if not (isinstance(gate, nn.Linear) and isinstance(up, nn.Linear)):
            raise TypeError("from_linears requires two nn.Linear layers")
        block = cls(STACRLinear.from_linear(gate, **options), up.weight, up.bias, activation=activation)
        return block.train(gate.training)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.ndim < 1 or x.shape[-1] != self.in_features:
            raise ValueError(f"Expected last input dimension {self.in_features}, got {tuple(x.shape)}")
        gate = self.gate
        w = [gate.weight, self.up_weight, gate.bias, self.up_bias]
        if not (self.training and torch.is_grad_enabled() and x.numel() > 0 and
                (gate.weight.requires_grad or self.up_weight.requires_grad)):
            return gated_feed_forward(x, *w, activation=self.activation)
        if torch.is_autocast_enabled("cuda"):
            dtype = torch.get_autocast_dtype("cuda")
            x, *w = (None if t is None else t.to(dtype) for t in (x, *w))
        _check_gated(x, *w, self.activation)
        basis, budget = gate._factor_state(x)
        with torch.autocast(device_type=x.device.type, enabled=False):
            return STACRGatedFunction.apply(x, *w, basis, budget, gate.residual_bits, gate.chunk_rows, gate.residual_mode,
                                            gate.residual_block_size, gate.residual_sample_ratio, self.activation)

    def stored_bytes(self, rows: int, value_bytes: int = 2) -> dict:
        """STACRLinear.stored_bytes of the shared input, and the kept pre-activations."""
        stored = self.gate.stored_bytes(rows, value_bytes)
        each = int(rows) * ((self.out_features + 7) // 8 * 8) * value_bytes
        stored["preactivations"] = 2 * ((each + 255) // 256 * 256)
        stored["total"] += stored["preactivations"]
        return stored


__all__ = ["ACTIVATIONS", "GatedFeedForwardFunction", "STACRGatedFeedForward", "STACRGatedFunction",
           "gated_feed_forward"]
