"""Norms with gradients: the differentiable forms of ops.norm.

The projection normalises its hidden rows on the way in (ops.head_logits, the reference's
Sources/StrimCore/Weights.swift:270-273), without a gradient; training a head through its norm
takes these.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import ops


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, center):
        y, rstd, mean = ops.norm(x, weight, bias, eps, center)
        ctx.save_for_backward(x, weight, bias, rstd, mean)
        return y

    @staticmethod
    @once_differentiable  # (the gradients' own derivatives are not built: asking for them raises)
    def backward(ctx, g):
        x, weight, bias, rstd, mean = ctx.saved_tensors
        if not g.is_contiguous() and (g.stride(1) != 1 or g.stride(0) < g.shape[1]):
            g = g.contiguous()  # (a sum's gradient is one number broadcast)
        want = ctx.needs_input_grad
        dx, dw, db = ops.norm_grad(x, weight, bias, g, rstd, mean, want_x=want[0], want_weight=want[1],
                                   want_bias=want[2])
        return dx, dw, db, None, None


def _norm(x, weight, bias, eps, center):
    rows = ops.as_rows(x)
    if rows.stride(1) != 1 or (rows.shape[0] > 1 and rows.stride(0) < rows.shape[1]):
        rows = rows.contiguous()  # (one row broadcast over several has a stride of 0)
    return _Norm.apply(rows, weight, bias, eps, center).reshape(x.shape)


def rms_norm(x: torch.Tensor, weight: torch.Tensor | None = None, eps: float = 1e-6) -> torch.Tensor:
    """x / sqrt(mean x^2 + eps) weight over the last dimension, in float32, rounded once to x's type
    (bf16 or float32); gradients for x and weight (first derivatives)."""
    return _norm(x, weight, None, eps, False)


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(variance + eps) weight + bias over the last dimension, as rms_norm."""
    return _norm(x, weight, bias, eps, True)
