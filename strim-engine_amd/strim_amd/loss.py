"""Training and scoring over the vocabulary: the differentiable form of ops.head_loss.

Cross entropy of a vocabulary projection's logits against target ids, over the whole
vocabulary and without keeping the logits, for training (or distilling) a draft head over its
truncated vocabulary, and the log-probabilities of given tokens. The reference trains
nothing; its counterpart is the projection itself (Sources/StrimCore/QwenModel.swift:202-212)
and the draft head's over the truncated vocabulary (Sources/StrimCore/MTP.swift:104-125).
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import ops

IGNORE = -100


def _ids(targets: torch.Tensor, V: int, ignore_index: int) -> torch.Tensor:
    """int32 target ids: an id outside [0, V) that is not ignored stays so (also one past 32 bits)."""
    ops.check_ignore_index(ignore_index)
    if targets.dtype == torch.int32:
        return targets.contiguous()
    if targets.dtype != torch.int64:
        raise TypeError(f"targets must be int32 or int64, got {targets.dtype}")
    inside = (targets >= 0) & (targets < V)
    outside = V if ignore_index != V else -1
    kept = torch.where(targets == ignore_index, ignore_index, torch.where(inside, targets, outside))
    return kept.to(torch.int32)


class _HeadLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, lm_head, targets, ignore_index):
        loss, lse, status = ops.head_loss(hidden, lm_head, targets, ignore_index)
        ctx.save_for_backward(hidden, lm_head, targets, lse)
        ctx.ignore_index = ignore_index
        ctx.mark_non_differentiable(status)
        ctx.set_materialize_grads(False)  # (an output that is not used has no gradient, not zeros)
        return loss, lse, status

    @staticmethod
    @once_differentiable  # (the gradients' own derivatives are not built: asking for them raises)
    def backward(ctx, g_loss, g_lse, _):
        hidden, lm_head, targets, lse = ctx.saved_tensors
        # (a sum's or a mean's gradient comes as one number broadcast over the rows)
        g_loss = torch.zeros_like(lse) if g_loss is None else g_loss.float().contiguous()
        g_lse = None if g_lse is None else g_lse.float().contiguous()
        dh, dw = ops.head_loss_grad(hidden, lm_head, targets, lse, g_loss, g_lse,
                                    want_hidden=ctx.needs_input_grad[0],
                                    want_lm_head=ctx.needs_input_grad[1],
                                    ignore_index=ctx.ignore_index)
        return dh, dw, None, None


def head_loss(hidden: torch.Tensor, lm_head: torch.Tensor, targets: torch.Tensor,
              ignore_index: int = IGNORE):
    """Per-position (loss, lse, status), as ops.head_loss, with gradients for hidden bf16
    [..., K] and lm_head bf16 [V, K] through loss and lse (first derivatives: differentiating a
    gradient raises). targets int32 or int64 [...]."""
    shape = hidden.shape[:-1]
    if targets.shape != shape:
        raise ValueError(f"targets must be {tuple(shape)}, got {tuple(targets.shape)}")
    rows = hidden.reshape(-1, hidden.shape[-1])
    out = _HeadLoss.apply(rows, lm_head, _ids(targets.reshape(-1), lm_head.shape[0], ignore_index),
                          ignore_index)
    return tuple(t.reshape(shape) for t in out)


def head_cross_entropy(hidden: torch.Tensor, lm_head: torch.Tensor, targets: torch.Tensor,
                       ignore_index: int = IGNORE, reduction: str = "mean") -> torch.Tensor:
    """Cross entropy over the vocabulary: "mean" over the positions that have a target (0 if
    none has), "sum", or "none"."""
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"reduction must be mean, sum or none, got {reduction}")
    loss, _, _ = head_loss(hidden, lm_head, targets, ignore_index)
    if reduction == "none":
        return loss
    if reduction == "sum":
        return loss.sum()
    live = (targets != ignore_index) & (targets >= 0) & (targets < lm_head.shape[0])
    return loss.sum() / live.sum().clamp_min(1)


def token_logprobs(hidden: torch.Tensor, lm_head: torch.Tensor, tokens: torch.Tensor) -> torch.Tensor:
    """log p(token) of each position under its projected distribution (temperature 1, no
    filters), float32; 0 where the token is not an id of the vocabulary."""
    return -head_loss(hidden, lm_head, tokens)[0]
