"""Training and scoring over the vocabulary: the differentiable forms of ops.head_loss,
ops.token_scores and ops.distill.

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


class _TokenScores(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, top, temperature, mask, ignore_index):
        out = ops.token_scores(logits, tokens, top, temperature, mask, ignore_index)
        ctx.save_for_backward(logits, tokens, mask, out.lse, out.entropy)
        ctx.args = temperature, ignore_index
        ctx.mark_non_differentiable(*(t for t in (out.top_ids, out.top_logprobs, out.status)
                                      if t is not None))
        ctx.set_materialize_grads(False)
        return tuple(out)

    @staticmethod
    @once_differentiable
    def backward(ctx, g_logprobs, g_entropy, g_lse, *_):
        logits, tokens, mask, lse, entropy = ctx.saved_tensors
        temperature, ignore_index = ctx.args
        g = [None if t is None else t.float().contiguous() for t in (g_logprobs, g_entropy, g_lse)]
        d = ops.token_scores_grad(logits, tokens, lse, entropy, *g, temperature=temperature, mask=mask,
                                  ignore_index=ignore_index)
        return d, None, None, None, None, None


def _rows(logits: torch.Tensor) -> torch.Tensor:
    """[..., V] as [R, V] with contiguous rows."""
    rows = ops.as_rows(logits)
    # (one row broadcast over several has a stride of 0)
    apart = rows.stride(1) == 1 and (rows.shape[0] < 2 or rows.stride(0) >= rows.shape[1])
    return rows if apart else rows.contiguous()


def token_scores(logits: torch.Tensor, tokens: torch.Tensor | None = None, top: int = 0,
                 temperature: float = 1.0, mask: torch.Tensor | None = None,
                 ignore_index: int = IGNORE) -> ops.TokenScores:
    """ops.token_scores over logits [..., V], with gradients for the logits through the tokens'
    log-probabilities, the entropy and the log-sum-exp (first derivatives; the alternatives have none).
    tokens int32 or int64 [...] or [..., S], mask [..., words]; results have the same leading shape."""
    lead, V = logits.shape[:-1], logits.shape[-1]
    given = None
    if tokens is not None:
        if tokens.shape[:len(lead)] != lead or tokens.dim() > len(lead) + 1:
            raise ValueError(f"tokens must be {tuple(lead)} or {tuple(lead)} + (n,), got {tuple(tokens.shape)}")
        given = tokens.shape
        R = lead.numel()
        tokens = _ids(tokens.reshape((R,) if tokens.dim() == len(lead) else (R, tokens.shape[-1])), V,
                      ignore_index)
    if mask is not None:
        if mask.shape[:-1] != lead:
            raise ValueError(f"mask must be {tuple(lead)} + (words,), got {tuple(mask.shape)}")
        mask = ops.as_rows(mask).contiguous()
    out = _TokenScores.apply(_rows(logits), tokens, top, temperature, mask, ignore_index)
    lp, entropy, lse, ids, ilp, status = out
    return ops.TokenScores(None if lp is None else lp.reshape(given), entropy.reshape(lead),
                           lse.reshape(lead), None if ids is None else ids.reshape(*lead, top),
                           None if ilp is None else ilp.reshape(*lead, top), status.reshape(lead))


class _Distill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, logprobs, temperature, tail):
        loss, lse, log_rest, status = ops.distill(logits, ids, logprobs, temperature, tail)
        ctx.save_for_backward(logits, ids, logprobs, lse, log_rest)
        ctx.args = temperature, tail
        ctx.mark_non_differentiable(status)
        ctx.set_materialize_grads(False)
        return loss, status

    @staticmethod
    @once_differentiable
    def backward(ctx, g_loss, _):
        if g_loss is None:
            return None, None, None, None, None
        logits, ids, logprobs, lse, log_rest = ctx.saved_tensors
        temperature, tail = ctx.args
        d = ops.distill_grad(logits, ids, logprobs, lse, log_rest, g_loss.float().contiguous(),
                             temperature, tail)
        return d, None, None, None, None


def _sum(t: torch.Tensor) -> torch.Tensor:
    """The sum of [N] numbers by one workgroup a time: over many numbers at once the library's sum
    clears a counter, which is not safe to replay from a captured graph."""
    while t.shape[0] > 4096:
        t = torch.nn.functional.pad(t, (0, -t.shape[0] % 1024)).view(-1, 1024).sum(1)
    return t.sum()


class _DistillSum(torch.autograd.Function):
    """The rows' losses times their weights, summed; the gradient comes with the loss, from one step."""

    @staticmethod
    def forward(ctx, logits, ids, logprobs, weights, temperature, tail):
        if ctx.needs_input_grad[0]:
            loss, ctx.d, _ = ops.distill_step(logits, ids, logprobs, weights, temperature, tail)
            ctx.save_for_backward(logits, ids, logprobs, weights)
            ctx.args = temperature, tail
        else:
            loss = ops.distill(logits, ids, logprobs, temperature, tail)[0]
        # (a row of weight 0 counts for nothing, an infinite or NaN loss included)
        return _sum(torch.where(weights != 0, loss * weights, 0.0))

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        logits, ids, logprobs, weights = ctx.saved_tensors
        d, ctx.d = ctx.d, None
        if d is None:  # (a second pass over a retained graph: the first one's result is the caller's)
            d = ops.distill_step(logits, ids, logprobs, weights, *ctx.args)[1]
        return ops.distill_scale(d, g.float().reshape(1)), None, None, None, None, None


def _alternatives(logits, ids, logprobs):
    lead = logits.shape[:-1]
    if ids.shape[:-1] != lead or logprobs.shape != ids.shape:
        raise ValueError(f"ids and logprobs must be {tuple(lead)} + (M,), got {tuple(ids.shape)} and "
                         f"{tuple(logprobs.shape)}")
    V = logits.shape[-1]
    if ids.dtype == torch.int64:  # (one past 32 bits stays outside the vocabulary)
        ids = torch.where(ids < 0, -1, ids.clamp_max(V)).to(torch.int32)
    if ids.dtype != torch.int32:
        raise TypeError(f"ids must be int32 or int64, got {ids.dtype}")
    if logprobs.requires_grad:
        raise ValueError("the teacher's log-probabilities take no gradient: detach them")
    return ops.as_rows(ids).contiguous(), ops.as_rows(logprobs).float().contiguous()


def distill_loss(logits: torch.Tensor, ids: torch.Tensor, logprobs: torch.Tensor,
                 temperature: float = 1.0, tail: bool = False, reduction: str = "mean") -> torch.Tensor:
    """Divergence of softmax(logits / temperature) from a teacher's alternatives (ids and logprobs
    [..., M], as token_scores gives them), with gradients for the logits [..., V] (first derivatives):
    "mean" over the positions that have alternatives (0 if none has), "sum", or "none" (per position).
    The mean and the sum make their gradient with the loss (ops.distill_step) and hold it until the
    backward pass; the gradient is then multiplied by what comes back, in a pass of its own unless that
    is 1 (and rounded again unless that is a power of two). "none" takes it from lse and log_rest as
    float32 holds them (ops.distill_grad)."""
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"reduction must be mean, sum or none, got {reduction}")
    lead, V = logits.shape[:-1], logits.shape[-1]
    ids, logprobs = _alternatives(logits, ids, logprobs)
    rows = _rows(logits)
    if reduction == "none":
        return _Distill.apply(rows, ids, logprobs, temperature, tail)[0].reshape(lead)
    if reduction == "sum":
        weights = torch.ones(rows.shape[0], dtype=torch.float32, device=rows.device)
    else:
        live = ((ids >= 0) & (logprobs != float("-inf"))).any(1) & (ids < V).all(1)
        weights = live.float()
        weights = weights / _sum(weights).clamp_min(1.0)  # (counts are exact in float32 up to 2^24)
    if not torch.is_grad_enabled():  # (nothing is recorded, though the logits may ask for a gradient)
        rows = rows.detach()
    return _DistillSum.apply(rows, ids, logprobs, weights, temperature, tail)
