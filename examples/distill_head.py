"""A head distilled from a teacher's alternatives.

    python examples/distill_head.py [--steps 60]

1. Teach: the teacher's logits become its `top` most probable ids and their log-probabilities, all
   that is kept of them (ops.token_scores).
2. Train: the student's states pass a norm and a projection, and the divergence from the alternatives
   (the rest of the teacher's mass as one more) goes back to the projection and the norm's weights.
3. Score: log-probabilities of the teacher's first ids and entropies under the student.

The teacher is synthetic: a fixed projection of states drawn at random, of which the student sees a
part, so that the script needs no checkpoint.
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "strim-engine_amd"))

from strim_amd import loss, norm, ops  # noqa: E402


def gradients(states, weight, head, alternatives, temperature=1.0):
    """The mean divergence from a teacher's alternatives, and its gradients for the norm's weights and
    the projection."""
    weight, head = (t.detach().requires_grad_() for t in (weight, head))
    logits = norm.rms_norm(states, weight) @ head.t()
    value = loss.distill_loss(logits, alternatives.top_ids, alternatives.top_logprobs, temperature, tail=True)
    return value.detach(), *torch.autograd.grad(value, (weight, head))


def run(V: int = 8_192, K: int = 512, rows: int = 1_024, top: int = 32, steps: int = 60, lr: float = 30.0,
        verbose: bool = True) -> dict:
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev)
    g.manual_seed(0)
    teacher = (4.0 * K ** -0.5 * torch.randn(V, 2 * K, device=dev, generator=g)).to(torch.bfloat16)
    weight, head = torch.ones(K, device=dev), torch.zeros(V, K, device=dev)
    losses = []
    for _ in range(steps):
        h = torch.randn(rows, 2 * K, device=dev, generator=g).to(torch.bfloat16)
        # 1. what is kept of the teacher: [rows, top] ids and log-probabilities
        kept = ops.token_scores(h @ teacher.t(), top=top)
        # 2. one step: float32 weights, their bf16 copies in the products
        value, d_weight, d_head = gradients(h[:, :K].contiguous(), weight.to(torch.bfloat16),
                                            head.to(torch.bfloat16), kept)
        weight -= 1e-3 * lr * d_weight.float()  # (each of its entries is in every logit)
        head -= lr * d_head.float()
        losses.append(value)
    # 3. the student about the teacher's first ids
    logits = norm.rms_norm(h[:, :K], weight.to(torch.bfloat16)) @ head.to(torch.bfloat16).t()
    scores = ops.token_scores(logits, kept.top_ids[:, 0].contiguous())
    losses = torch.stack(losses).tolist()
    result = dict(loss_first=losses[0], loss_last=losses[-1], logprob=float(scores.logprobs.mean()),
                  entropy=float(scores.entropy.mean()), kept_bytes=8 * rows * top, logits_bytes=2 * rows * V)
    if verbose:
        print(f"divergence {losses[0]:.3f} -> {losses[-1]:.3f} over {steps} steps; kept of a step's logits "
              f"{result['kept_bytes'] / 1e6:.2f} of {result['logits_bytes'] / 1e6:.1f} MB")
        print(f"the teacher's first ids under the student: mean log-probability {result['logprob']:.3f}, "
              f"mean entropy {result['entropy']:.3f}")
    return result


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=60)
    run(steps=ap.parse_args().steps)
