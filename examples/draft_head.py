"""A draft head over a truncated vocabulary, from training to speculative decoding.

    python examples/draft_head.py [--steps 60]

1. Train: the head's projection [Vd, K] learns a fixed target model's next tokens from its
   hidden states, by the cross entropy over the draft vocabulary (targets outside it count
   for nothing).
2. Pack: the trained projection goes into 4 bits with group scales.
3. Serve: each round drafts a token per stream from the packed projection, and the target's
   logits accept or replace it.

The target model is synthetic: its hidden states are drawn at random and its projection is
fixed, so that the script needs no checkpoint.
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "strim-engine_amd"))

from strim_amd import _native as N  # noqa: E402
from strim_amd import loss, ops  # noqa: E402


def states(target: torch.Tensor, rows: int, g: torch.Generator):
    """Hidden states of a model that mostly knows its next token, and those tokens: the
    commoner the smaller their id."""
    V, K = target.shape
    dev = target.device
    u = torch.rand(rows, device=dev, generator=g)
    tokens = (V * u ** 3).long().clamp_max(V - 1)
    h = torch.randn(rows, K, device=dev, generator=g)
    h += 0.25 * K ** 0.5 * target[tokens].float()
    return h.to(torch.bfloat16), tokens


def run(V: int = 16_384, Vd: int = 4_096, K: int = 1_024, rows: int = 2_048, streams: int = 8,
        steps: int = 60, lr: float = 2.0, verbose: bool = True) -> dict:
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev)
    g.manual_seed(0)
    target = torch.randn(V, K, device=dev, generator=g).to(torch.bfloat16)
    table = torch.arange(Vd, device=dev, dtype=torch.int32)  # draft id -> id of the vocabulary
    to_draft = torch.full((V,), loss.IGNORE, dtype=torch.int64, device=dev)
    to_draft[table.long()] = torch.arange(Vd, device=dev)

    # 1. train: float32 weights, their bf16 copy in the products
    master = torch.zeros(Vd, K, device=dev)
    losses = []
    for _ in range(steps):
        h, tokens = states(target, rows, g)
        head = master.to(torch.bfloat16).requires_grad_()
        value = loss.head_cross_entropy(h, head, to_draft[tokens])
        value.backward()
        master -= lr * head.grad.float()
        losses.append(value.detach())
    losses = torch.stack(losses).tolist()

    # 2. pack
    trained = master.to(torch.bfloat16)
    packed = ops.q4_pack(trained, group=64)
    held = sum(t.numel() * t.element_size() for t in (packed.words, packed.scales, packed.biases))

    # 3. serve: the drafts of 16-bit and packed weights, verified by the target's logits
    ctx = ops.Context(0, max_rows=2 * streams, max_vocab=V)
    accepted = {}
    for name in ("bf16", "4 bits"):
        g.manual_seed(1)
        hits = rounds = 0
        for _ in range(16):
            h, _ = states(target, streams, g)
            logits = ops.head_logits(h, trained) if name == "bf16" else ops.head_logits_q4(h, packed)
            drafts = ops.draft_argmax(logits, table)
            # the target's rows: after the pending token, and after the draft
            nxt, _ = states(target, streams, g)
            rows_t = torch.stack([ops.head_logits(h, target), ops.head_logits(nxt, target)], 1)
            out = ctx.verify(rows_t, drafts[:, None], N.params_array(streams, temperature=0.0))
            hits += int(out["accepted"].sum())
            rounds += streams
        accepted[name] = hits / rounds
    # how far the packed head's log-probabilities of the training targets moved
    h, tokens = states(target, rows, g)
    live = to_draft[tokens] >= 0
    t = torch.where(live, to_draft[tokens], 0)
    lp = loss.token_logprobs(h, trained, t)[live].mean()
    lq = loss.token_logprobs(h, ops.q4_unpack(packed), t)[live].mean()
    ctx.close()
    result = dict(loss_first=losses[0], loss_last=losses[-1], accepted=accepted,
                  bytes_bf16=2 * Vd * K, bytes_packed=held, logprob_bf16=float(lp),
                  logprob_packed=float(lq))
    if verbose:
        print(f"loss {losses[0]:.3f} -> {losses[-1]:.3f} over {steps} steps")
        print(f"projection {2 * Vd * K / 1e6:.1f} MB -> {held / 1e6:.1f} MB; mean log-probability of the "
              f"targets {float(lp):.3f} -> {float(lq):.3f}")
        print("drafts accepted: " + ", ".join(f"{k} {v:.2f}" for k, v in accepted.items()))
    return result


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=60)
    run(steps=ap.parse_args().steps)
