"""The example of a head distilled from a teacher's alternatives: it runs, and its gradients are those of
the loss it names."""
import importlib.util
import math
from pathlib import Path

import pytest
import torch

from strim_amd import ops

pytestmark = pytest.mark.gpu

spec = importlib.util.spec_from_file_location(
    "distill_head", Path(__file__).resolve().parents[1] / "examples" / "distill_head.py")
example = importlib.util.module_from_spec(spec)
spec.loader.exec_module(example)


def test_it_runs():
    print("[example] distilled head", flush=True)
    r = example.run(V=1_000, K=64, rows=96, top=8, steps=3, verbose=False)
    assert all(math.isfinite(v) for v in r.values())


def test_its_gradients():
    print("[example] gradients", flush=True)
    V, K, R, M = 300, 48, 20, 8
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    draw = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    kept = ops.token_scores(draw(R, V), top=M)
    h, w, head = draw(R, K), 1 + 0.1 * draw(K), K ** -0.5 * draw(V, K)
    value, dw, dh = example.gradients(h, w, head, kept)
    w64, head64 = w.double().requires_grad_(), head.double().requires_grad_()
    x = h.double()
    logits = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w64 @ head64.t()
    lq = torch.log_softmax(logits, -1)
    ids, t = kept.top_ids.long(), kept.top_logprobs.double()
    p, rest = t.exp(), lq.exp().scatter(1, ids, 0.0).sum(-1)
    r = 1 - p.sum(-1)
    ref = ((p * (t - lq.gather(1, ids))).sum(-1) + r * (r.log() - rest.log())).mean()
    gw, gh = torch.autograd.grad(ref, (w64, head64))
    # float32 throughout: logits off by K 2^-24 sum |y w| < 48 2^-24 20 = 6e-5, probabilities by as much of themselves
    assert abs(value.item() - ref.item()) <= 2e-4 * abs(ref.item())
    for a, b in ((dw, gw), (dh, gh)):
        assert (a.double() - b).abs().max() <= 2e-4 * b.abs().max()
