"""Operators of the vocabulary projection: what is measured, in plain torch and in this framework.

Three operators over hidden states [N, K] and a projection lm_head [V, K]:

  loss   cross entropy of the projected logits against target ids, over the whole
         vocabulary, without keeping the logits ("score": the loss and the log-sum-exp
         alone), and its gradients ("train": for the hidden states and, unless the
         projection is frozen, for the projection)
  q4     the logits of a few rows from a projection held in 4 bits with group scales
  pack   a projection brought into 4 bits with group scales, and read back

Sizes are those of the repository's configurations (the 151,936-token vocabulary and the
32,768-token draft vocabulary at 5,120 channels, 1 to 64 decode rows) and others of the
same ranges. `own` False: elementary torch operations in 32 bits, rounded once at the end;
True: the framework's calls.
"""
import math
import sys

import torch

own = False

DEV = "cuda:0"

LOSS = dict(op="loss", N=512, K=5120, V=151_936, grad="none", ignored=0.0)
Q4 = dict(op="q4", B=1, K=5120, V=151_936, group=64, symmetric=False, out="bf16")
PACK = dict(op="pack", V=32_768, K=5120, group=64, symmetric=False, dtype="bf16", out="bf16")


def listed():
    return [
        # the log-probability of one token under the draft vocabulary: the smallest call,
        # where launches and latency are all there is
        dict(LOSS, name="score_n1", N=1, K=1024, V=32_768),
        # log-probabilities of a prompt's tokens over the full vocabulary
        dict(LOSS, name="score_n512", N=512),
        # one small accumulation step of a draft head: 96 positions, 10 % of them padding
        dict(LOSS, name="train_n96_draft", N=96, K=1024, V=32_768, grad="both", ignored=0.1),
        # a draft head trained over its truncated vocabulary, a ragged batch of positions
        dict(LOSS, name="train_n2000_draft", N=2000, V=32_768, grad="both", ignored=0.2),
        # states trained against a projection that stays as it is, odd sizes throughout
        dict(LOSS, name="train_frozen_odd", N=1003, K=2056, V=100_003, grad="hidden", ignored=0.1),
        # a training step over the full vocabulary: the largest
        dict(LOSS, name="train_n4096", N=4096, grad="both", ignored=0.1),
        # one token's logits over the full vocabulary from 4-bit weights: single-stream decode
        dict(Q4, name="q4_b1"),
        # a draft step of 8 streams over the truncated vocabulary
        dict(Q4, name="q4_b8_draft", B=8, V=32_768),
        # the largest decode batch, wide groups, float32 logits
        dict(Q4, name="q4_b64", B=64, group=128, out="f32"),
        # a small projection, narrow symmetric groups, an odd number of rows, a verify round's
        # four positions
        dict(Q4, name="q4_b4_small", B=4, K=1024, V=8_193, group=32, symmetric=True),
        # the truncated projection of a draft head brought into 4 bits and read back
        dict(PACK, name="pack_draft"),
        # float32 weights, narrow symmetric groups, an odd number of rows
        dict(PACK, name="pack_f32_odd", V=10_007, K=1280, group=32, symmetric=True, dtype="f32",
             out="f32"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, step):
    """Channels: one of the usual widths, or an odd multiple of `step`."""
    if rng.random() < 0.4:
        return rng.choice([1024, 1280, 2048, 2560, 4096, 5120])
    return step * (2 * (_log_int(rng, 1024, 5120) // (2 * step)) + 1)


def draw(rng):
    op = rng.choice(["score"] * 3 + ["train"] * 5 + ["q4"] * 5 + ["pack"] * 2)
    V = _log_int(rng, 4_096, 248_320)
    if op in ("score", "train"):
        K = _width(rng, 8)
        N = _log_int(rng, 1, 4096)
        N = max(1, min(N, 4096 * 151_936 * 5120 // (V * K)))
        grad = "none" if op == "score" else rng.choice(["both", "both", "hidden"])
        return dict(LOSS, N=N, K=K, V=V, grad=grad, ignored=rng.choice([0.0, 0.1, 0.5]))
    group = rng.choice([32, 64, 64, 128])
    K = _width(rng, group)
    if op == "q4":
        return dict(Q4, B=_log_int(rng, 1, 64), K=K, V=V, group=group,
                    symmetric=rng.random() < 0.3, out=rng.choice(["bf16", "bf16", "f32"]))
    return dict(PACK, V=min(V, 151_936), K=K, group=group, symmetric=rng.random() < 0.3,
                dtype=rng.choice(["bf16", "bf16", "f32"]), out=rng.choice(["bf16", "f32"]))


# ---- inputs -----------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 6151 + 29)
    return g


def _dt(name):
    return torch.bfloat16 if name == "bf16" else torch.float32


def _weights(g, V, K, dtype):
    """Rows of unit norm on average, a tenth of them larger, and a few unused (zero) rows."""
    w = torch.randn(V, K, device=DEV, generator=g, dtype=torch.bfloat16)
    big = 1.0 + 2.0 * (torch.rand(V, 1, device=DEV, generator=g) < 0.1)
    w = w.mul_((big * K ** -0.5).to(torch.bfloat16))
    w[torch.randint(0, V, (max(1, V // 4096),), device=DEV, generator=g)] = 0
    return w.to(dtype)


def prepare(case, seed):
    g = _gen(seed)
    c = dict(case)
    if c["op"] == "loss":
        N, K, V = c["N"], c["K"], c["V"]
        w = _weights(g, V, K, torch.bfloat16)
        targets = torch.randint(0, V, (N,), device=DEV, generator=g)
        # states that point towards their targets by various amounts: losses of 0 to 20
        pull = 16.0 * torch.rand(N, 1, device=DEV, generator=g)
        h = 2.0 * torch.randn(N, K, device=DEV, generator=g) + pull * w[targets].float()
        padded = torch.rand(N, device=DEV, generator=g) < c["ignored"]
        targets = torch.where(padded, -100, targets).to(torch.int32)
        c.update(hidden=h.to(torch.bfloat16), lm_head=w, targets=targets)
        if c["grad"] != "none":  # the mean over the positions that count
            count = (~padded).sum().clamp_min(1)
            c["grad_loss"] = torch.where(padded, 0.0, 1.0 / count).float()
    elif c["op"] == "q4":
        B, K, V, G = c["B"], c["K"], c["V"], c["group"]
        # the codes are uniform in the range that their group's scale spans
        words = torch.randint(-2 ** 31, 2 ** 31, (V, K // 8), device=DEV, generator=g)
        scales = (0.2 + torch.rand(V, K // G, device=DEV, generator=g)) * (K ** -0.5 / 4)
        c.update(words=words.to(torch.int32), scales=scales.to(torch.bfloat16), biases=None)
        if not c["symmetric"]:
            lean = 7.5 + 1.5 * torch.randn(V, K // G, device=DEV, generator=g)
            c["biases"] = (-scales * lean).to(torch.bfloat16)
        c["hidden"] = (2.0 * torch.randn(B, K, device=DEV, generator=g)).to(torch.bfloat16)
    else:
        c["weight"] = _weights(g, c["V"], c["K"], _dt(c["dtype"]))
        if c["dtype"] == "f32":  # all of a float32's bits in use
            c["weight"] *= 1.0 + 0.01 * torch.rand(c["V"], c["K"], device=DEV, generator=g)
    return c


# ---- the plain forms ----------------------------------------------------------------------
def _plain_loss(s):
    counts = s["targets"] >= 0
    t = torch.where(counts, s["targets"], 0).long()
    h, w = s["hidden"].float(), s["lm_head"].float()
    x = h @ w.T
    top = x.amax(1, keepdim=True)
    lse = torch.log(torch.exp(x - top).sum(1)) + top[:, 0]
    loss = torch.where(counts, lse - x.gather(1, t[:, None])[:, 0], 0.0)
    if s["grad"] == "none":
        return {"loss": loss, "lse": lse}
    g = torch.where(counts, s["grad_loss"], 0.0)
    p = torch.exp(x.sub_(lse[:, None]))
    p[torch.arange(t.numel(), device=t.device), t] -= 1.0
    p *= g[:, None]
    out = {"loss": loss, "d_hidden": (p @ w).to(torch.bfloat16)}
    if s["grad"] == "both":
        out["d_lm_head"] = (p.T @ h).to(torch.bfloat16)
    return out


def _codes(words):
    """int32 words [V, K / 8] -> codes [V, K], the lowest four bits first."""
    shift = 4 * torch.arange(8, device=words.device, dtype=torch.int32)
    return ((words[..., None] >> shift) & 15).flatten(-2)


def _values(q, scales, biases, G):
    q = q.unflatten(-1, (-1, G))
    if biases is None:
        return ((q - 8) * scales[..., None]).flatten(-2)
    return (q * scales[..., None] + biases[..., None]).flatten(-2)


def _plain_q4(s):
    b = None if s["biases"] is None else s["biases"].float()
    w = _values(_codes(s["words"]).float(), s["scales"].float(), b, s["group"])
    return (s["hidden"].float() @ w.T).to(_dt(s["out"]))


def _plain_pack(s):
    w = s["weight"].float().unflatten(-1, (-1, s["group"]))
    if s["symmetric"]:
        scales, biases = (w.abs().amax(-1) / 7.0).to(torch.bfloat16), None
        d = scales.float()[..., None]
        q = torch.round(torch.where(d > 0, w / d, 0.0)) + 8.0
    else:
        lo = w.amin(-1)
        scales = ((w.amax(-1) - lo) / 15.0).to(torch.bfloat16)
        biases = lo.to(torch.bfloat16)
        d, b = scales.float()[..., None], biases.float()[..., None]
        q = torch.round(torch.where(d > 0, (w - b) / d, 0.0))
    q = q.clamp(0.0, 15.0).flatten(-2)
    b = None if biases is None else biases.float()
    out = {"scales": scales, "values": _values(q, scales.float(), b, s["group"]).to(_dt(s["out"]))}
    return out if biases is None else dict(out, biases=biases)


# ---- the framework's calls ------------------------------------------------------------------
_OPS = None


def _ops():
    global _OPS
    if _OPS is None:
        sys.path.insert(0, "strim-engine_amd")
        from strim_amd import ops
        _OPS = ops
    return _OPS


def _own_loss(s):
    ops = _ops()
    loss, lse, _ = ops.head_loss(s["hidden"], s["lm_head"], s["targets"])
    if s["grad"] == "none":
        return {"loss": loss, "lse": lse}
    dh, dw = ops.head_loss_grad(s["hidden"], s["lm_head"], s["targets"], lse, s["grad_loss"],
                                want_lm_head=s["grad"] == "both")
    out = {"loss": loss, "d_hidden": dh}
    return out if dw is None else dict(out, d_lm_head=dw)


def _own_q4(s):
    ops = _ops()
    q = ops.Q4Weight(s["words"], s["scales"], s["biases"], s["group"])
    return ops.head_logits_q4(s["hidden"], q, out_dtype=_dt(s["out"]))


def _own_pack(s):
    ops = _ops()
    q = ops.q4_pack(s["weight"], s["group"], symmetric=s["symmetric"])
    out = {"scales": q.scales, "values": ops.q4_unpack(q, _dt(s["out"]))}
    return out if q.biases is None else dict(out, biases=q.biases)


def run(state):
    if own:
        return {"loss": _own_loss, "q4": _own_q4, "pack": _own_pack}[state["op"]](state)
    return {"loss": _plain_loss, "q4": _plain_q4, "pack": _plain_pack}[state["op"]](state)


# ---- what a pass cannot do without ------------------------------------------------------------
def work(case):
    c = case
    if c["op"] == "loss":
        N, K, V = c["N"], c["K"], c["V"]
        io = 2 * V * K + 2 * N * K + 4 * N  # the projection, the states and the targets
        if c["grad"] == "none":
            return {"bytes": io + 8 * N, "flops": 2 * N * V * K}
        both = c["grad"] == "both"
        return {"bytes": io + 8 * N + 2 * N * K + (2 * V * K if both else 0),
                "flops": (6 if both else 4) * N * V * K}
    per_group = 2 if c["symmetric"] else 4
    V, K = c["V"], c["K"]
    held = V * K // 2 + V * (K // c["group"]) * per_group
    if c["op"] == "q4":
        size = 2 if c["out"] == "bf16" else 4
        return {"bytes": held + c["B"] * (2 * K + size * V), "flops": 2 * c["B"] * V * K}
    read = V * K * (2 if c["dtype"] == "bf16" else 4)
    back = V * K * (2 if c["out"] == "bf16" else 4)
    return {"bytes": read + 2 * held + back, "flops": 6 * V * K}


# ---- 64 bits ----------------------------------------------------------------------------------
def _exact_loss(s):
    h, w, t = s["hidden"].double(), s["lm_head"].double(), s["targets"].long()
    live = (t != -100).double()
    x = torch.mm(h, w.t())
    lse = torch.logsumexp(x, 1)
    at = t.clamp_min(0).unsqueeze(1)
    loss = (lse - torch.gather(x, 1, at).squeeze(1)) * live
    if s["grad"] == "none":
        return {"loss": loss, "lse": lse}
    x = torch.softmax(x, 1)
    x.scatter_add_(1, at, -torch.ones_like(at, dtype=torch.float64))
    x.mul_((s["grad_loss"].double() * live).unsqueeze(1))
    out = {"loss": loss, "d_hidden": torch.mm(x, w)}
    if s["grad"] == "both":
        out["d_lm_head"] = torch.mm(x.t(), h)
    return out


def _exact_dequantised(words, scales, biases, G):
    V, W = words.shape
    v = torch.empty(V, W, 8, dtype=torch.float64, device=words.device)
    for i in range(8):
        v[:, :, i] = torch.bitwise_and(torch.bitwise_right_shift(words, 4 * i), 15).double()
    v = v.view(V, W * 8 // G, G)
    zero = -8.0 * scales.double() if biases is None else biases.double()
    return v.mul_(scales.double().unsqueeze(2)).add_(zero.unsqueeze(2)).view(V, W * 8)


def _exact_pack(s):
    G, V, K = s["group"], s["V"], s["K"]
    w = s["weight"].double().view(V, K // G, G)
    hi, lo = w.max(2).values, w.min(2).values
    if s["symmetric"]:
        step = (torch.maximum(hi, -lo) / 7).to(torch.bfloat16).double().unsqueeze(2)
        base, first, last = torch.zeros_like(step), -8, 7
    else:
        step = ((hi - lo) / 15).to(torch.bfloat16).double().unsqueeze(2)
        base, first, last = lo.to(torch.bfloat16).double().unsqueeze(2), 0, 15
    q = torch.nan_to_num((w - base) / step, nan=0.0).round().clamp(first, last)
    out = {"scales": step.squeeze(2), "values": (q * step + base).view(V, K)}
    return out if s["symmetric"] else dict(out, biases=base.squeeze(2))


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "loss":
        return _exact_loss(s)
    if s["op"] == "q4":
        w = _exact_dequantised(s["words"], s["scales"], s["biases"], s["group"])
        return torch.mm(s["hidden"].double(), w.t())
    return _exact_pack(s)
