"""Operators of training and scoring: what is measured, in plain torch and in this framework.

Three operators that a draft head's training and a server's answers need:

  score    rows of logits [R, V]: the log-probabilities of given tokens, the entropy, the
           log-sum-exp and the top alternatives, under an allow-mask and a temperature; with
           `grad`, the logits' gradient for given gradients of log-probability and entropy
  distill  a student's logits [N, V] against a teacher's top alternatives (ids and
           log-probabilities [N, M]): the loss alone ("loss"), or with its gradient for given
           weights of the rows ("step"); `tail` keeps the teacher's remaining mass as one
           bucket, else the alternatives are renormalised
  norm     rows [N, K] normalised by their root mean square, or by mean and variance ("layer");
           with `grad`, the gradients of the rows and of the weights

Sizes are those of the repository's configurations (the 151,936-token vocabulary, the
32,768-token draft vocabulary, 5,120 channels, 1 to 64 decode rows) and others of the same
ranges. `own` False: elementary torch operations in 32 bits, rounded once at the end; True:
the framework's calls.
"""
import math
import sys

import torch

own = False

DEV = "cuda:0"

SCORE = dict(op="score", R=1, V=151_936, dtype="bf16", tokens=1, top=0, T=1.0, mask=False, grad=False)
DISTILL = dict(op="distill", N=96, V=32_768, M=16, dtype="bf16", T=1.0, tail=False, ragged=0.0,
               what="step")
NORM = dict(op="norm", N=1, K=5120, dtype="bf16", kind="rms", grad=False)


def listed():
    return [
        # one stream's next token with its 20 alternatives: the smallest answer a server gives
        dict(SCORE, name="score_b1", top=20),
        # a decode batch under grammar masks and a sampling temperature, five alternatives a row
        dict(SCORE, name="score_b64_masked", R=64, top=5, T=0.8, mask=True),
        # a teacher's alternatives for a batch of positions: what distillation learns from
        dict(SCORE, name="score_teacher", R=2048, top=64),
        # log-probabilities and entropies of a policy's tokens with their gradient, float32 logits,
        # odd sizes
        dict(SCORE, name="score_train_odd", R=1003, V=100_003, dtype="f32", grad=True),
        # one small accumulation step of a draft head over its truncated vocabulary
        dict(DISTILL, name="distill_n96_draft"),
        # a ragged batch: a tenth of the rows without a teacher, rows of fewer alternatives
        dict(DISTILL, name="distill_n2000_draft", N=2000, M=32, T=2.0, ragged=0.1),
        # the loss alone, over held-out positions: float32 logits, odd sizes
        dict(DISTILL, name="distill_eval_odd", N=500, V=50_021, M=33, dtype="f32", T=2.0, tail=True,
             what="loss"),
        # a training step over the full vocabulary: the largest
        dict(DISTILL, name="distill_n4096", N=4096, V=151_936, M=64, tail=True),
        # the final norm of one decode step
        dict(NORM, name="norm_n1"),
        # a training step's positions at full width
        dict(NORM, name="norm_train_n4096", N=4096, grad=True),
        # mean and variance, weights and biases, float32, odd sizes
        dict(NORM, name="layer_train_odd", N=1003, K=2051, dtype="f32", kind="layer", grad=True),
        # narrow rows, as the heads of 4,096 positions have them
        dict(NORM, name="norm_train_heads", N=131_072, K=128, grad=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["score"] * 4 + ["distill"] * 4 + ["norm"] * 3)
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    if op == "norm":
        K = rng.choice([64, 128, 1024, 2048, 4096, 5120, 8192]) if rng.random() < 0.5 else _log_int(rng, 33, 9001)
        N = min(_log_int(rng, 1, 200_000), 96_000_000 // K)
        return dict(NORM, N=N, K=K, dtype=dtype, kind=rng.choice(["rms", "rms", "layer"]),
                    grad=rng.random() < 0.7)
    V = rng.choice([32_768, 151_936]) if rng.random() < 0.3 else _log_int(rng, 4_096, 248_320)
    T = rng.choice([1.0, 1.0, 0.7, 2.0])
    if op == "score":
        R = min(_log_int(rng, 1, 4096), 2048 * 151_936 // V)
        if rng.random() < 0.3:
            return dict(SCORE, R=R, V=V, dtype=dtype, T=T, mask=rng.random() < 0.3, grad=True)
        return dict(SCORE, R=R, V=V, dtype=dtype, T=T, mask=rng.random() < 0.4,
                    tokens=rng.choice([1, 1, 4]), top=rng.choice([0, 1, 5, 20, 20, 64, 100]))
    N = min(_log_int(rng, 1, 4096), 4096 * 151_936 // (V if dtype == "bf16" else 2 * V))
    return dict(DISTILL, N=N, V=V, M=_log_int(rng, 1, 128), dtype=dtype, T=T, tail=rng.random() < 0.5,
                ragged=rng.choice([0.0, 0.1]), what=rng.choice(["step", "step", "loss"]))


# ---- inputs -----------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 7561 + 11)
    return g


def _dt(name):
    return torch.bfloat16 if name == "bf16" else torch.float32


def _logits(g, R, V):
    """A body of spread 2 and eight tokens of every row far above it by various amounts."""
    x = torch.randn(R, V, device=DEV, generator=g)
    x *= 2.0
    at = torch.randint(0, V, (R, 8), device=DEV, generator=g)
    return x.scatter_(1, at, 5.0 + 9.0 * torch.rand(R, 8, device=DEV, generator=g))


def _mask_words(g, R, V):
    """Grammar masks: rows that forbid little, rows that allow about a thirtieth, and rows that
    allow one run of some hundred ids. int32 words, bit i of word w for id 32 w + i."""
    W = (V + 31) // 32
    kind = torch.randint(0, 3, (R, 1), device=DEV, generator=g)
    u = torch.rand(R, 32 * W, device=DEV, generator=g)
    v = torch.arange(32 * W, device=DEV)
    first = torch.randint(0, V - 400, (R, 1), device=DEV, generator=g)
    run = (v >= first) & (v < first + 400)
    ok = torch.where(kind == 0, u < 0.97, torch.where(kind == 1, u < 0.03, run))
    ok[:, 5:300:3] |= kind < 2  # (some ids that every grammar of these two kinds allows)
    bits = ok.view(R, W, 32).to(torch.int64) << torch.arange(32, device=DEV)
    words = bits.sum(2)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)


def prepare(case, seed):
    g = _gen(seed)
    c = dict(case)
    if c["op"] == "score":
        R, V = c["R"], c["V"]
        x = _logits(g, R, V)
        c["mask_words"] = _mask_words(g, R, V) if c["mask"] else None
        if c["mask"]:  # tokens that the masks allow, as a sampler gave them
            t = torch.where(_allowed(c["mask_words"], V), x, -math.inf).topk(c["tokens"], 1).indices
        else:
            t = torch.randint(0, V, (R, c["tokens"]), device=DEV, generator=g)
        c.update(logits=x.to(_dt(c["dtype"])), ids=t.to(torch.int32))
        if c["grad"]:
            c["g_logprob"] = torch.randn(R, 1, device=DEV, generator=g) / R
            c["g_entropy"] = torch.full((R,), -0.01 / R, device=DEV)
    elif c["op"] == "distill":
        N, V, M = c["N"], c["V"], c["M"]
        x = _logits(g, N, V).to(_dt(c["dtype"]))
        ids = torch.empty(N, M, dtype=torch.int32, device=DEV)
        lp = torch.empty(N, M, device=DEV)
        for a in range(0, N, 512):  # the teacher: the student's logits, moved
            t = x[a:a + 512].float() + torch.randn(x[a:a + 512].shape, device=DEV, generator=g)
            t /= c["T"]
            top = t.topk(M, 1)
            ids[a:a + 512] = top.indices.to(torch.int32)
            lp[a:a + 512] = top.values - torch.logsumexp(t, 1, keepdim=True)
        weights = torch.ones(N, device=DEV)
        if c["ragged"]:
            held = torch.randint(1, M + 1, (N, 1), device=DEV, generator=g)
            held[torch.rand(N, 1, device=DEV, generator=g) < c["ragged"]] = 0
            ids[torch.arange(M, device=DEV) >= held] = -1
            weights = (held[:, 0] > 0).float()
        c.update(logits=x, ids=ids, logprobs=lp, weights=weights / weights.sum().clamp_min(1))
    else:
        N, K, dt = c["N"], c["K"], _dt(c["dtype"])
        # rows of various scales, a few channels larger than the rest
        x = torch.randn(N, K, device=DEV, generator=g) * (0.3 + torch.rand(N, 1, device=DEV, generator=g))
        x[:, ::61] *= 8.0
        c["x"] = (x + 0.2).to(dt)
        c["weight"] = (1.0 + 0.2 * torch.randn(K, device=DEV, generator=g)).to(dt)
        c["bias"] = (0.1 * torch.randn(K, device=DEV, generator=g)).to(dt) if c["kind"] == "layer" else None
        c["eps"] = 1e-5 if c["kind"] == "layer" else 1e-6
        if c["grad"]:
            c["g_y"] = torch.randn(N, K, device=DEV, generator=g).to(dt)
    return c


# ---- the plain forms ----------------------------------------------------------------------
def _allowed(words, V):
    """int32 words [R, W] -> truth values [R, V]."""
    bits = (words[:, :, None] >> torch.arange(32, device=words.device, dtype=torch.int32)) & 1
    return bits.flatten(1)[:, :V] != 0


def _plain_score(s):
    V, T, t = s["V"], s["T"], s["ids"].long()
    x = s["logits"].float()
    if s["mask_words"] is not None:
        x = torch.where(_allowed(s["mask_words"], V), x, -math.inf)
    z = x / T
    top = z.amax(1, keepdim=True)
    z -= top  # (not the log-probabilities yet: the sums keep their digits next to the largest)
    e = torch.exp(z)
    total = e.sum(1, keepdim=True)
    rest = torch.log(total)
    entropy = rest[:, 0] - (torch.where(e > 0, z * e, 0.0)).sum(1) / total[:, 0]
    lse = (rest + top)[:, 0]
    out = {"logprobs": z.gather(1, t) - rest, "entropy": entropy, "lse": lse}
    if s["top"]:
        # one whole number per token that orders by logit, then by id: all different
        b = (x + 0.0).view(torch.int32).long()
        b = torch.where(b < 0, -(b & 0x7FFFFFFF), b)
        key = (b << 20) + (2 ** 20 - 1 - torch.arange(V, device=x.device))
        key = key.topk(s["top"], 1).values
        ids = 2 ** 20 - 1 - (key & (2 ** 20 - 1))
        out.update(top_ids=ids.to(torch.int32), top_logprobs=z.gather(1, ids) - rest)
    if s["grad"]:
        g, h = s["g_logprob"], s["g_entropy"][:, None]
        p = e / total
        d = torch.where(p > 0, -p * (g + h * (z - rest + entropy[:, None])), 0.0)
        d.scatter_add_(1, t, g)
        out["d_logits"] = (d / T).to(s["logits"].dtype)
    return out


def _plain_distill(s):
    N, V, T = s["N"], s["V"], s["T"]
    live = (s["ids"] >= 0) & (s["logprobs"] > -math.inf)
    at = torch.where(live, s["ids"], V).long()  # (column V takes what belongs nowhere)
    t = torch.where(live, s["logprobs"], -math.inf).double()
    if s["tail"]:
        p = torch.exp(t)
        r = (1.0 - p.sum(1)).clamp_min(0.0)
    else:
        p = torch.exp(t - t.amax(1, keepdim=True).nan_to_num(neginf=0.0))
        p = p / p.sum(1, keepdim=True).clamp_min(1e-300)
        r = torch.zeros(N, dtype=torch.float64, device=t.device)
    has = live.any(1)
    r = torch.where(has, r, 0.0)
    logp, logr = torch.log(torch.where(p > 0, p, 1.0)), torch.log(torch.where(r > 0, r, 1.0))
    mass = p.sum(1) + r
    z = torch.zeros(N, V + 1, device=t.device)
    torch.div(s["logits"].float(), T, out=z[:, :V])
    z[:, V] = -math.inf
    z -= z.amax(1, keepdim=True)
    e = torch.exp(z)
    # (the rows' own numbers in 64 bits: a small loss is the difference of much larger ones)
    total = e.sum(1, keepdim=True, dtype=torch.float64)
    logq = torch.where(live, z.gather(1, at) - torch.log(total), 0.0)
    loss = (p * (logp - logq)).sum(1)
    if s["tail"]:
        outside = e.scatter_(1, at, 0.0).sum(1, dtype=torch.float64) / total[:, 0]
        loss = loss + r * (logr - torch.log(outside))
    loss = torch.where(has, loss, 0.0).float()
    if s["what"] == "loss":
        return {"loss": loss}
    w = torch.where(has, s["weights"], 0.0) / T
    d = torch.exp(z - torch.log(total).float())
    p, factor = (w[:, None] * p).float(), w * mass
    at_ids = factor.float()[:, None] * d.gather(1, at)
    for m in range(s["M"]):  # (an id may stand twice)
        same = (at == at[:, m:m + 1]) & live
        at_ids[:, m] -= torch.where(same, p, 0.0).sum(1)
    if s["tail"]:
        factor = factor - w * r / outside
    d *= factor.float()[:, None]
    d.scatter_(1, at, at_ids)
    return {"loss": loss, "d_logits": d[:, :V].to(s["logits"].dtype)}


def _plain_norm(s):
    x, w, dt = s["x"].float(), s["weight"].float(), s["x"].dtype
    if s["kind"] == "layer":
        x = x - x.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt((x * x).mean(1, keepdim=True) + s["eps"])
    xh = x * rstd
    y = xh * w
    if s["kind"] == "layer":
        y = y + s["bias"].float()
    if not s["grad"]:
        return {"y": y.to(dt)}
    g = s["g_y"].float()
    out = {"y": y.to(dt), "d_weight": (g * xh).sum(0).to(dt)}
    if s["kind"] == "layer":
        out["d_bias"] = g.sum(0).to(dt)
    g = g * w
    dx = g - xh * (g * xh).mean(1, keepdim=True)
    if s["kind"] == "layer":
        dx = dx - g.mean(1, keepdim=True)
    out["d_x"] = (rstd * dx).to(dt)
    return out


# ---- the framework's calls ------------------------------------------------------------------
_OPS = None


def _ops():
    global _OPS
    if _OPS is None:
        sys.path.insert(0, "strim-engine_amd")
        from strim_amd import ops
        _OPS = ops
    return _OPS


def _own_score(s):
    ops = _ops()
    out = ops.token_scores(s["logits"], s["ids"], top=s["top"], temperature=s["T"], mask=s["mask_words"])
    res = {"logprobs": out.logprobs, "entropy": out.entropy, "lse": out.lse}
    if s["top"]:
        res.update(top_ids=out.top_ids, top_logprobs=out.top_logprobs)
    if s["grad"]:
        res["d_logits"] = ops.token_scores_grad(s["logits"], s["ids"], out.lse, out.entropy, s["g_logprob"],
                                                s["g_entropy"], temperature=s["T"], mask=s["mask_words"])
    return res


def _own_distill(s):
    ops = _ops()
    if s["what"] == "loss":
        return {"loss": ops.distill(s["logits"], s["ids"], s["logprobs"], temperature=s["T"],
                                    tail=s["tail"])[0]}
    loss, d_logits, _ = ops.distill_step(s["logits"], s["ids"], s["logprobs"], s["weights"],
                                         temperature=s["T"], tail=s["tail"])
    return {"loss": loss, "d_logits": d_logits}


def _own_norm(s):
    ops = _ops()
    layer = s["kind"] == "layer"
    y, rstd, mean = ops.norm(s["x"], s["weight"], s["bias"], eps=s["eps"], center=layer)
    if not s["grad"]:
        return {"y": y}
    dx, dw, db = ops.norm_grad(s["x"], s["weight"], s["bias"], s["g_y"], rstd, mean)
    out = {"y": y, "d_weight": dw, "d_x": dx}
    return dict(out, d_bias=db) if layer else out


def run(state):
    if own:
        return {"score": _own_score, "distill": _own_distill, "norm": _own_norm}[state["op"]](state)
    return {"score": _plain_score, "distill": _plain_distill, "norm": _plain_norm}[state["op"]](state)


# ---- what a pass cannot do without ------------------------------------------------------------
def work(case):
    c = case
    size = 2 if c["dtype"] == "bf16" else 4
    if c["op"] == "score":
        R, V = c["R"], c["V"]
        moved = R * V * size * (2 if c["grad"] else 1) + (R * V // 8 if c["mask"] else 0)
        small = R * (8 * c["tokens"] + 8 * c["top"] + 8 + (8 if c["grad"] else 0))
        return {"bytes": moved + small, "flops": R * V * (16 if c["grad"] else 8)}
    if c["op"] == "distill":
        N, V = c["N"], c["V"]
        step = c["what"] == "step"
        return {"bytes": N * V * size * (2 if step else 1) + N * (8 * c["M"] + 8),
                "flops": N * V * (9 if step else 5)}
    N, K = c["N"], c["K"]
    return {"bytes": N * K * size * (4 if c["grad"] else 2) + 4 * K * size,
            "flops": N * K * (16 if c["grad"] else 5)}


# ---- 64 bits ----------------------------------------------------------------------------------
def _exact_score(s):
    T, parts = s["T"], []
    for a in range(0, s["R"], 128):
        b = slice(a, a + 128)
        x = s["logits"][b].double()
        if s["mask_words"] is not None:
            x = x.masked_fill(~_allowed(s["mask_words"][b], s["V"]), -math.inf)
        lp = torch.log_softmax(x / T, 1)
        p = lp.exp()
        h = -(p * lp.nan_to_num(neginf=0.0)).sum(1)
        t = s["ids"][b].long()
        one = {"logprobs": torch.take_along_dim(lp, t, 1), "entropy": h, "lse": torch.logsumexp(x / T, 1)}
        if s["top"]:
            order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :s["top"]]
            one.update(top_ids=order.to(torch.int32), top_logprobs=torch.take_along_dim(lp, order, 1))
        if s["grad"]:
            g, gh = s["g_logprob"][b].double(), s["g_entropy"][b].double().unsqueeze(1)
            d = torch.zeros_like(p).scatter_add_(1, t, g)
            d.addcmul_(p, g.sum(1, keepdim=True), value=-1.0)
            d.addcmul_(p * (lp.nan_to_num(neginf=0.0) + h.unsqueeze(1)), gh, value=-1.0)
            one["d_logits"] = d / T
        parts.append(one)
    return {k: torch.cat([o[k] for o in parts]) for k in parts[0]}


def _exact_distill(s):
    N, V, T, M = s["N"], s["V"], s["T"], s["M"]
    losses, grads = [], []
    for a in range(0, N, 128):
        b = slice(a, a + 128)
        ids, t = s["ids"][b].long(), s["logprobs"][b].double()
        t = t.masked_fill(ids < 0, -math.inf)
        live = t > -math.inf
        has = live.any(1)
        n = ids.shape[0]
        if s["tail"]:
            p = t.exp()
            r = (-torch.special.expm1(torch.logsumexp(t, 1))).clamp_min(0.0)
        else:
            p = torch.softmax(t, 1).nan_to_num(nan=0.0)
            r = torch.zeros(n, dtype=torch.float64, device=t.device)
        lq = torch.log_softmax(s["logits"][b].double() / T, 1)
        safe = ids.clamp_min(0)
        inside = torch.zeros(n, V, dtype=torch.int32, device=t.device)
        inside.scatter_add_(1, safe, live.to(torch.int32))
        inside = inside > 0
        lrest = torch.logsumexp(lq.masked_fill(inside, -math.inf), 1)
        loss = torch.xlogy(p, p).sum(1) - (p * torch.take_along_dim(lq, safe, 1)).sum(1)
        loss = loss + torch.xlogy(r, r) - torch.where(r > 0, r * lrest, 0.0)
        losses.append(torch.where(has, loss, 0.0))
        if s["what"] == "step":
            q = lq.exp()
            target = torch.zeros(n, V, dtype=torch.float64, device=t.device).scatter_add_(1, safe, p * live)
            target += torch.where(inside, 0.0, (lq - lrest.unsqueeze(1)).exp() * r.unsqueeze(1))
            mass = (p * live).sum(1) + r
            w = torch.where(has, s["weights"][b].double(), 0.0) / T
            grads.append((q * mass.unsqueeze(1) - target) * w.unsqueeze(1))
            if N * V > 200_000_000:  # (the whole in 64 bits only where it fits well)
                grads[-1] = grads[-1].float()
    out = {"loss": torch.cat(losses)}
    return out if s["what"] == "loss" else dict(out, d_logits=torch.cat(grads))


def _exact_norm(s):
    x, w = s["x"].double(), s["weight"].double()
    n = x.shape[1]
    mu = x.sum(1, keepdim=True) / n if s["kind"] == "layer" else 0.0
    c = x - mu
    rstd = torch.rsqrt(torch.einsum("ij,ij->i", c, c).unsqueeze(1) / n + s["eps"])
    y = c * (rstd * w)
    if s["bias"] is not None:
        y += s["bias"].double()
    if not s["grad"]:
        return {"y": y}
    gy = s["g_y"].double()
    out = {"y": y, "d_weight": (gy * c * rstd).sum(0)}
    if s["bias"] is not None:
        out["d_bias"] = gy.sum(0)
    gw = gy * w
    along = (gw * c).sum(1, keepdim=True) * rstd ** 3 / n
    dx = gw * rstd - c * along
    if s["kind"] == "layer":
        dx -= (gw.sum(1, keepdim=True) / n) * rstd
    out["d_x"] = dx
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"score": _exact_score, "distill": _exact_distill, "norm": _exact_norm}[s["op"]](s)
