"""Finite logits far from zero: masks by a large negative number in some, most or all places, rows whose
largest logit is itself far, and small temperatures, for the scores and the distillation's loss.

The bounds are those of tests/test_scores_gpu.py and tests/test_distill_gpu.py, but that none grows with the
size of the logits where the result does not: with d = (max - x) / T, D = sum p d, c = (V / 256 + 40) 2^-24 and
e = c + 2^-22 (8 + D), a log-probability, (x - max) / T less the logarithm of the sum, is off by e and 2^-22 of d;
a loss by 2 e of its mass, 2^-22 of its terms' sizes (the probabilities' float32 exponentials) and one rounding."""
import pytest
import torch

from strim_amd import _native as N
from strim_amd import loss as L
from strim_amd import ops
from test_scores_gpu import Exact, gen, pitched, within, words_of

pytestmark = pytest.mark.gpu
NINF = float("-inf")
FILLS = [-1e9, -1e10, -1e12, -1e20, -1e30]
BF16, F32 = torch.bfloat16, torch.float32


def f32(T):
    """The temperature as the kernels get it."""
    return float(torch.tensor(T, dtype=F32))


def rows(V, dtype, seed=0):
    """A row for each fill and place; the largest logits far above zero or below it."""
    at = torch.arange(V, device="cuda")
    base = 3.0 * torch.randn(V, device="cuda", generator=gen(seed + V))
    few = torch.zeros(V, dtype=torch.bool, device="cuda")
    few[torch.tensor([1, V // 3, V // 2 + 5, V - 2], device="cuda")] = True
    last = few & (at == V - 2)
    places = [~few, ~last, at < min(4096, V // 2), at >= V - V // 3, at // 8 % 64 == 5, at // 512 % 4 != 2, at % 2 == 0]
    out = []
    for fill in FILLS:
        out += [torch.where(p, fill, base) for p in places]
        out.append(torch.full_like(base, fill))
        out.append(torch.where(at % 3 == 0, 2 * fill, torch.full_like(base, fill)))
        out.append(torch.where(at % 3 == 0, -fill, base))
        out.append(torch.where(last, -fill, torch.full_like(base, fill)))
        out.append(torch.where(few, base - fill, torch.where(at % 2 == 0, fill, base)))
    return torch.stack(out).to(dtype)


def as32(t):
    """Numbers past float32 as it has them."""
    return t.float().double()


def check(x, T, top, allowed=None, label=""):
    T = f32(T)
    R, V = x.shape
    xd = x.double() if allowed is None else torch.where(allowed, x.double(), NINF)
    most = xd.amax(1, keepdim=True)
    E = Exact(xd - most, T)  # (in 64 bits the log-sum-exp of logits of 1e20 keeps no digit of the sum)
    lse = E.lse + most[:, 0] / T
    mask = None if allowed is None else words_of(allowed)
    t = torch.stack([xd.argmax(1), torch.full((R,), V - 2, device="cuda"),
                     torch.zeros(R, dtype=torch.int64, device="cuda")], 1)
    out = ops.token_scores(x, t.int(), top, T, mask)
    assert bool((out.status == N.OK).all()), f"{label}: {out.status.unique()}"
    within(out.lse, as32(lse), E.e + 2.0 ** -22 * lse.abs(), f"{label} lse")
    within(out.entropy, E.H, E.tol_H, f"{label} entropy")
    within(out.logprobs, as32(E.lp.gather(1, t)), E.e[:, None] + 2.0 ** -22 * E.d.gather(1, t), f"{label} log-probabilities")
    vals, ids = torch.sort(xd, dim=1, descending=True, stable=True)
    vals, ids = vals[:, :top], ids[:, :top]
    assert torch.equal(out.top_ids, torch.where(vals == NINF, -1, ids).int()), label
    within(out.top_logprobs, as32(E.lp.gather(1, ids)), E.e[:, None] + 2.0 ** -22 * E.d.gather(1, ids), f"{label} alternatives")
    # without the alternatives and without tokens: the same statistics
    bare = ops.token_scores(x, None, 0, T, mask)
    assert torch.equal(bare.lse, out.lse) and torch.equal(bare.entropy, out.entropy) and bool((bare.status == 0).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T", [0.7, 0.8, 1.0, 2.0])
@pytest.mark.parametrize("V,top,copies", [(600, 20, 1), (4_000, 5, 1), (9_001, 20, 1), (9_001, 20, 36), (151_936, 64, 1)])
def test_scores(V, top, copies, T, dtype):
    print(f"[far] scores V={V} copies={copies} T={T} {dtype}", flush=True)
    check(rows(V, dtype).repeat(copies, 1), T, top, label=f"V={V} T={T}")


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_masked_scores(dtype):
    print(f"[far] masked {dtype}", flush=True)
    x = rows(20_011, dtype)
    allowed = torch.rand(x.shape, device="cuda", generator=gen(3)) < 0.5
    allowed[:, [0, 20_009]] = True
    allowed.scatter_(1, x.float().argmax(1, keepdim=True), True)
    check(x, 0.9, 20, allowed, "masked")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T", [1e-3, 1e-6, 1e-10, 1e-30, 1.2e-38])
def test_small_temperatures(T, dtype):
    """max / T past every guard; past float32, where the log-sum-exp is infinite and the others are not."""
    print(f"[far] T={T} {dtype}", flush=True)
    V, T = 9_001, f32(T)
    x = (4.0 * torch.randn(6, V, device="cuda", generator=gen(4))).to(dtype)
    x[0, :4_500] = x[0].amax()
    x[1, ::2] = -x[1].abs().amax()
    x[1, 1::2] = x[1, 0]  # all equal
    x[2] -= 40.0
    check(x, T, 20, label=f"T={T}")


# ---- distillation ---------------------------------------------------------------------------
def exact_loss(x, ids, lp, T, tail):
    """(loss, bound) in 64 bits, the tokens and the rest each against their own largest logit."""
    R, V = x.shape
    x, live = x.double(), ids >= 0
    at = torch.where(live, ids, 0).long()
    t = torch.where(live, lp.double(), NINF)
    p = torch.exp(t) if tail else torch.softmax(t, 1)
    r = (1 - p.sum(1)).clamp_min(0.0) if tail else torch.zeros(R, device="cuda").double()
    top = x.amax(1, keepdim=True)
    z = (x - top) / T
    ls = torch.exp(z).sum(1).log()
    lq = z.gather(1, at) - ls[:, None]
    inside = torch.zeros(R, V, dtype=torch.int32, device="cuda").scatter_add_(1, at, live.int()) > 0
    rest = torch.where(inside, NINF, x)
    most = rest.amax(1, keepdim=True)
    lsr = torch.exp((rest - most) / T).sum(1).log()
    log_rest = (most - top)[:, 0] / T + lsr - ls
    logp = torch.log(p.clamp_min(1e-300))
    loss = torch.where(p > 0, p * (logp - lq), 0.0).sum(1)
    size = torch.where(p > 0, p * (logp.abs() + lq.abs()), 0.0).sum(1)
    q = torch.exp(z - ls[:, None])
    D = (q * -z).sum(1)
    if tail:
        logr = torch.log(r.clamp_min(1e-300))
        loss = loss + torch.where(r > 0, r * (logr - log_rest), 0.0)
        # (r is off by as much as the probabilities' sum is)
        size = size + torch.where(r > 0, (p.sum(1) + r) * (logr.abs() + log_rest.abs()), 0.0)
    e = (V / 256 + 40) * 2.0 ** -24 + 2.0 ** -22 * (8 + D)
    return loss, (p.sum(1) + r) * 2 * e + 2.0 ** -22 * size + 2.0 ** -24 * loss.abs()


def teacher(R, V, M, seed):
    """Ids anywhere in the row, the two ends among them, with nine tenths of the mass."""
    ids = torch.rand(R, V, device="cuda", generator=gen(seed)).topk(M, 1).indices.int()
    ids[:, 0], ids[:, 1] = 1, V - 2
    for m in range(2, M):  # (no id twice)
        ids[:, m] = torch.where((ids[:, m] == 1) | (ids[:, m] == V - 2), -1, ids[:, m])
    lp = torch.log_softmax(torch.where(ids < 0, NINF, torch.randn(R, M, device="cuda", generator=gen(seed + 1))), 1)
    return ids, lp + torch.log(torch.tensor(0.9))


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T", [0.8, 1.0, 2.0])
@pytest.mark.parametrize("V,copies", [(600, 1), (9_001, 1), (30_001, 3), (60_001, 1), (60_001, 5)])
def test_distillation_losses(V, copies, T, dtype, tail):
    print(f"[far] distill V={V} copies={copies} T={T} {dtype} tail={tail}", flush=True)
    T = f32(T)
    x = rows(V, dtype).repeat(copies, 1)
    x = pitched(x, 3)
    R = x.shape[0]
    ids, lp = teacher(R, V, 9, V)
    ref, tol = exact_loss(x, ids, lp, T, tail)
    for loss, st in (ops.distill(x, ids, lp, T, tail)[::3],
                     ops.distill_step(x, ids, lp, torch.ones(R, device="cuda"), T, tail)[::2]):
        assert bool((st == N.OK).all()), st.unique()
        within(loss, ref, tol, "loss")


def test_a_filled_tail_through_the_differentiable_forms():
    """A vocabulary padded with -1e10: scores and gradients of the real tokens as without the padding."""
    R, V, pad = 5, 8_000, 1_500
    g = gen(9)
    x = 3.0 * torch.randn(R, V, device="cuda", generator=g)
    wide = torch.cat([x, torch.full((R, pad), -1e10, device="cuda")], 1)
    t = torch.randint(0, V, (R,), device="cuda", generator=g)
    ids, lp = ops.token_scores(x + torch.randn(R, V, device="cuda", generator=g), top=12)[3:5]
    out = []
    for y in (x, wide):
        leaf = y.clone().requires_grad_()
        s = L.token_scores(leaf, t, temperature=0.8)
        value = s.logprobs.sum() + 0.1 * s.entropy.sum() + L.distill_loss(leaf, ids, lp, 0.8, reduction="sum")
        out.append((value.detach(), torch.autograd.grad(value, leaf)[0]))
    # (the same sums in other orders: 2^-20 of probabilities of at most 1, entropies of at most 9)
    assert abs(float(out[0][0] - out[1][0])) <= 1e-5 * abs(float(out[0][0]))
    assert bool((out[1][1][:, V:] == 0).all())
    assert float((out[0][1] - out[1][1][:, :V]).abs().max()) <= 4e-5


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T", [2.0 ** -126, 1e20, 1e38, 3.4e38])
def test_the_ends_of_the_temperature(T, dtype):
    print(f"[far] T={T} {dtype}", flush=True)
    x = (4.0 * torch.randn(5, 9_001, device="cuda", generator=gen(6))).to(dtype)
    x[1, ::2] = -1e30
    check(x, T, 20, label=f"T={T}")
    for bad in (2.0 ** -127, 1e-45, 0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="temperature"):
            ops.token_scores(x, temperature=bad)
        with pytest.raises(ValueError, match="temperature"):
            ops.distill(x, torch.zeros(5, 1, dtype=torch.int32, device="cuda"), torch.zeros(5, 1, device="cuda"), bad)
