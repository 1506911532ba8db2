"""The gradient of a distillation step where the logits are far from zero, or the temperature is small.

A step takes a token's probability from its distance to a row's largest logit, so its bound does not grow with
the logits: with D = sum q (max - x) / T and e = (V / 256 + 40) 2^-24 + 2^-22 (8 + D) (tests/test_scores_gpu.py), a
probability is off by 2 e and, of its exponent's terms, 2^-21 (8 + (max - x) / T); bf16 rows by 2^-14 more (their
exponents' common term is rounded to that); the teacher's float32 exponentials by 2^-22; then one rounding to the
type."""
import pytest
import torch

from strim_amd import _native as N
from strim_amd import ops
from test_far_logits_gpu import f32, teacher
from test_scores_gpu import gen, within

pytestmark = pytest.mark.gpu
NINF = float("-inf")
BF16, F32 = torch.bfloat16, torch.float32


def exact(x, ids, lp, w, T, tail, rest_bound, held=0.0):
    """(gradient, bound) in 64 bits. rest_bound: the rest's tokens by their distance to the rest's largest logit,
    else to the row's. held: what each probability is off by besides."""
    R, V = x.shape
    half, bf16 = torch.finfo(x.dtype).eps / 2, x.dtype == BF16
    x, live = x.double(), ids >= 0
    at = torch.where(live, ids, 0).long()
    t = torch.where(live, lp.double(), NINF)
    p = torch.exp(t) if tail else torch.softmax(t, 1)
    mass = p.sum(1, keepdim=True)
    r = (1 - mass).clamp_min(0.0) if tail else torch.zeros_like(mass)
    z = (x - x.amax(1, keepdim=True)) / T
    q = torch.softmax(z, 1)
    inside = torch.zeros(R, V, dtype=torch.int32, device="cuda").scatter_add_(1, at, live.int()) > 0
    rest = torch.where(inside, NINF, x)
    zr = (rest - rest.amax(1, keepdim=True)) / T
    bucket = r * torch.softmax(zr, 1) if tail else torch.zeros_like(x)
    target = torch.zeros_like(x).scatter_add_(1, at, p * live)
    soft = q * (mass + r)
    e = (V / 256 + 40) * 2.0 ** -24 + 2.0 ** -22 * (8 + (q * -z).sum(1, keepdim=True))
    rel = 2 * e + 2.0 ** -21 * 8 + (2.0 ** -14 if bf16 else 0.0) + held
    far = (-zr).nan_to_num(posinf=0.0) if tail and rest_bound else -z
    w = w.double()[:, None] / T
    tol = soft * (rel - 2.0 ** -21 * z) + bucket * (rel + 2.0 ** -21 * far + 2.0 ** -22 * mass / r.clamp_min(1e-9))
    tol = w.abs() * (tol + target * 2.0 ** -22)
    d = w * (soft - bucket - target)
    return d, tol + (d.abs() + tol) * half + 1e-37


OFFSETS = [0.0, 300.0, -300.0, 3e4, -3e4, 1.2e6, -1e6, 1e8, -3e8, 1e12, -1e20]


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T", [1.0, 0.3, 1e-2, 1e-4, 1e-6])
@pytest.mark.parametrize("V,copies", [(2_500, 1), (20_000, 1), (60_001, 1), (60_001, 13), (60_001, 25)])
def test_step(V, copies, T, dtype, tail):
    """Many tokens share a row's largest logit, at any distance from zero."""
    print(f"[far] gradient V={V} copies={copies} T={T} {dtype} tail={tail}", flush=True)
    T = f32(T)
    g = gen(V + copies)
    x = torch.randn(len(OFFSETS) * copies, V, device="cuda", generator=g)
    x = (x * 2).round() * max(T, 0.01) + torch.tensor(OFFSETS * copies, device="cuda")[:, None]
    x = torch.minimum(x, x.quantile(0.9, 1, keepdim=True) if V < 20_000 else x[:, :2_000].quantile(0.9, 1, keepdim=True))
    x = x.to(dtype)
    R = x.shape[0]
    ids, lp = teacher(R, V, 11, V)
    w = torch.randn(R, device="cuda", generator=g)
    ref, tol = exact(x, ids, lp, w, T, tail, False)
    loss, d, st = ops.distill_step(x, ids, lp, w, T, tail)
    assert bool((st == N.OK).all())
    within(d, ref, tol, "gradient")
    # into the logits themselves: the same bits
    y = x.clone()
    assert torch.equal(ops.distill_step(y, ids, lp, w, T, tail, out=y)[1], d)


BELOW = [0.0, 30.0, 300.0, 700.0, 1e4, 1e6, 1e8, 1e10, 1e20, 1e30]


def apart(V, copies, dtype, seed, lift=1.0):
    """Rows whose alternatives are far above the rest (lift 1) or far below it (-1)."""
    g = gen(seed)
    R = len(BELOW) * copies
    ids, lp = teacher(R, V, 11, V)
    x = 2.0 * torch.randn(R, V, device="cuda", generator=g) - lift * torch.tensor(BELOW * copies, device="cuda")[:, None]
    at = torch.where(ids < 0, ids[:, :1], ids).long()
    x.scatter_(1, at, 3.0 * torch.randn(R, 1, device="cuda", generator=g).expand(R, 11))
    return x.to(dtype), ids, lp, torch.randn(R, device="cuda", generator=g)


SHAPES = [(2_500, 1), (20_000, 1), (60_001, 1), (60_001, 13), (60_001, 27)]


@pytest.mark.parametrize("lift", [1.0, -1.0])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T", [1.0, 0.3, 2.0])
@pytest.mark.parametrize("V,copies", SHAPES)
def test_step_with_the_rest_apart(V, copies, T, dtype, lift):
    """The teacher's remaining mass goes to a rest that the student all but excludes (a masked vocabulary), and
    the reverse: the rest's gradients sum to that mass, whatever its distance."""
    print(f"[far] apart V={V} copies={copies} T={T} {dtype} lift={lift}", flush=True)
    T = f32(T)
    x, ids, lp, w = apart(V, copies, dtype, V + copies, lift)
    ref, tol = exact(x, ids, lp, w, T, True, True)
    loss, d, st = ops.distill_step(x, ids, lp, w, T, True)
    assert bool((st == N.OK).all())
    within(d, ref, tol, "gradient")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V,copies", SHAPES)
def test_gradient_alone_with_the_rest_apart(V, copies, dtype):
    """From lse and log_rest as float32 holds them: 2^-23 of either, no more, in each probability."""
    print(f"[far] apart, the gradient alone V={V} copies={copies} {dtype}", flush=True)
    x, ids, lp, w = apart(V, copies, dtype, V + copies)
    near = (torch.tensor(BELOW * copies) <= 1e4).nonzero()[:, 0].cuda()
    x, ids, lp, w = x[near].contiguous(), ids[near].contiguous(), lp[near].contiguous(), w[near].contiguous()
    _, lse, rest, _ = ops.distill(x, ids, lp, 1.0, True)
    held = 2.0 ** -23 * (lse.abs() + rest.abs()).double()[:, None]
    d = ops.distill_grad(x, ids, lp, lse, rest, w, 1.0, True)
    within(d, *exact(x, ids, lp, w, 1.0, True, True, held), "gradient")
