"""Distillation from a teacher's top logits (strim_distill, strim_distill_grad, strim_distill_step and
their differentiable form) against the formulas in float64, and against differences.

The bounds: a log-sum-exp of float32 terms is off by e = c + 2^-22 (8 + D), with c = (V / 256 + 40) 2^-24
and D = sum q |x - max| / T (tests/test_scores_gpu.py derives it); the alternatives' own numbers are in 64
bits. So a loss is off by (sum p + r) 2 e and its rounding, 2^-24 of it, and 2^-23 of sum p |x| / T; a
gradient by |terms| (2 e + 2^-21 (1 + |lse| + |x| / T)) and one rounding to its type, where the bucket's
term also carries log_rest's rounding, 2^-24 of it."""
import pytest
import torch

from strim_amd import _native as N
from strim_amd import loss as L
from strim_amd import ops
from test_scores_gpu import gen, logits, pitched, within

pytestmark = pytest.mark.gpu
NINF = float("-inf")


def teacher(x, M, T, seed, move=1.0, ragged=True):
    """Alternatives of logits near the student's; some rows with fewer, some with none."""
    R, V = x.shape
    t = x.double() + move * torch.randn(R, V, device="cuda", generator=gen(seed), dtype=torch.float64)
    t = t / T
    n = min(M, V)
    top = t.topk(n, 1)
    ids = torch.full((R, M), -1, dtype=torch.int32, device="cuda")
    lp = torch.full((R, M), NINF, device="cuda")
    ids[:, :n] = top.indices.to(torch.int32)
    lp[:, :n] = (top.values - torch.logsumexp(t, 1, keepdim=True)).float()
    if ragged and R > 2:
        held = torch.randint(1, M + 1, (R, 1), device="cuda", generator=gen(seed + 1))
        held[1::7] = 0
        ids[torch.arange(M, device="cuda") >= held] = -1
    return ids, lp


class Exact:
    def __init__(self, x, ids, lp, T=1.0, tail=False):
        R, V = x.shape
        self.T, eps = T, torch.finfo(x.dtype).eps / 2
        live = (ids >= 0) & ~(lp == NINF)
        self.bad = (ids >= V).any(1)
        self.has = live.any(1) & ~self.bad
        live &= self.has[:, None]
        at = torch.where(live, ids, 0).long()
        t = torch.where(live, lp.double(), NINF)
        p = torch.exp(t) if tail else torch.softmax(torch.where(self.has[:, None], t, 0.0), 1) * live
        r = (1.0 - p.sum(1)).clamp_min(0.0) if tail else torch.zeros(R, dtype=torch.float64, device="cuda")
        xd = torch.where(self.has[:, None], x.double(), 0.0)
        z = xd / T
        self.lse = torch.logsumexp(z, 1)
        lq = z - self.lse[:, None]
        q = torch.exp(lq)
        inside = torch.zeros(R, V, dtype=torch.int32, device="cuda").scatter_add_(1, at, live.int()) > 0
        self.rest = torch.logsumexp(torch.where(inside, NINF, lq), 1)
        # (nothing outside the ids: a mass that float32 log-probabilities do not tell from none is none)
        r = torch.where((self.rest == NINF) & (r < 2.0 ** -20), 0.0, r)
        lqa = lq.gather(1, at)
        self.loss = torch.where(p > 0, p * (torch.log(p.clamp_min(1e-300)) - lqa), 0.0).sum(1)
        self.loss += torch.where(r > 0, r * (torch.log(r.clamp_min(1e-300)) - self.rest), 0.0)
        self.loss = torch.where(self.has, self.loss, 0.0)
        top = xd.amax(1, keepdim=True)
        D = (q * ((top - xd) / T).nan_to_num(posinf=0.0)).sum(1)
        self.e = (V / 256 + 40) * 2.0 ** -24 + 2.0 ** -22 * (8 + D)
        mass = p.sum(1) + r
        size = (p * (lqa.abs() + torch.log(p.clamp_min(1e-300)).abs())).nan_to_num(posinf=0.0).sum(1)
        self.tol = mass * 2 * self.e + 2.0 ** -23 * size + 2.0 ** -24 * self.loss.abs() + 1e-12
        target = torch.zeros(R, V, dtype=torch.float64, device="cuda").scatter_add_(1, at, p * live)
        bucket = torch.where(inside | (r == 0)[:, None], 0.0, r[:, None] * torch.exp(lq - self.rest[:, None]))
        rel = 2 * self.e[:, None] + 2.0 ** -21 * (1 + self.lse.abs()[:, None] + z.abs().nan_to_num(posinf=0.0))
        soft = q * mass[:, None]
        self.d = (soft - target - bucket) / T
        self.tol_d = (soft * rel + bucket * (rel + 2.0 ** -22 * self.rest.abs()[:, None].nan_to_num(posinf=0.0))
                      + target * 2.0 ** -22) / T
        self.eps = eps

    def grad(self, w):
        w = torch.where(self.has, w.double(), 0.0)[:, None]
        d = torch.where(self.has[:, None], w * self.d, 0.0)
        tol = torch.where(self.has[:, None], w.abs() * self.tol_d, 0.0)
        return d, tol + (d.abs() + tol) * self.eps + 1e-37


def check(x, ids, lp, w, T=1.0, tail=False, label=""):
    E = Exact(x, ids, lp, T, tail)
    loss, lse, rest, st = ops.distill(x, ids, lp, T, tail)
    within(loss, E.loss, E.tol, f"{label} loss")
    has = E.has
    within(lse[has], E.lse[has], (E.e + 2.0 ** -23 * E.lse.abs())[has], f"{label} lse")
    if tail:
        within(rest[has], E.rest[has], (2 * E.e + 2.0 ** -23 * E.rest.abs())[has].nan_to_num(posinf=0.0), f"{label} rest")
    else:
        assert bool((rest == 0).all())
    assert bool((loss[~has] == 0).all()) and bool((lse[~has] == 0).all())
    finite = E.loss.isfinite()
    want = torch.where(E.bad, N.EINVAL, torch.where(finite, N.OK, N.ENONFINITE)).to(torch.int32)
    assert torch.equal(st, want)
    d = ops.distill_grad(x, ids, lp, lse, rest, w, T, tail)
    within(d, *E.grad(w), f"{label} gradient")
    loss2, d2, st2 = ops.distill_step(x, ids, lp, w, T, tail)
    assert torch.equal(st2, st)
    within(loss2, E.loss, E.tol, f"{label} step's loss")
    within(d2, *E.grad(w), f"{label} step's gradient")
    assert bool((d2[~has] == 0).all())
    return d2, E


SIZES = [(1, 1, 1), (1, 5, 3), (2, 64, 64), (3, 257, 7), (5, 4_095, 33), (4, 4_097, 128), (17, 9_001, 1),
         (96, 32_768, 16), (300, 1_500, 20), (700, 5_003, 64), (1, 151_936, 64), (3, 248_320, 50),
         (300, 155_650, 64), (260, 160_001, 20), (258, 90_001, 20), (258, 150_001, 64), (130, 230_001, 33)]


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("R,V,M", SIZES)
def test_loss_and_gradients(R, V, M, dtype, tail):
    print(f"[distill] N={R} V={V} M={M} {dtype} tail={tail}", flush=True)
    x = logits(R, V, dtype, seed=R + V)
    T = 2.0 if M % 2 else 1.0
    ids, lp = teacher(x, M, T, seed=V)
    w = torch.randn(R, device="cuda", generator=gen(3))
    check(x, ids, lp, w, T, tail, f"N={R} V={V} M={M}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("pad,shift", [(3, 0), (8, 8), (1, 1)])
def test_strides_and_unaligned_rows(pad, shift, dtype):
    for R, V in ((5, 1_003), (3, 30_001), (300, 5_000)):
        print(f"[distill] pitch +{pad} shift {shift} N={R} V={V} {dtype}", flush=True)
        x = pitched(logits(R, V, dtype, seed=7), pad, shift)
        ids, lp = teacher(x, 20, 1.0, seed=8)
        w = torch.randn(R, device="cuda", generator=gen(9))
        d, E = check(x, ids, lp, w, 1.0, True, "pitched")
        into = pitched(torch.zeros_like(x), pad + 2, shift)
        guard = into.as_strided((R, pad + 2), (V + pad + 2, 1), into.storage_offset() + V)
        _, got, _ = ops.distill_step(x, ids, lp, w, 1.0, True, out=into)
        assert got is into and torch.equal(got, d) and bool(guard[:-1].isnan().all())
        # into the logits themselves, both ways
        loss, lse, rest, _ = ops.distill(x, ids, lp, 1.0, True)
        y = x.clone()
        assert torch.equal(ops.distill_grad(y, ids, lp, lse, rest, w, 1.0, True, out=y),
                           ops.distill_grad(x, ids, lp, lse, rest, w, 1.0, True))
        y = x.clone()
        assert torch.equal(ops.distill_step(y, ids, lp, w, 1.0, True, out=y)[1], d)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("R", [8, 400])
def test_rows_that_count_for_nothing(R, tail):
    """Rows without alternatives, with an id outside the vocabulary or weightless: no loss, no gradient,
    whatever they hold; the same id twice; padding between the alternatives; alternatives without mass."""
    V, M = 3_001, 12
    x = logits(R, V, torch.bfloat16, seed=5)
    ids, lp = teacher(x, M, 1.0, seed=6, ragged=False)
    w = torch.rand(R, device="cuda", generator=gen(7)) + 0.5
    x[0], ids[0] = float("nan"), -1              # nothing given, nothing finite
    lp[1] = NINF                                 # nothing with mass
    ids[2, 5] = V                                # an unknown id
    ids[3, 1::2] = -1                            # padding between, whatever its number is
    lp[3, 1::2] = float("nan")
    ids[4, 3] = ids[4, 0]                        # twice
    lp[4] -= 0.5                                 # (so that the teacher keeps some mass)
    lp[5, 4:] = NINF                             # ids without mass: padding, their tokens are the rest's
    w[6] = 0.0
    ids[7, 0], lp[7, 0] = ids[7, 0], 0.0         # all the mass on one
    lp[7, 1:] = -80.0
    check(x, ids, lp, w, 1.0, tail, "rows")
    d = ops.distill_step(x, ids, lp, w, 1.0, tail)[1]
    assert bool((d[[0, 1, 2, 6]] == 0).all())


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("R", [6, 300])
def test_extreme_rows(R, tail):
    """Student rows far from zero, certain of one token, almost empty outside the alternatives, or with
    -inf among them: a loss that is infinite has its status, and finite gradients."""
    V, M = 2_500, 8
    x = logits(R, V, torch.float32, seed=15)
    ids, lp = teacher(x, M, 1.0, seed=16, ragged=False)
    x[0] -= 3e4
    x[1, ids[1, 0].long()] = 300.0               # the rest's mass is exp(-290)
    x[2, torch.randint(0, V, (2_000,), device="cuda", generator=gen(17))] = NINF
    x[2].scatter_(0, ids[2].long(), 2.0)
    x[3] = NINF                                  # only the alternatives are possible
    x[3].scatter_(0, ids[3].long(), 1.0)
    x[4, ids[4, 2].long()] = NINF                # an alternative that the student excludes
    w = torch.ones(R, device="cuda")
    E = Exact(x, ids, lp, 1.0, tail)
    loss, lse, rest, st = ops.distill(x, ids, lp, 1.0, tail)
    want = torch.where(E.loss.isfinite(), N.OK, N.ENONFINITE).to(torch.int32)
    assert st[4] == N.ENONFINITE and torch.equal(st, want)
    fine = E.loss.isfinite()
    within(loss[fine], E.loss[fine], E.tol[fine], "loss")
    assert bool(loss[~fine].isinf().all())
    for d in (ops.distill_grad(x, ids, lp, lse, rest, w, 1.0, tail), ops.distill_step(x, ids, lp, w, 1.0, tail)[1]):
        ref, tol = E.grad(w)
        rows = [r for r in range(R) if r != 3]   # (row 3's bucket has no token to move)
        within(d[rows], ref[rows], tol[rows], "gradient")
        assert bool(d[3].isfinite().all()) and bool((d[3][x[3] == NINF] == 0).all())
    bad = x.clone()
    bad[0, 7], bad[1, 9] = float("nan"), float("inf")
    loss, _, _, st = ops.distill(bad, ids, lp, 1.0, tail)
    assert st[:2].tolist() == [N.ENONFINITE] * 2 and bool(loss[:2].isnan().all())


def test_a_teacher_of_its_own():
    """A teacher that is the student: no divergence, no gradient but for rounding, also in the bucket."""
    x = logits(50, 20_000, torch.float32, seed=21)
    out = ops.token_scores(x, top=64, temperature=1.5)
    w = torch.ones(50, device="cuda")
    for tail in (False, True):
        E = Exact(x, out.top_ids, out.top_logprobs, 1.5, tail)
        loss, d, st = ops.distill_step(x, out.top_ids, out.top_logprobs, w, 1.5, tail)
        assert bool((st == 0).all())
        within(loss, E.loss, E.tol, "loss")
        within(d, *E.grad(w), "gradient")
    assert float(loss.abs().max()) < 1e-5


def test_differences():
    """The gradient along directions against differences of the loss: steps of 1/16 on a grid of 1/8; the
    third derivative along a step h of the logits is below 8 (sum p + r) h^3, the loss is off by 1e-5."""
    R, V, M = 16, 900, 12
    x = (torch.randn(R, V, device="cuda", generator=gen(20)) * 8).round() / 8
    ids, lp = teacher(x, M, 1.0, seed=22)
    for tail in (False, True):
        _, lse, rest, _ = ops.distill(x, ids, lp, 1.0, tail)
        grad = ops.distill_grad(x, ids, lp, lse, rest, torch.ones(R, device="cuda"), 1.0, tail)
        for s in range(6):
            d = torch.where(torch.rand(R, V, device="cuda", generator=gen(30 + s)) < 0.5, -1.0, 1.0)
            up, dn = (ops.distill(x + k * d, ids, lp, 1.0, tail)[0] for k in (1 / 16, -1 / 16))
            diff, lin = (up - dn).double() * 8, (grad.double() * d).sum(1)
            tol = 16e-5 + 8 * 8 / 16 ** 3 / 6
            assert bool(((diff - lin).abs() <= tol).all()), float(((diff - lin).abs() - tol).max())


def test_past_32_bits():
    R, V, M = 14_200, 151_936, 4
    x = torch.zeros(R, V, dtype=torch.bfloat16, device="cuda")
    last = [0, 7_000, R - 1]
    x[last] = logits(3, V, torch.bfloat16, seed=3)
    ids = torch.full((R, M), -1, dtype=torch.int32, device="cuda")
    lp = torch.zeros(R, M, device="cuda")
    ids[last], lp[last] = teacher(x[last], M, 1.0, seed=4, ragged=False)
    w = torch.ones(R, device="cuda")
    E = Exact(x[last], ids[last], lp[last], 1.0, True)
    loss, d, st = ops.distill_step(x, ids, lp, w, 1.0, True, out=x)
    within(loss[last], E.loss, E.tol, "loss")
    within(d[last], *E.grad(w[:3]), "gradient")
    assert int((loss != 0).sum()) == 3 and bool((d[1:7_000] == 0).all())


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_autograd(reduction):
    """Shapes, id types, reductions, a gradient that comes back other than 1, a graph gone through twice,
    no gradient wanted, second derivatives refused."""
    x = logits(60, 700, torch.float32, seed=31)
    ids, lp = teacher(x, 9, 1.0, seed=32)
    ids3 = ids.reshape(3, 20, 9).long()
    ids3[0, 0, 0] = 2 ** 40
    ids[0, 0] = 700
    lp3 = lp.reshape(3, 20, 9)
    E = Exact(x, ids, lp, 1.0, True)
    count = int(E.has.sum())
    w = torch.full((60,), {"mean": 1.0 / count, "sum": 1.0, "none": 0.25}[reduction], device="cuda")
    leaf = x.reshape(3, 20, 700).clone().requires_grad_()
    value = L.distill_loss(leaf, ids3, lp3, tail=True, reduction=reduction)
    assert value.shape == ((3, 20) if reduction == "none" else ())
    total = (value * 0.25).sum() if reduction == "none" else value
    total.backward(retain_graph=True)
    within(leaf.grad.reshape(60, 700), *E.grad(w), "gradient")
    first = leaf.grad.clone()
    leaf.grad = None
    total.backward()
    assert torch.equal(leaf.grad, first)
    scale = 1.0 if reduction == "none" else float(w[0])
    if reduction != "none":
        assert abs(float(value.detach()) - float(E.loss.sum()) * scale) <= float((E.tol.sum() + 1e-5 * E.loss.sum()) * scale)
        leaf.grad = None
        (L.distill_loss(leaf, ids3, lp3, tail=True, reduction=reduction) * 4.0).backward()
        assert torch.equal(leaf.grad, first * 4.0)
    assert not L.distill_loss(x, ids, lp, reduction=reduction).requires_grad
    (d,) = torch.autograd.grad(L.distill_loss(leaf, ids3, lp3, reduction=reduction).sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        d.square().sum().backward()


def test_scale():
    for dtype in (torch.bfloat16, torch.float32):
        for n in (1, 7, 1_000_003):
            x = torch.randn(n, device="cuda", generator=gen(n)).to(dtype)
            for f in (1.0, 0.5, -3.0, 0.0):
                y = x.clone()
                assert ops.distill_scale(y, torch.tensor(f, device="cuda")) is y
                assert torch.equal(y, (x.float() * f).to(dtype))


def test_repeatable_streams_and_graphs():
    for R, V in ((40, 50_003), (300, 9_001)):
        x, x2 = (logits(R, V, torch.bfloat16, seed=s) for s in (41, 42))
        ids, lp = teacher(x, 30, 1.0, seed=43)
        w = torch.randn(R, device="cuda", generator=gen(44))

        def run(**kw):
            loss, lse, rest, st = ops.distill(x, ids, lp, 1.0, True, **kw)
            return [loss, lse, rest, st, ops.distill_grad(x, ids, lp, lse, rest, w, 1.0, True, **kw),
                    *ops.distill_step(x, ids, lp, w, 1.0, True, **kw)]

        ref = run()
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        got = run(stream=stream)
        torch.cuda.current_stream().wait_stream(stream)
        for a, b in zip(got, ref):
            assert torch.equal(a, b)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = run()
        keep = x.clone()
        for src in (x2, keep, x2):
            x.copy_(src)
            ref = run()
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(res, ref):
                assert torch.equal(a, b)


def test_refusals():
    x = logits(4, 100, torch.bfloat16, seed=1)
    ids, lp = teacher(x, 5, 1.0, seed=2, ragged=False)
    w = torch.ones(4, device="cuda")
    _, lse, rest, _ = ops.distill(x, ids, lp)
    bad = [lambda: ops.distill(x.T, ids, lp), lambda: ops.distill(x, ids[:3], lp),
           lambda: ops.distill(x, ids.long(), lp), lambda: ops.distill(x, ids, lp.double()),
           lambda: ops.distill(x, ids, lp[:, :4]), lambda: ops.distill(x, ids[:, :0], lp[:, :0]),
           lambda: ops.distill(x, ids.repeat(1, 26), lp.repeat(1, 26)),
           lambda: ops.distill(x, ids, lp, temperature=-1.0), lambda: ops.distill(x, ids.cpu(), lp),
           lambda: ops.distill(x, ids[:, ::2], lp[:, ::2]), lambda: ops.distill(x.cpu(), ids, lp),
           lambda: ops.distill_grad(x, ids, lp, lse[:3], rest, w),
           lambda: ops.distill_grad(x, ids, lp, lse, rest, w.double()),
           lambda: ops.distill_step(x, ids, lp, w[:3]),
           lambda: ops.distill_step(x, ids, lp, w, out=x.float()),
           lambda: ops.distill_step(x, ids, lp, w, out=torch.empty(100, 4, dtype=x.dtype, device="cuda").T),
           lambda: ops.distill_scale(x, w), lambda: ops.distill_scale(x.T, w[:1]),
           lambda: L.distill_loss(x, ids, lp, reduction="max"), lambda: L.distill_loss(x, ids[:3], lp[:3]),
           lambda: L.distill_loss(x, ids, lp.clone().requires_grad_())]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        ops.distill(x.half(), ids, lp)
    with pytest.raises(TypeError):
        L.distill_loss(x, ids.float(), lp)
