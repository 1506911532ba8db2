"""Cross entropy over the vocabulary (strim_head_loss, strim_head_loss_grad and their
differentiable form) against the formulas in float64, and against differences.

The bounds follow from how the kernels round, with S = max_v sum_k |hidden||lm_head|:
  a logit: 1e-6 S (float32 accumulation, as tests/test_head_gpu.py has it); so a loss or a
  log-sum-exp: e = 2e-6 S + 4e-6 (the exponentials' and the logarithm's rounding, the sums)
  + 2^-22 |lse|;
  p: 2^-8 of it (bf16) and 2 e + 2^-20 of the softmax term (its exponent);
  a gradient: those errors times |weights| summed, 1e-6 of the sum of |products| for the
  float32 accumulation, and 2^-8 of itself (bf16)."""
import ctypes

import numpy as np
import pytest
import torch

from strim_amd import _native as N
from strim_amd import loss as L
from strim_amd import ops

pytestmark = pytest.mark.gpu


def inputs(R, K, V, seed, ignored=0.2, wscale=None, stride=None):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    w = torch.randn(V, K, device="cuda", generator=g) * (wscale or K ** -0.5)
    t = torch.randint(0, V, (R,), device="cuda", generator=g)
    h = 2.0 * torch.randn(R, K, device="cuda", generator=g)
    h += 8.0 * torch.rand(R, 1, device="cuda", generator=g) * w[t]
    t = torch.where(torch.rand(R, device="cuda", generator=g) < ignored, -100, t)
    gl = torch.randn(R, device="cuda", generator=g)
    h, w = h.to(torch.bfloat16), w.to(torch.bfloat16)
    if stride:
        h, w = pitched(h, stride), pitched(w, stride)
    return h, w, t.to(torch.int32), gl


def pitched(t, pad):
    buf = torch.full((t.shape[0], t.shape[1] + pad), float("nan"), dtype=t.dtype, device=t.device)
    buf[:, :t.shape[1]] = t
    return buf[:, :t.shape[1]]


class Exact:
    """The formulas in float64, and the bounds above."""

    def __init__(self, h, w, t, gl=None, gz=None):
        self.live = (t >= 0) & (t < w.shape[0])
        hd = torch.where(self.live[:, None], h.double(), 0.0)  # what padding holds counts for nothing
        wd = w.double()
        at = torch.where(self.live, t, 0).long()[:, None]
        x = hd @ wd.T
        S = (hd.abs() @ wd.abs().T).amax(1)
        self.lse = torch.logsumexp(x, 1)
        self.loss = torch.where(self.live, self.lse - x.gather(1, at)[:, 0], 0.0)
        e = 2e-6 * S + 4e-6 + 2.0 ** -22 * self.lse.abs()
        self.tol = e
        if gl is None:
            return
        g = torch.where(self.live, gl.double(), 0.0)
        top = g if gz is None else g + torch.where(self.live, gz.double(), 0.0)
        soft = torch.exp(x - self.lse[:, None]) * top[:, None]
        p = soft.clone()
        p.scatter_add_(1, at, -g[:, None])
        ep = 2.0 ** -8 * p.abs() + (2 * e + 2.0 ** -20)[:, None] * soft.abs() + 1e-6 * p.abs()
        self.dh, eh = p @ wd, ep @ wd.abs()
        self.dw, ew = p.T @ hd, ep.T @ hd.abs()
        self.tol_h = eh + 2.0 ** -8 * (self.dh.abs() + eh) + 1e-30
        self.tol_w = ew + 2.0 ** -8 * (self.dw.abs() + ew) + 1e-30


def within(got, ref, tol, what):
    err = (got.double() - ref).abs()
    bad = ~(err <= tol)
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} past the bound, worst "
                                 f"{float((err / tol).nan_to_num(1e9).max()):.3g} of it")


def check(h, w, t, gl, gz=None, label=""):
    R = h.shape[0]
    E = Exact(h, w, t, gl, gz)
    loss, lse, st = ops.head_loss(h, w, t)
    within(loss, E.loss, E.tol, f"{label} loss")
    within(lse[E.live], E.lse[E.live], E.tol[E.live], f"{label} lse")
    assert bool((loss[~E.live] == 0).all())
    bad = ~E.live & (t != -100)
    assert torch.equal(st, torch.where(bad, N.EINVAL, N.OK).to(torch.int32))
    dh, dw = ops.head_loss_grad(h, w, t, lse, gl, gz)
    within(dh, E.dh, E.tol_h, f"{label} d_hidden")
    within(dw, E.dw, E.tol_w, f"{label} d_lm_head")
    assert bool((dh[~E.live] == 0).all())
    # one at a time, the same bits
    only_h, none = ops.head_loss_grad(h, w, t, lse, gl, gz, want_lm_head=False)
    assert none is None and torch.equal(only_h, dh)
    none, only_w = ops.head_loss_grad(h, w, t, lse, gl, gz, want_hidden=False)
    assert none is None and torch.equal(only_w, dw)
    return loss, lse, dh, dw


SIZES = [(1, 8, 1), (1, 64, 5), (2, 72, 64), (3, 128, 257), (17, 136, 300), (63, 256, 1000),
         (64, 264, 255), (65, 64, 777), (128, 520, 511), (129, 1032, 513), (255, 72, 2049),
         (257, 248, 1500), (300, 2056, 3001), (1025, 40, 260), (40, 5120, 4099)]


@pytest.mark.parametrize("R,K,V", SIZES)
def test_loss_and_gradients(R, K, V):
    print(f"[loss] N={R} K={K} V={V}", flush=True)
    check(*inputs(R, K, V, seed=R + 7 * K + V), label=f"N={R} K={K} V={V}")


@pytest.mark.parametrize("R,K,V", [(5, 72, 130), (70, 64, 300), (200, 136, 515)])
def test_strided_rows_and_gradient_of_lse(R, K, V):
    print(f"[loss] strided N={R} K={K} V={V}", flush=True)
    h, w, t, gl = inputs(R, K, V, seed=3, stride=24)
    assert h.stride(0) == K + 24
    gz = torch.linspace(-1.0, 2.0, R, device="cuda")
    check(h, w, t, gl, gz, "strided")


def test_pieces_of_the_vocabulary():
    """Enough rows and vocabulary for several pieces, the last one short."""
    R, K, V = 2050, 64, 200_003
    need = ops.head_loss_workspace(R, K, V, True, True)
    assert need < 2 * R * V  # the probabilities are not all held
    h, w, t, gl = inputs(R, K, V, seed=11)
    loss, lse, _ = ops.head_loss(h, w, t)
    dh, dw = ops.head_loss_grad(h, w, t, lse, gl)
    # the formula by pieces of the rows
    dwr = torch.zeros(V, K, dtype=torch.float64, device="cuda")
    tol_w = torch.zeros_like(dwr)
    for a in range(0, R, 410):
        s = slice(a, a + 410)
        E = Exact(h[s], w, t[s], gl[s])
        within(loss[s], E.loss, E.tol, "loss")
        within(dh[s], E.dh, E.tol_h, "d_hidden")
        dwr += E.dw
        tol_w += E.tol_w
    within(dw, dwr, tol_w + 2.0 ** -8 * dwr.abs(), "d_lm_head")


@pytest.mark.parametrize("R,K,V", [(1000, 1536, 66_003), (1003, 2048, 33_100), (2050, 1024, 33_281)])
def test_rest_in_smaller_tiles(R, K, V):
    """More tiles than whole rounds over the chip, so that the last of the vocabulary is computed
    apart in smaller ones: targets on both sides of every seam."""
    print(f"[loss] rest N={R} K={K} V={V}", flush=True)
    h, w, t, gl = inputs(R, K, V, seed=V, ignored=0.1)
    edge = V - 1 - 64 * torch.arange(200, device="cuda")
    t[:200] = edge.to(torch.int32)
    check(h, w, t, gl, label=f"N={R} K={K} V={V}")


def test_padding_counts_for_nothing():
    """Rows without a target, and with one outside the vocabulary: no loss, no gradient,
    whatever their states and their gradients hold."""
    R, K, V = 140, 128, 700
    h, w, t, gl = inputs(R, K, V, seed=5, ignored=0.3)
    t[3], t[77], t[78] = V, -1, 2 ** 31 - 1
    dead = (t < 0) | (t >= V)
    h[dead] = float("nan")
    h[3] = float("inf")
    gl[dead] = float("nan")
    check(h, w, t, gl, label="padding")
    # another ignore index: an id of the vocabulary
    t2 = torch.where(dead, 9, t).to(torch.int32)
    live = t2 != 9
    loss, lse, st = ops.head_loss(h, w, t2, ignore_index=9)
    assert bool((st == 0).all()) and bool((loss[~live] == 0).all())
    dh, dw = ops.head_loss_grad(h, w, t2, lse, gl, ignore_index=9)
    E = Exact(h, w, torch.where(live, t2, -100), gl)
    within(dh, E.dh, E.tol_h, "d_hidden")
    within(dw, E.dw, E.tol_w, "d_lm_head")


def test_all_rows_ignored_and_no_rows():
    h, w, t, gl = inputs(6, 64, 300, seed=2, ignored=1.0)
    loss, lse, st = ops.head_loss(h, w, t)
    dh, dw = ops.head_loss_grad(h, w, t, lse, gl)
    assert bool((loss == 0).all()) and bool((dh == 0).all()) and bool((dw == 0).all())
    loss, lse, st = ops.head_loss(h[:0], w, t[:0])
    assert loss.shape == (0,)
    dh, dw = ops.head_loss_grad(h[:0], w, t[:0], lse, gl[:0])
    assert dh.shape == (0, 64) and bool((dw == 0).all())


def test_extreme_logits():
    """Rows whose logits are all far below zero, hugely spread, or equal; and statuses of rows
    that are not finite."""
    K, V = 64, 600
    w = torch.zeros(V, K, device="cuda")
    w[:, 0] = -1.0
    w[5, 0] = 1.0
    w[:, 1] = torch.linspace(-50, 50, V, device="cuda")
    h = torch.zeros(5, K, device="cuda")
    h[0, 0], h[1, 0], h[2, 1], h[4, 2] = 3e4, 64.0, 8.0, 1.0
    t = torch.tensor([5, 7, 599, 0, 1], dtype=torch.int32, device="cuda")
    h, w = h.to(torch.bfloat16), w.to(torch.bfloat16)
    gl = torch.ones(5, device="cuda")
    check(h, w, t, gl, label="extreme")
    bad = h.clone()
    bad[1, 0], bad[2, 1] = float("nan"), float("inf")
    loss, lse, st = ops.head_loss(bad, w, t)
    assert st.tolist() == [N.OK, N.ENONFINITE, N.ENONFINITE, N.OK, N.OK]
    # -inf logits beside finite ones, a whole tile of them
    wi = torch.full((700, K), -1.0, device="cuda", dtype=torch.bfloat16)
    wi[:600, 0] = float("-inf")
    hi = torch.zeros(1, K, device="cuda", dtype=torch.bfloat16)
    hi[0, 0] = 1.0
    loss, lse, st = ops.head_loss(hi, wi, torch.tensor([650], dtype=torch.int32, device="cuda"))
    assert abs(float(loss) - np.log(100)) < 1e-5 and st.tolist() == [N.OK]


def test_differences():
    """The gradient along directions against differences of the loss itself: states on a grid
    of 1/8, so that a step of 1/16 either way is exact in bf16. The third-order term is (step
    change of a logit, below 0.1)^3 / 6 over a step of 1/16; the loss's own error 1e-5."""
    R, K, V = 33, 64, 900
    g = torch.Generator(device="cuda")
    g.manual_seed(8)
    h = (torch.randn(R, K, device="cuda", generator=g) * 8).round().clamp(-60, 60) / 8
    w = (torch.randn(V, K, device="cuda", generator=g) * 0.1).to(torch.bfloat16)
    t = torch.randint(0, V, (R,), device="cuda", generator=g).to(torch.int32)
    _, lse, _ = ops.head_loss(h.to(torch.bfloat16), w, t)
    one = torch.ones(R, device="cuda")
    dh, _ = ops.head_loss_grad(h.to(torch.bfloat16), w, t, lse, one)
    for _ in range(8):
        d = torch.where(torch.rand(R, K, device="cuda", generator=g) < 0.5, -1.0, 1.0)
        d *= torch.rand(R, K, device="cuda", generator=g) < 0.25
        up, _, _ = ops.head_loss((h + d / 16).to(torch.bfloat16), w, t)
        dn, _, _ = ops.head_loss((h - d / 16).to(torch.bfloat16), w, t)
        diff = (up - dn).double() * 8
        lin = (dh.double() * d).sum(1)
        tol = 16e-5 + 0.1 ** 3 / 6 * 16 + 2.0 ** -8 * (dh.double() * d).abs().sum(1)
        assert bool(((diff - lin).abs() <= tol).all()), float(((diff - lin).abs() - tol).max())


def test_autograd():
    """The differentiable form: shapes, target types, reductions, gradients through both
    outputs, a broadcast upstream gradient, a frozen projection, int64 ids past 32 bits."""
    h, w, t, _ = inputs(60, 72, 500, seed=31, ignored=0.3)
    h3, t3 = h.reshape(3, 20, 72).clone().requires_grad_(), t.reshape(3, 20).long()
    t3[0, 0], t3[0, 1], t3[2, 19] = 500, 2 ** 40, -2 ** 40
    ids = torch.where((t3 >= 0) & (t3 < 500), t3, -100).reshape(-1).int()
    count = int((ids >= 0).sum())
    w1 = w.clone().requires_grad_()
    value = L.head_cross_entropy(h3, w1, t3)
    value.backward()
    value = value.detach()
    g = torch.full((60,), 1.0 / count, device="cuda")
    E = Exact(h, w, ids, g)
    assert abs(float(value) - float(E.loss.sum()) / count) < float(E.tol.max()) + 1e-6 * float(value)
    within(h3.grad.reshape(60, 72), E.dh, E.tol_h, "d_hidden")
    within(w1.grad, E.dw, E.tol_w, "d_lm_head")
    # the sum, with a frozen projection; the log-sum-exp's gradient beside it
    h4 = h.clone().requires_grad_()
    value, lse, status = L.head_loss(h4, w, ids)
    assert not status.requires_grad
    (value.sum() + (lse * 0.25).sum()).backward()
    E = Exact(h, w, ids, torch.ones(60, device="cuda"), torch.full((60,), 0.25, device="cuda"))
    within(h4.grad, E.dh, E.tol_h, "d_hidden")
    # the log-sum-exp alone
    w2 = w.clone().requires_grad_()
    L.head_loss(h, w2, ids)[1].sum().backward()
    E = Exact(h, w, ids, torch.zeros(60, device="cuda"), torch.ones(60, device="cuda"))
    within(w2.grad, E.dw, E.tol_w, "d_lm_head")
    lp = L.token_logprobs(h, w, ids.clamp_min(0))
    E = Exact(h, w, ids.clamp_min(0))
    within(-lp, E.loss, E.tol, "log-probabilities")
    assert float(L.head_cross_entropy(h, w, torch.full_like(ids, -100))) == 0.0
    with pytest.raises(ValueError):
        L.head_cross_entropy(h, w, t3)
    with pytest.raises(TypeError):
        L.head_cross_entropy(h, w, ids.float())
    with pytest.raises(ValueError):
        L.head_cross_entropy(h, w, ids, reduction="max")


def test_weights_of_many_sizes():
    """Rows whose weights span many powers of two, the first of them ignored or weightless."""
    h, w, t, gl = inputs(150, 64, 400, seed=41, ignored=0.0)
    t[:70] = -100
    gl *= torch.exp2(torch.arange(150, device="cuda") % 40 - 20.0)
    gl[70:75] = 0.0
    check(h, w, t, gl, label="weights")
    gz = gl.flip(0).contiguous()
    check(h, w, t, torch.zeros_like(gl), gz, label="weights of lse")


def test_repeatable_and_in_a_graph():
    h, w, t, gl = inputs(200, 256, 3000, seed=21)
    loss, lse, _ = ops.head_loss(h, w, t)
    dh, dw = ops.head_loss_grad(h, w, t, lse, gl)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        out = [ops.head_loss(h, w, t)[:2]]
        out += [ops.head_loss_grad(h, w, t, out[0][1], gl)]
    torch.cuda.current_stream().wait_stream(st)
    for a, b in zip((loss, lse, dh, dw), (*out[0], *out[1])):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gloss, glse, _ = ops.head_loss(h, w, t)
        gdh, gdw = ops.head_loss_grad(h, w, t, glse, gl)
    h2, _, t2, gl2 = inputs(200, 256, 3000, seed=22)
    for a, b, c in ((h, t, gl), (h2, t2, gl2), (h, t, gl)):
        sa, sb, sc = a.clone(), b.clone(), c.clone()
        h.copy_(sa), t.copy_(sb), gl.copy_(sc)
        graph.replay()
        torch.cuda.synchronize()
        loss, lse, _ = ops.head_loss(h, w, t)
        dh, dw = ops.head_loss_grad(h, w, t, lse, gl)
        for x, y in zip((loss, lse, dh, dw), (gloss, glse, gdh, gdw)):
            assert torch.equal(x, y)


def test_refusals():
    h, w, t, gl = inputs(4, 64, 100, seed=1)
    _, lse, _ = ops.head_loss(h, w, t)
    with pytest.raises(TypeError):
        ops.head_loss(h.float(), w, t)
    with pytest.raises(ValueError):
        ops.head_loss(h, w, t.long())
    with pytest.raises(ValueError):
        ops.head_loss(h, w[:, :56], t)
    with pytest.raises(ValueError):
        ops.head_loss(h.cpu(), w, t)
    with pytest.raises(ValueError):
        ops.head_loss(h.T, w, t)
    with pytest.raises(ValueError):
        ops.head_loss_grad(h, w, t, lse, gl.double())
    with pytest.raises(ValueError):
        ops.head_loss_grad(h, w, t, lse, gl[:1].expand(4))
    with pytest.raises(ValueError):
        ops.head_loss(h, w, t, workspace=torch.empty(8, dtype=torch.uint8, device="cuda"))
    with pytest.raises(N.StrimError):  # K not a multiple of 8
        ops.head_loss(h[:, :60].contiguous(), w[:, :60].contiguous(), t)
    with pytest.raises(N.StrimError):  # rows not 16-byte aligned
        ops.head_loss(h[:, 4:60], w[:, 4:60].contiguous(), t)
    lib, s = N.lib(), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    ws = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    f = torch.empty(3, 4, device="cuda")

    def p(x):
        return ctypes.c_void_p(x.data_ptr())

    def call(**kw):
        a = dict(N=4, K=64, V=100, hs=64, ws=64, t=p(t), wsp=p(ws), wb=1 << 20, loss=p(f[0]))
        a.update(kw)
        return lib.strim_head_loss(s, p(h), a["hs"], a["N"], a["K"], p(w), a["ws"], a["V"], a["t"],
                                   -100, a["wsp"], a["wb"], a["loss"], None, None)

    assert call() == N.OK
    assert call(N=0) == N.OK
    assert call(N=-1) == N.EINVAL
    assert call(V=0) == N.EINVAL
    assert call(K=0) == N.EINVAL
    assert call(hs=56) == N.EINVAL
    assert call(ws=68) == N.EINVAL
    assert call(ws=N.LOSS_MAX_STRIDE + 8) == N.EINVAL
    assert call(t=None) == N.EINVAL
    assert call(loss=None) == N.EINVAL
    assert call(wsp=None) == N.EINVAL
    assert call(wb=16) == N.ECAPACITY
    assert lib.strim_head_loss_workspace(4, 60, 100, 0, 0) == N.EINVAL
    torch.cuda.synchronize()


def test_offsets_past_32_bits():
    """A projection, and its gradient, of more than 2^31 elements: rows at both ends."""
    V, K, R = 210_000, 10_240, 3
    print("[loss] 2^31 elements", flush=True)
    g = torch.Generator(device="cuda")
    g.manual_seed(51)
    w = torch.randn(V, K, device="cuda", generator=g, dtype=torch.bfloat16).mul_(0.01)
    t = torch.tensor([V - 1, 0, V - 131], dtype=torch.int32, device="cuda")
    h = (torch.randn(R, K, device="cuda", generator=g) + 30 * w[t.long()].float()).to(torch.bfloat16)
    x = torch.cat([h.double() @ w[a:a + 30_000].double().T for a in range(0, V, 30_000)], 1)
    lse = torch.logsumexp(x, 1)
    ref = lse - x.gather(1, t.long()[:, None])[:, 0]
    S = max(float((h[i].double().abs() * w[t[i].long()].double().abs()).sum()) for i in range(R)) * 2
    e = 2e-6 * S + 4e-6 + 2.0 ** -22 * float(lse.abs().max())
    loss, got, _ = ops.head_loss(h, w, t)
    assert float((loss.double() - ref).abs().max()) <= e
    one = torch.ones(R, device="cuda")
    _, dw = ops.head_loss_grad(h, w, t, got, one, want_hidden=False)
    p = torch.exp(x - lse[:, None])
    p.scatter_add_(1, t.long()[:, None], -one.double()[:, None])
    for rows in (slice(0, 40), slice(V - 140, V)):
        want = p[:, rows].T @ h.double()
        bound = (p[:, rows].abs().T @ h.double().abs()) * (2.0 ** -7 + 4 * e) + 1e-30
        # (not the targets' rows, where p is the small difference of two rounded terms)
        other = torch.ones(V, dtype=torch.bool, device="cuda")
        other[t.long()] = False
        other = other[rows]
        within(dw[rows][other], want[other], bound[other], "d_lm_head")


def test_many_rows():
    """More rows than a workgroup's worth of everything, at the smallest sizes."""
    R, K, V = 70_001, 16, 300
    h, w, t, gl = inputs(R, K, V, seed=61)
    check(h, w, t, gl, label="many rows")


LOW = [(1, 64, 5), (3, 72, 601), (17, 64, 1023), (40, 136, 4099), (257, 64, 1501), (129, 256, 50_257),
       (1000, 1536, 66_003), (1003, 2048, 33_100), (2050, 1024, 33_281)]


def low_inputs(R, K, V, seed):
    """Every row's logits around one number, from -30,000 to 64, most of them below -88.7 (where
    exp(-lse) is past float32), and a vocabulary that ends inside a 16-byte piece."""
    h, w, t, gl = inputs(R, K, V, seed=seed, ignored=0.1)
    w[:, 0] = -1.0
    h[:, 0] = torch.tensor([96.0, 88.0, 128.0, 90.0, -64.0, 1024.0, 100.0, 30_000.0, 0.0],
                           device="cuda").repeat(-(-R // 9))[:R].to(torch.bfloat16)
    return h, w, t, gl


@pytest.mark.parametrize("R,K,V", LOW)
def test_logits_far_below_zero(R, K, V):
    """Nothing bounds a row's logits from below: no weight of a token past the vocabulary, whose
    logit would be 0, reaches the gradients. Single tiles, whole rounds, and what is left of them
    in smaller tiles."""
    print(f"[loss] far below zero N={R} K={K} V={V}", flush=True)
    assert V % 8
    check(*low_inputs(R, K, V, seed=V), label=f"N={R} K={K} V={V}")


def test_logits_far_below_zero_in_pieces():
    """The same where the last of several pieces of the vocabulary is the short one."""
    R, K, V = 2050, 64, 200_003
    assert ops.head_loss_workspace(R, K, V, True, False) < 2 * R * V + 4 * R * K
    h, w, t, gl = low_inputs(R, K, V, seed=12)
    _, lse, _ = ops.head_loss(h, w, t)
    dh, _ = ops.head_loss_grad(h, w, t, lse, gl, want_lm_head=False)
    for a in range(0, R, 410):
        s = slice(a, a + 410)
        E = Exact(h[s], w, t[s], gl[s])
        within(dh[s], E.dh, E.tol_h, "d_hidden")


def test_more_tiles_than_a_launch_has():
    """As many rows as there may be by a wide vocabulary: 2^23 tiles of 512 threads, more threads
    than one launch can have. The rows repeat a thousand."""
    R, K, V, M = 1024, 8, 131_584, 4096
    print(f"[loss] N={R * M} K={K} V={V}", flush=True)
    h, w, t, _ = inputs(R, K, V, seed=71)
    E = Exact(h, w, t)
    loss, lse, st = ops.head_loss(h.repeat(M, 1), w, t.repeat(M))
    assert int(st.abs().max()) == N.OK
    for i in range(0, M, 512):
        a = slice(i * R, (i + 512) * R)
        err = (loss[a].double().view(-1, R) - E.loss).abs().amax(0)
        assert bool((err <= E.tol).all()), (i, float((err / E.tol).max()))
        err = (lse[a].double().view(-1, R) - E.lse).abs().amax(0)
        assert bool((err <= E.tol)[E.live].all()), (i, float((err / E.tol)[E.live].max()))


def test_more_gradients_than_a_launch_has():
    """The hidden states' gradients of more elements than 2^34, four of which a thread adds. The
    rows repeat 64."""
    R, K, V, M = 64, 4104, 8, 1 << 16
    print(f"[loss] N={R * M} K={K} V={V}", flush=True)
    h, w, t, gl = inputs(R, K, V, seed=72)
    _, lse, _ = ops.head_loss(h, w, t)
    need = ops.head_loss_workspace(R * M, K, V, True, False) + 5 * R * M * K
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < need:
        pytest.skip(f"needs {need >> 30} GB of memory")
    E = Exact(h, w, t, gl)
    rows = [x.repeat(M, *[1] * (x.dim() - 1)) for x in (h, t, lse, gl)]
    dh, _ = ops.head_loss_grad(rows[0], w, *rows[1:], want_lm_head=False)
    for i in range(0, M, 512):
        got = dh[i * R:(i + 512) * R].float().view(-1, R, K)
        lo, hi = got.amin(0).double(), got.amax(0).double()
        within(lo, E.dh, E.tol_h, f"d_hidden, least of rows {i * R} on")
        within(hi, E.dh, E.tol_h, f"d_hidden, largest of rows {i * R} on")
    del rows, dh, got
    torch.cuda.empty_cache()


def test_products_without_steps():
    """Workgroups that have nothing to add (no rows; a part of the vocabulary's last piece that is
    empty) leave nothing under way for those that have their place next."""
    h, w, t, gl = inputs(300, 256, 40_000, seed=81)
    ref = ops.head_loss(h, w, t)
    grads = ops.head_loss_grad(h, w, t, ref[1], gl)
    for _ in range(4):
        _, zero = ops.head_loss_grad(h[:0], w, t[:0], ref[1][:0], gl[:0], want_hidden=False)
        got = ops.head_loss(h, w, t)
        assert torch.equal(zero, torch.zeros_like(w))
        again = ops.head_loss_grad(h, w, t, got[1], gl)
        for a, b in zip((*got, *again), (*ref, *grads)):
            assert torch.equal(a, b)
    # a vocabulary in pieces
    R, K, V = 2050, 64, 65_536 * 2 + 65
    h, w, t, gl = inputs(R, K, V, seed=82)
    _, lse, _ = ops.head_loss(h, w, t)
    dh, _ = ops.head_loss_grad(h, w, t, lse, gl, want_lm_head=False)
    for a in range(0, R, 410):
        s = slice(a, a + 410)
        E = Exact(h[s], w, t[s], gl[s])
        within(dh[s], E.dh, E.tol_h, "d_hidden")


@pytest.mark.parametrize("V", [9, 300, 5001])
def test_small_losses_beside_large_logits(V):
    """A loss is as exact as its own size allows, and not only to the log-sum-exp's spacing: logits
    that are exact in bf16 and float32, the target's the largest by d, so that the loss is log(1 +
    (V - 1) exp(-d)). Bound: some thirty additions of a sum near 1 (2^-24 each), and an exponential's
    and a logarithm's few 2^-24 of their own."""
    for top in (40.0, 992.0, -992.0, -30_464.0):
        for d in (8.0, 16.0) if abs(top) < 1000 else (256.0, 512.0):
            w = torch.zeros(V, 8, device="cuda")
            w[:, 0], w[V // 2, 0] = top - d, top
            h = torch.zeros(2, 8, device="cuda")
            h[:, 0] = 1.0
            w, h = w.to(torch.bfloat16), h.to(torch.bfloat16)
            assert float(w[V // 2, 0]) == top and float(w[0, 0]) == top - d
            loss, lse, _ = ops.head_loss(h, w, torch.tensor([V // 2, 0], dtype=torch.int32, device="cuda"))
            ref = np.log1p((V - 1) * np.exp(-d))
            assert abs(float(loss[0]) - ref) <= 2e-6 + 4e-6 * ref, (top, d)
            assert abs(float(loss[1]) - (ref + d)) <= 2e-6 + 4e-6 * ref + 2.0 ** -24 * (ref + d), (top, d)
            assert abs(float(lse[0]) - (top + ref)) <= 2e-6 + 4e-6 * ref + 2.0 ** -24 * abs(top + ref), (top, d)
