"""Norms with gradients (strim_norm, strim_norm_grad and their differentiable forms) against the formulas
in float64, and against differences.

The bounds: a sum over a row has chains of at most K / 16 + 16 float32 additions, so a = (K / 16 + 16) 2^-24
of the sum of its terms' sizes; rstd is off by a + 2^-22 of it and, with a mean m off by a mean|x|, by what
that moves; a weight's gradient has chains of at most N additions."""
import pytest
import torch

from strim_amd import _native as N
from strim_amd import norm, ops
from test_scores_gpu import gen, pitched, within

pytestmark = pytest.mark.gpu


def rows(R, K, dtype, seed):
    g = gen(seed)
    x = torch.randn(R, K, device="cuda", generator=g) * (0.2 + 3.0 * torch.rand(R, 1, device="cuda", generator=g))
    x[:, ::17] *= 6.0
    return (x + 0.3).to(dtype)


def weights(K, dtype, seed):
    return (1.0 + 0.3 * torch.randn(K, device="cuda", generator=gen(seed))).to(dtype)


class Exact:
    def __init__(self, x, w, b, eps, center, dy=None):
        K = x.shape[1]
        a = (K / 16 + 16) * 2.0 ** -24
        xd = x.double()
        self.mean = xd.mean(1, keepdim=True) if center else torch.zeros_like(xd[:, :1])
        em = a * xd.abs().mean(1, keepdim=True) if center else 0.0
        c = xd - self.mean
        self.rstd = 1.0 / torch.sqrt((c * c).mean(1, keepdim=True) + eps)
        er = a + 2.0 ** -22 + (em * self.rstd) ** 2  # relative
        xh = c * self.rstd
        exh = xh.abs() * (er + 2.0 ** -23) + (em + 2.0 ** -24 * xd.abs()) * self.rstd
        wd = torch.ones_like(xd[0]) if w is None else w.double()
        bd = torch.zeros_like(wd) if b is None else b.double()
        half = torch.finfo(x.dtype).eps / 2
        self.y = xh * wd + bd
        ey = exh * wd.abs() + 2.0 ** -23 * (xh * wd).abs() + 2.0 ** -24 * self.y.abs()
        self.tol_y = ey + half * (self.y.abs() + ey) + 1e-37
        self.tol_rstd = (self.rstd * er)[:, 0] * 1.01
        self.tol_mean = (em + 2.0 ** -24 * self.mean.abs())[:, 0] if center else None
        if dy is None:
            return
        g = dy.double()
        h = g * wd
        m1, m2 = (h * xh).mean(1, keepdim=True), h.mean(1, keepdim=True)
        e1 = (h.abs() * exh + (a + 2.0 ** -22) * (h * xh).abs()).mean(1, keepdim=True)
        e2 = (a + 2.0 ** -23) * h.abs().mean(1, keepdim=True)
        inner = h - xh * m1 - (m2 if center else 0.0)
        size = h.abs() + (xh * m1).abs() + (m2.abs() if center else 0.0)
        ei = size * 2.0 ** -22 + exh * m1.abs() + xh.abs() * e1 + (e2 if center else 0.0)
        self.dx = self.rstd * inner
        ex = self.rstd * ei + self.dx.abs() * (er + 2.0 ** -23)
        self.tol_dx = ex + half * (self.dx.abs() + ex) + 1e-37
        wt = w.dtype if w is not None else b.dtype if b is not None else torch.float32
        half = torch.finfo(wt).eps / 2
        n = x.shape[0] * 2.0 ** -24
        self.dw, self.db = (g * xh).sum(0), g.sum(0)
        ew = (g.abs() * exh + (n + 2.0 ** -23) * (g * xh).abs()).sum(0)
        eb = n * g.abs().sum(0)
        self.tol_dw = ew + half * (self.dw.abs() + ew) + 1e-37
        self.tol_db = eb + half * (self.db.abs() + eb) + 1e-37


def check(x, w, b, center, dy, eps=1e-5, label=""):
    E = Exact(x, w, b, eps, center, dy)
    y, rstd, mean = ops.norm(x, w, b, eps, center)
    within(y, E.y, E.tol_y, f"{label} y")
    within(rstd, E.rstd[:, 0], E.tol_rstd, f"{label} rstd")
    assert (mean is None) == (not center)
    if center:
        within(mean, E.mean[:, 0], E.tol_mean, f"{label} mean")
    dx, dw, db = ops.norm_grad(x, w, b, dy, rstd, mean)
    within(dx, E.dx, E.tol_dx, f"{label} d_x")
    assert (dw is None) == (w is None) and (db is None) == (b is None)
    if w is not None:
        within(dw, E.dw, E.tol_dw, f"{label} d_weight")
    if b is not None:
        within(db, E.db, E.tol_db, f"{label} d_bias")
    # one at a time: the same bits
    only, none, none2 = ops.norm_grad(x, w, b, dy, rstd, mean, want_weight=False, want_bias=False)
    assert none is None and none2 is None and torch.equal(only, dx)
    if w is not None:
        none, only, _ = ops.norm_grad(x, w, b, dy, rstd, mean, want_x=False, want_bias=False)
        assert none is None and torch.equal(only, dw)
    if b is not None:
        none, none2, only = ops.norm_grad(x, w, b, dy, rstd, mean, want_x=False, want_weight=False)
        assert none is None and none2 is None and torch.equal(only, db)
    return y, rstd, mean, dx, dw, db


SIZES = [(1, 1), (3, 1), (1, 7), (2, 8), (5, 33), (17, 64), (64, 128), (1000, 128), (33, 130), (7, 1003),
         (1, 5120), (130, 1024), (300, 2051), (2049, 512), (40, 5120), (600, 5120), (9, 8192), (5, 9001),
         (3, 20_000), (2, 65_536), (70_000, 16), (1, 256), (4099, 72), (1030, 1000), (2500, 514), (1025, 2047),
         (513, 1500), (300, 6144), (30, 16_384), (30, 16_381), (800, 5120), (1600, 4100), (530, 8190), (530, 8192),
         (270, 9001), (530, 16_384), (9000, 200), (9001, 260)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("R,K", SIZES)
def test_norm(R, K, kind, dtype):
    print(f"[norm] N={R} K={K} {kind} {dtype}", flush=True)
    center = kind == "layer"
    x, dy = rows(R, K, dtype, seed=R + K), torch.randn(R, K, device="cuda", generator=gen(K)).to(dtype)
    check(x, weights(K, dtype, 1), weights(K, dtype, 2) if center else None, center, dy, label=f"N={R} K={K}")


@pytest.mark.parametrize("center", [False, True])
def test_weights_of_another_type_or_none(center):
    for dtype, wdtype in ((torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16)):
        x, dy = rows(70, 1_030, dtype, 3), torch.randn(70, 1_030, device="cuda", generator=gen(4)).to(dtype)
        w, b = weights(1_030, wdtype, 5), weights(1_030, wdtype, 6)
        check(x, w, b, center, dy)
        check(x, w, None, center, dy)
        check(x, None, b, center, dy)
        check(x, None, None, center, dy)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("pad,shift", [(3, 0), (8, 8), (1, 1)])
def test_strides_and_unaligned_rows(pad, shift, dtype):
    for R, K in ((5, 129), (200, 1_003), (40, 5_120), (3, 9_000)):
        print(f"[norm] pitch +{pad} shift {shift} N={R} K={K} {dtype}", flush=True)
        x, dy = rows(R, K, dtype, 7), torch.randn(R, K, device="cuda", generator=gen(8)).to(dtype)
        w = torch.cat([weights(1, dtype, 1), weights(K, dtype, 9)])[1:]  # (not aligned to more than its type)
        check(pitched(x, pad, shift), w, w, True, pitched(dy, pad + 5, shift + 3))
        check(pitched(x, pad, shift), w, None, False, dy)


def test_hard_rows():
    """Rows of zeros, of one value, of one large element, tiny and large ones; NaN and infinities stay in
    their rows (and reach the weights' gradients)."""
    K = 300
    x = rows(8, K, torch.float32, 11)
    x[0], x[1], x[2], x[3] = 0.0, 3.0, x[2] * 1e-18, x[3] * 1e15
    x[4] = 0.0
    x[4, 17] = 1e4
    dy = torch.randn(8, K, device="cuda", generator=gen(12))
    w, b = weights(K, torch.float32, 13), weights(K, torch.float32, 14)
    check(x, w, None, False, dy, eps=1e-6, label="rms")
    check(x[[0, 2, 4, 5, 6, 7]], w, b, True, dy[[0, 2, 4, 5, 6, 7]], label="layer")
    bad = x.clone()
    bad[5, 3], bad[6, 4] = float("nan"), float("inf")
    y, rstd, _ = ops.norm(bad, w)
    ref, rr, _ = ops.norm(x, w)
    keep = [0, 1, 2, 3, 4, 7]
    assert torch.equal(y[keep], ref[keep]) and bool(y[5].isnan().all())
    dx, dw, _ = ops.norm_grad(bad, w, None, dy, rstd)
    rx, _, _ = ops.norm_grad(x, w, None, dy, rr)
    assert torch.equal(dx[keep], rx[keep]) and bool(dx[5].isnan().all()) and bool(dw[3].isnan())
    assert float(rstd[6]) == 0.0


def test_no_rows():
    w = weights(40, torch.bfloat16, 1)
    x = torch.empty(0, 40, dtype=torch.bfloat16, device="cuda")
    y, rstd, _ = ops.norm(x, w)
    dx, dw, db = ops.norm_grad(x, w, w, x, rstd)
    assert y.shape == (0, 40) and dx.shape == (0, 40) and bool((dw == 0).all()) and bool((db == 0).all())


def test_differences():
    """Gradients along directions against differences of sum y g: steps of 1/64 on a grid of 1/32. The third
    derivative of a normalised row along a unit step is below 30 rstd^3 |g| |w|; y is off by 1e-6."""
    R, K = 12, 200
    x = (torch.randn(R, K, device="cuda", generator=gen(20)) * 64).round() / 32
    g = torch.randn(R, K, device="cuda", generator=gen(21))
    w, b = weights(K, torch.float32, 22), weights(K, torch.float32, 23)
    for center in (False, True):
        _, rstd, mean = ops.norm(x, w, b, 1e-5, center)
        dx, dw, db = ops.norm_grad(x, w, b, g, rstd, mean)
        for s in range(4):
            d = torch.where(torch.rand(R, K, device="cuda", generator=gen(30 + s)) < 0.5, -1.0, 1.0)
            d *= torch.rand(R, K, device="cuda", generator=gen(40 + s)) < 0.1
            f = lambda h: (ops.norm(x + h * d, w, b, 1e-5, center)[0].double() * g).sum(1)
            diff, lin = (f(1 / 64) - f(-1 / 64)) * 32, (dx.double() * d).sum(1)
            step = d.double().norm(dim=1) / 64
            tol = 64 * 1e-6 * g.double().abs().sum(1) + 30 * 64 * (rstd.double() * step) ** 3 * (g * w).double().norm(dim=1)
            assert bool(((diff - lin).abs() <= tol).all())
        # linear in the weights
        f = lambda k: (ops.norm(x, w + k, b + k, 1e-5, center)[0].double() * g).sum()
        want = float((dw + db).double().sum())
        assert abs(float(f(0.5) - f(-0.5)) - want) <= 1e-6 * float((g.abs() * 4).double().sum()) * K ** 0.5


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_autograd(dtype):
    x = rows(60, 136, dtype, 31).reshape(3, 20, 136)
    w, b = weights(136, dtype, 32), weights(136, dtype, 33)
    for center in (False, True):
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        y = norm.layer_norm(*leaves) if center else norm.rms_norm(*leaves[:2], eps=1e-5)
        assert y.shape == x.shape and y.dtype == dtype
        y.sum().backward()  # (a broadcast gradient)
        E = Exact(x.reshape(60, 136), w, b if center else None, 1e-5, center, torch.ones(60, 136, device="cuda", dtype=dtype))
        within(leaves[0].grad.reshape(60, 136), E.dx, E.tol_dx, "d_x")
        within(leaves[1].grad, E.dw, E.tol_dw, "d_weight")
        if center:
            within(leaves[2].grad, E.db, E.tol_db, "d_bias")
        # frozen weights, no weights, rows that are not contiguous, a transposed gradient
        leaf = x.transpose(1, 2).contiguous().transpose(1, 2).detach().requires_grad_()
        g = torch.randn(3, 136, 20, device="cuda", generator=gen(35)).to(dtype).transpose(1, 2)
        y = norm.layer_norm(leaf, w, b) if center else norm.rms_norm(leaf, w, eps=1e-5)
        y.backward(g)
        E = Exact(x.reshape(60, 136), w, b if center else None, 1e-5, center, g.reshape(60, 136))
        within(leaf.grad.reshape(60, 136), E.dx, E.tol_dx, "d_x")
    (d,) = torch.autograd.grad(norm.rms_norm(leaf).float().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        d.float().square().sum().backward()


def test_as_the_projection_normalises():
    """rms_norm beside the norm in front of the projection (which rounds once more: the normalised row, then
    its product with the weight)."""
    x, w = rows(8, 512, torch.bfloat16, 41), weights(512, torch.bfloat16, 42)
    xn = torch.empty_like(x)
    ops.head_logits(x, torch.zeros(64, 512, dtype=torch.bfloat16, device="cuda"), norm_weight=w, xn=xn)
    y = ops.norm(x, w)[0]
    assert float(((xn.double() - y.double()).abs() - 2.0 ** -6 * y.double().abs()).max()) <= 0


def test_repeatable_streams_and_graphs():
    for R, K in ((700, 1_024), (3, 5_120)):
        x, x2 = rows(R, K, torch.bfloat16, 51), rows(R, K, torch.bfloat16, 52)
        dy = torch.randn(R, K, device="cuda", generator=gen(53)).to(torch.bfloat16)
        w, b = weights(K, torch.bfloat16, 54), weights(K, torch.bfloat16, 55)

        def run(**kw):
            y, rstd, mean = ops.norm(x, w, b, center=True, **kw)
            return [y, rstd, mean, *ops.norm_grad(x, w, b, dy, rstd, mean, **kw)]

        ref = run()
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        got = run(stream=stream)
        torch.cuda.current_stream().wait_stream(stream)
        for a, c in zip(got, ref):
            assert torch.equal(a, c)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = run()
        keep = x.clone()
        for src in (x2, keep, x2):
            x.copy_(src)
            ref = run()
            graph.replay()
            torch.cuda.synchronize()
            for a, c in zip(res, ref):
                assert torch.equal(a, c)


def test_refusals():
    x, w = rows(4, 64, torch.bfloat16, 1), weights(64, torch.bfloat16, 2)
    y, rstd, _ = ops.norm(x, w)
    bad = [lambda: ops.norm(x.T, w[:4]), lambda: ops.norm(x, w[:63]), lambda: ops.norm(x, w, eps=-1.0),
           lambda: ops.norm(x, w, eps=float("nan")), lambda: ops.norm(x.cpu(), w), lambda: ops.norm(x, w.cpu()),
           lambda: ops.norm(x, w, w.float()), lambda: ops.norm(x[0], w),
           lambda: ops.norm(torch.zeros(1, 65_537, device="cuda")), lambda: ops.norm(x[:, :0]),
           lambda: ops.norm_grad(x, w, None, y.float(), rstd), lambda: ops.norm_grad(x, w, None, y[:3], rstd),
           lambda: ops.norm_grad(x, w, None, y, rstd[:3]), lambda: ops.norm_grad(x, w, None, y.T.contiguous().T, rstd)]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        ops.norm(x.half(), w)


def test_past_32_bits():
    """Rows that begin past 2^31 elements: the same bits as of their copies."""
    print("[norm] rows past 2^31 elements", flush=True)
    R, K, stride = 5, 1_030, 600_000_001
    buf = torch.empty((R - 1) * stride + K, dtype=torch.bfloat16, device="cuda")
    x = buf.as_strided((R, K), (stride, 1))
    x.copy_(rows(R, K, torch.bfloat16, 1))
    dy, w = rows(R, K, torch.bfloat16, 2), weights(K, torch.bfloat16, 3)
    y, rstd, mean = ops.norm(x, w, w, center=True)
    got = [y, rstd, mean, *ops.norm_grad(x, w, w, dy, rstd, mean)]
    c = x.contiguous()
    y, rstd, mean = ops.norm(c, w, w, center=True)
    for a, b in zip(got, [y, rstd, mean, *ops.norm_grad(c, w, w, dy, rstd, mean)]):
        assert torch.equal(a, b)
