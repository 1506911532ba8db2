"""The scores', distillation's and norms' own logic without a GPU: what the C entries refuse before any
launch, their workspaces, and the differentiable forms with plain torch in the device calls' place."""
import ctypes

import pytest
import torch

from strim_amd import _native as N
from strim_amd import loss as L
from strim_amd import norm, ops

P = ctypes.c_void_p(4096)  # (never read: every call here is refused, or has no rows)
ODD = ctypes.c_void_p(4097)
BIG = 1 << 40


def scores(**kw):
    a = dict(logits=P, dtype=1, R=2, V=100, stride=100, T=1.0, mask=None, mask_stride=0, tokens=P, S=1,
             ignore=-100, top=3, ws=P, wsb=BIG, lp=P, H=P, lse=P, ids=P, ilp=P, status=None)
    a.update(kw)
    return N.lib().strim_token_scores(None, *a.values())


def scores_grad(**kw):
    a = dict(logits=P, dtype=1, R=2, V=100, stride=100, T=1.0, mask=None, mask_stride=0, tokens=P, S=1,
             ignore=-100, lse=P, H=P, g=P, gh=P, gl=None, d=P, d_stride=100)
    a.update(kw)
    return N.lib().strim_token_scores_grad(None, *a.values())


ROWS = [dict(dtype=2), dict(R=-1), dict(R=(1 << 22) + 1), dict(V=0), dict(V=(1 << 20) + 1, stride=1 << 21),
        dict(stride=99), dict(T=0.0), dict(T=-1.0), dict(T=float("inf")), dict(T=float("nan")),
        dict(logits=None), dict(logits=ODD), dict(logits=ctypes.c_void_p(4098), dtype=0)]


@pytest.mark.parametrize("bad", ROWS + [
    dict(tokens=None), dict(S=-1), dict(S=129), dict(top=-1), dict(top=129), dict(lp=None), dict(H=None),
    dict(lse=None), dict(ids=None), dict(ilp=None), dict(mask=P, mask_stride=3)])
def test_scores_refuse(bad):
    assert scores(**bad) == N.EINVAL


@pytest.mark.parametrize("bad", ROWS + [
    dict(tokens=None), dict(S=129), dict(lse=None), dict(H=None), dict(d=None), dict(d=ODD), dict(d_stride=99),
    dict(mask=P, mask_stride=3)])
def test_scores_grad_refuses(bad):
    assert scores_grad(**bad) == N.EINVAL


def test_no_rows_is_no_call():
    assert scores(R=0, logits=None, tokens=None, lp=None, H=None, lse=None, ids=None, ilp=None) == N.OK
    assert scores_grad(R=0, logits=None, tokens=None, lse=None, d=None) == N.OK
    assert distill(N=0, logits=None, ids=None, lps=None, loss=None) == N.OK
    assert step(N=0, logits=None, ids=None, lps=None, w=None, loss=None, d=None) == N.OK
    assert normed(N=0, x=None, y=None) == N.OK
    assert N.lib().strim_distill_scale(None, None, 1, 0, None) == N.OK


def distill(**kw):
    a = dict(logits=P, dtype=1, N=2, V=100, stride=100, T=1.0, ids=P, lps=P, M=4, tail=0, ws=P, wsb=BIG,
             loss=P, lse=None, rest=None, status=None)
    a.update(kw)
    return N.lib().strim_distill(None, *a.values())


def distill_grad(**kw):
    a = dict(logits=P, dtype=1, N=2, V=100, stride=100, T=1.0, ids=P, lps=P, M=4, tail=1, lse=P, rest=P, g=P,
             d=P, d_stride=100)
    a.update(kw)
    return N.lib().strim_distill_grad(None, *a.values())


def step(**kw):
    a = dict(logits=P, dtype=1, N=2, V=100, stride=100, T=1.0, ids=P, lps=P, M=4, tail=0, w=P, ws=P, wsb=BIG,
             loss=P, d=P, d_stride=100, status=None)
    a.update(kw)
    return N.lib().strim_distill_step(None, *a.values())


@pytest.mark.parametrize("bad", [{("N" if k == "R" else k): v for k, v in r.items()} for r in ROWS] + [
    dict(ids=None), dict(lps=None), dict(M=0), dict(M=129)])
def test_distillation_refuses(bad):
    assert distill(**bad) == distill_grad(**bad) == step(**bad) == N.EINVAL


def test_distillation_refuses_what_is_its_own():
    assert distill(loss=None) == step(loss=None) == step(w=None) == step(d=None) == step(d_stride=99) == N.EINVAL
    for bad in (dict(lse=None), dict(rest=None), dict(g=None), dict(d=None), dict(d=ODD), dict(d_stride=99)):
        assert distill_grad(**bad) == N.EINVAL
    scale = N.lib().strim_distill_scale
    assert scale(None, None, 1, 4, P) == scale(None, P, 1, 4, None) == scale(None, P, 1, -1, P) == N.EINVAL
    assert scale(None, ODD, 1, 4, P) == scale(None, P, 3, 4, P) == N.EINVAL


def normed(**kw):
    a = dict(x=P, dtype=1, N=2, K=64, stride=64, w=P, b=None, wdtype=1, eps=1e-6, center=0, y=P, y_stride=64,
             rstd=P, mean=None)
    a.update(kw)
    return N.lib().strim_norm(None, *a.values())


def norm_grad(**kw):
    a = dict(x=P, dtype=1, N=2, K=64, stride=64, g=P, g_stride=64, w=P, wdtype=1, rstd=P, mean=None, ws=P,
             wsb=BIG, dx=P, dx_stride=64, dw=P, db=P)
    a.update(kw)
    return N.lib().strim_norm_grad(None, *a.values())


NORM = [dict(dtype=2), dict(wdtype=-1), dict(N=-1), dict(N=(1 << 28) + 1), dict(K=0), dict(K=(1 << 16) + 1, stride=1 << 17),
        dict(stride=63), dict(x=None), dict(x=ODD), dict(w=ODD)]


@pytest.mark.parametrize("bad", NORM + [dict(eps=-1.0), dict(eps=float("nan")), dict(y=None), dict(y=ODD),
                                        dict(y_stride=63), dict(b=ODD), dict(center=1, mean=None)])
def test_norm_refuses(bad):
    assert normed(**bad) == N.EINVAL


@pytest.mark.parametrize("bad", NORM + [dict(g=None), dict(g=ODD), dict(g_stride=63), dict(rstd=None),
                                        dict(dx=ODD), dict(dx_stride=63), dict(dw=ODD), dict(db=ODD)])
def test_norm_grad_refuses(bad):
    assert norm_grad(**bad) == N.EINVAL


def test_workspaces():
    """Sizes that the calls need: none without rows, refused where the call is, and a call that has less."""
    L_ = N.lib()
    assert ops.token_scores_workspace(0, 100, 5) == ops.distill_workspace(0, 100, 5) == ops.norm_workspace(0, 8, True) == 0
    for bad in ((-1, 100, 5), (1, 0, 5), (1, 100, 129), (1, (1 << 20) + 1, 5)):
        assert L_.strim_token_scores_workspace(*bad) == N.EINVAL
        with pytest.raises(N.StrimError):
            ops.token_scores_workspace(*bad)
    assert L_.strim_distill_workspace(1, 100, 0, 0) == L_.strim_norm_workspace(1, 0, 1, 1) == N.EINVAL
    for R, V, top in ((1, 151_936, 20), (64, 151_936, 128), (2048, 32_768, 5), (1 << 22, 1 << 20, 128)):
        need = ops.token_scores_workspace(R, V, top)
        assert need >= 0
        if need:
            a = dict(R=R, V=V, stride=V, top=top)
            assert scores(**a, wsb=need - 1) == N.ECAPACITY
            assert scores(**a, ws=None) == scores(**a, ws=ctypes.c_void_p(4100)) == N.EINVAL
        for st in (False, True):
            need = ops.distill_workspace(R, V, max(1, top), st)
            if need:
                a = dict(N=R, V=V, stride=V, M=max(1, top), wsb=need - 1)
                assert (step(**a, d_stride=V) if st else distill(**a)) == N.ECAPACITY
    for R, K in ((1, 1), (5000, 5120), (1 << 28, 64)):
        need = ops.norm_workspace(R, K, True, True)
        if need:
            assert norm_grad(N=R, K=K, stride=K, g_stride=K, dx_stride=K, wsb=need - 1) == N.ECAPACITY


def test_device_calls_refuse_host_tensors():
    x, t = torch.zeros(2, 8), torch.zeros(2, dtype=torch.int32)
    for call in (lambda: ops.token_scores(x, t), lambda: ops.token_scores_grad(x, t, x[:, 0]),
                 lambda: ops.distill(x, t[:, None], x[:, :1]), lambda: ops.norm(x), lambda: ops.distill_scale(x, x[0, :1]),
                 lambda: ops.distill_step(x, t[:, None], x[:, :1], x[:, 0])):
        with pytest.raises(ValueError, match="on the GPU"):
            call()


# ---- the differentiable forms ---------------------------------------------------------------
@pytest.fixture
def plain(monkeypatch):
    """The device calls by their formulas; what each gradient call was asked."""
    seen = []

    def token_scores(x, t, top=0, T=1.0, mask=None, ignore=-100):
        lp = torch.log_softmax(x / T, 1)
        tok = None if t is None else lp.gather(1, t.long().reshape(len(x), -1)).reshape(t.shape)
        ids = lp.topk(top, 1).indices.int() if top else None
        return ops.TokenScores(tok, -(lp.exp() * lp).sum(1), torch.logsumexp(x / T, 1), ids,
                               lp.gather(1, ids.long()) if top else None, torch.zeros(len(x), dtype=torch.int32))

    def token_scores_grad(x, t, lse, H, g=None, gh=None, gl=None, temperature=1.0, mask=None, ignore_index=-100):
        seen.append((g, gh, gl))
        leaf = x.detach().requires_grad_()
        with torch.enable_grad():
            out = token_scores(leaf, t, 0, temperature)
            total = sum((a * b).sum() for a, b in zip(out[:3], (g, gh, gl)) if b is not None)
        return torch.autograd.grad(total, leaf)[0]

    def distill(x, ids, lp, T=1.0, tail=False):
        lq = torch.log_softmax(x / T, 1)
        p = torch.softmax(lp, 1)
        loss = (p * (p.log() - lq.gather(1, ids.long()))).sum(1)
        return loss, loss, loss, torch.zeros(len(x), dtype=torch.int32)

    def distill_grad(x, ids, lp, lse, rest, g, T=1.0, tail=False):
        leaf = x.detach().requires_grad_()
        with torch.enable_grad():
            total = (distill(leaf, ids, lp, T, tail)[0] * g).sum()
        return torch.autograd.grad(total, leaf)[0]

    def distill_step(x, ids, lp, w, T=1.0, tail=False):
        seen.append("step")
        loss, lse, rest, st = distill(x.detach(), ids, lp, T, tail)
        return loss, distill_grad(x, ids, lp, lse, rest, w, T, tail), st

    for f in (token_scores, token_scores_grad, distill, distill_grad, distill_step):
        monkeypatch.setattr(L.ops, f.__name__, f)
    monkeypatch.setattr(L.ops, "distill_scale", lambda d, f: d.mul_(f))
    return seen


def test_unused_outputs_take_no_gradient(plain):
    x = torch.randn(6, 20, generator=torch.Generator().manual_seed(0)).requires_grad_()
    t = torch.arange(6)
    L.token_scores(x, t).logprobs.sum().backward()
    assert plain[-1][0] is not None and plain[-1][1] is None and plain[-1][2] is None
    L.token_scores(x, t, top=2).entropy.mean().backward()
    assert plain[-1][0] is None and plain[-1][1].is_contiguous() and plain[-1][2] is None
    with pytest.raises(ValueError):
        L.token_scores(x, t[:5])
    with pytest.raises(TypeError):
        L.token_scores(x, t.float())
    with pytest.raises(ValueError):
        L.token_scores(x, t, mask=torch.zeros(5, 1, dtype=torch.int32))


def test_a_mean_takes_one_step_and_survives_a_second_pass(plain):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(5, 30, generator=g).requires_grad_()
    ids, lp = torch.arange(20).reshape(5, 4), torch.randn(5, 4, generator=g)
    value = L.distill_loss(x, ids, lp)
    assert plain == ["step"]
    value.backward(retain_graph=True)
    assert plain == ["step"]
    first, x.grad = x.grad, None
    kept = first.clone()
    (value * 3).backward()
    assert plain == ["step", "step"] and torch.allclose(x.grad, 3 * kept) and torch.equal(first, kept)
    ref = torch.autograd.grad(L.ops.distill(x, ids, lp)[0].mean(), x)[0]
    assert torch.allclose(kept, ref, rtol=1e-5, atol=1e-7)
    # nothing to train: the loss alone
    plain.clear()
    L.distill_loss(x.detach(), ids, lp)
    assert plain == []
    # rows without alternatives are not counted, infinite ones of weight 0 neither
    ids2 = ids.clone()
    ids2[0] = 2 ** 40
    with pytest.raises(TypeError):
        L.distill_loss(x, ids.float(), lp)
    live = L._alternatives(x, ids2, lp)[0]
    assert live.dtype == torch.int32 and bool((live[0] == 30).all())


def test_norms_refuse_second_derivatives(monkeypatch):
    def fwd(x, w, b, eps, center):
        mean = x.mean(1) if center else None
        c = x - (mean[:, None] if center else 0.0)
        rstd = torch.rsqrt((c * c).mean(1) + eps)
        y = c * rstd[:, None] * (1.0 if w is None else w)
        return (y if b is None else y + b), rstd, mean

    def bwd(x, w, b, g, rstd, mean, want_x=True, want_weight=True, want_bias=True):
        assert g.is_contiguous()
        leaves = [None if t is None else t.detach().requires_grad_() for t in (x, w, b)]
        with torch.enable_grad():
            y = fwd(*leaves, 1e-5, mean is not None)[0]
        grads = iter(torch.autograd.grad(y, [t for t in leaves if t is not None], g))
        out = [None if t is None else next(grads) for t in leaves]
        return tuple(o if k else None for o, k in zip(out, (want_x, want_weight, want_bias)))

    monkeypatch.setattr(norm.ops, "norm", fwd)
    monkeypatch.setattr(norm.ops, "norm_grad", bwd)
    x, w = torch.randn(2, 3, 8).requires_grad_(), torch.ones(8, requires_grad=True)
    norm.rms_norm(x, w, eps=1e-5).sum().backward()
    assert x.grad.shape == x.shape and w.grad.shape == (8,)
    y = norm.layer_norm(x, w, w * 0.5)
    ref = torch.nn.functional.layer_norm(x, (8,), w, w * 0.5)
    assert torch.allclose(y, ref, atol=1e-5)
    (d,) = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()
