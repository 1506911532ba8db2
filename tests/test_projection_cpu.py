"""Host-side checks of the projection's operators: arguments that no launch should see are
refused before one, and the sizes of workspaces."""
import ctypes

import pytest

from strim_amd import _native as N

P = ctypes.c_void_p(1 << 20)  # never read: every call below is refused, or has nothing to launch


def loss(**kw):
    a = dict(h=P, hs=64, R=4, K=64, w=P, ws=64, V=100, t=P, wsp=P, wb=1 << 40, out=P)
    a.update(kw)
    return N.lib().strim_head_loss(None, a["h"], a["hs"], a["R"], a["K"], a["w"], a["ws"], a["V"],
                                   a["t"], -100, a["wsp"], a["wb"], a["out"], None, None)


def grad(**kw):
    a = dict(h=P, hs=64, R=4, K=64, w=P, ws=64, V=100, t=P, lse=P, gl=P, wsp=P, wb=1 << 40, dh=P,
             dhs=64, dw=P, dws=64)
    a.update(kw)
    return N.lib().strim_head_loss_grad(None, a["h"], a["hs"], a["R"], a["K"], a["w"], a["ws"],
                                        a["V"], a["t"], -100, a["lse"], a["gl"], None, a["wsp"],
                                        a["wb"], a["dh"], a["dhs"], a["dw"], a["dws"])


@pytest.mark.parametrize("bad", [
    dict(h=None), dict(w=None), dict(t=None), dict(wsp=None), dict(out=None), dict(R=-1),
    dict(R=N.LOSS_MAX_ROWS + 1), dict(K=0), dict(K=60), dict(K=N.LOSS_MAX_STRIDE + 8), dict(V=0),
    dict(V=N.LOSS_MAX_STRIDE + 1), dict(hs=56), dict(hs=68), dict(ws=56),
    dict(ws=N.LOSS_MAX_STRIDE + 8), dict(h=ctypes.c_void_p((1 << 20) + 8)),
    dict(w=ctypes.c_void_p((1 << 20) + 2)), dict(wsp=ctypes.c_void_p((1 << 20) + 4))])
def test_loss_refuses(bad):
    assert loss(**bad) == N.EINVAL


@pytest.mark.parametrize("bad", [
    dict(h=None), dict(lse=None), dict(gl=None), dict(t=None), dict(wsp=None),
    dict(dh=None, dw=None), dict(dhs=56), dict(dws=60), dict(dh=ctypes.c_void_p((1 << 20) + 8)),
    dict(K=12), dict(V=-1)])
def test_loss_grad_refuses(bad):
    assert grad(**bad) == N.EINVAL


def test_loss_workspaces():
    f = N.lib().strim_head_loss_workspace
    assert loss(wb=8) == N.ECAPACITY and grad(wb=8) == N.ECAPACITY
    assert loss(R=0, h=None, t=None, wsp=None, out=None) == N.OK
    assert f(0, 64, 100, 1, 1) == 0 and f(4, 60, 100, 1, 1) == N.EINVAL
    # p in pieces: far less than the logits, however long the batch
    R, K, V = 16_384, 5_120, 151_936
    assert f(R, K, V, 1, 1) < R * V
    # the loss alone: a pair of float32 for 128 of the vocabulary, and the targets' logits
    assert f(R, K, V, 0, 0) <= R * (-(-V // 256) * 2 * 8 + 4) + 512
    assert f(R, K, V, 0, 0) < f(R, K, V, 1, 0) <= f(R, K, V, 1, 1)


def test_packed_refuses():
    def logits(**kw):
        a = dict(h=P, hs=256, B=2, K=256, nw=None, xn=None, w=P, wst=32, s=P, ss=4, g=64, V=20, wsp=P,
                 wb=1 << 30, out=P, dt=N.DTYPE_BF16, os=20)
        a.update(kw)
        return N.lib().strim_head_logits_packed(
            None, a["h"], a["hs"], a["B"], a["K"], a["nw"], 1e-6, a["xn"], a["w"], a["wst"], a["s"],
            None, a["ss"], a["g"], a["V"], a["wsp"], a["wb"], a["out"], a["dt"], a["os"])

    for bad in (dict(h=None), dict(w=None), dict(s=None), dict(out=None), dict(wsp=None), dict(B=0),
                dict(K=0), dict(K=224), dict(g=48), dict(V=0), dict(V=(1 << 24) + 1), dict(hs=248),
                dict(hs=260), dict(wst=28), dict(wst=34), dict(ss=3), dict(os=19), dict(dt=2),
                dict(nw=P), dict(w=ctypes.c_void_p((1 << 20) + 4))):
        assert logits(**bad) == N.EINVAL, bad
    assert logits(wb=16) == N.ECAPACITY
    f = N.lib().strim_head_logits_packed_workspace
    assert f(1, 5_120) == 0 and f(8, 5_120) == 0 and f(9, 5_120) > 0 and f(1, 512) > 0
    assert f(0, 64) == N.EINVAL and f(1, 0) == N.EINVAL
    pack = N.lib().strim_pack_weights
    assert pack(None, P, N.DTYPE_BF16, 64, 4, 64, 16, P, P, None) == N.EINVAL
    assert pack(None, P, 5, 64, 4, 64, 64, P, P, None) == N.EINVAL
    assert pack(None, P, N.DTYPE_F32, 66, 4, 64, 64, P, P, None) == N.EINVAL
    assert pack(None, P, N.DTYPE_BF16, 64, 0, 64, 64, P, P, None) == N.EINVAL
    assert pack(None, P, N.DTYPE_BF16, 64, 4, 64, 64, P, None, None) == N.EINVAL
    unpack = N.lib().strim_unpack_weights
    assert unpack(None, P, 7, P, None, 1, 4, 64, 64, P, N.DTYPE_BF16, 64) == N.EINVAL
    assert unpack(None, P, 8, P, None, 0, 4, 64, 64, P, N.DTYPE_BF16, 64) == N.EINVAL
    assert unpack(None, P, 8, P, None, 1, 4, 64, 64, P, N.DTYPE_F32, 66) == N.EINVAL
