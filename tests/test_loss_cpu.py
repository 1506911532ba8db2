"""The differentiable loss's own logic, without a GPU: the formulas in plain torch stand in for the
device calls."""
import pytest
import torch

from strim_amd import loss as L
from strim_amd import ops


@pytest.fixture
def calls(monkeypatch):
    """head_loss and head_loss_grad by their formulas; the arguments of each gradient call."""
    seen = []

    def rows(h, w, t, ignore_index):
        live = (t != ignore_index) & (t >= 0) & (t < w.shape[0])
        return h.float() @ w.float().T, live, torch.where(live, t, 0).long()[:, None]

    def head_loss(h, w, t, ignore_index=-100):
        x, live, at = rows(h, w, t, ignore_index)
        lse = torch.logsumexp(x, 1)
        return torch.where(live, lse - x.gather(1, at)[:, 0], 0.0), lse, torch.zeros_like(t)

    def head_loss_grad(h, w, t, lse, gl, gz=None, want_hidden=True, want_lm_head=True, ignore_index=-100):
        seen.append(dict(grad_loss=gl, grad_lse=gz, want_hidden=want_hidden, want_lm_head=want_lm_head))
        x, live, at = rows(h, w, t, ignore_index)
        p = torch.exp(x - lse[:, None]) * (gl if gz is None else gl + gz)[:, None]
        p.scatter_add_(1, at, -gl[:, None])
        p = torch.where(live[:, None], p, 0.0)
        return ((p @ w.float()).to(h.dtype) if want_hidden else None,
                (p.T @ h.float()).to(w.dtype) if want_lm_head else None)

    monkeypatch.setattr(L.ops, "head_loss", head_loss)
    monkeypatch.setattr(L.ops, "head_loss_grad", head_loss_grad)
    return seen


def inputs(R=6, K=8, V=20):
    g = torch.Generator().manual_seed(0)
    h, w = torch.randn(R, K, generator=g), torch.randn(V, K, generator=g)
    return h.requires_grad_(), w.requires_grad_(), torch.randint(0, V, (R,), generator=g)


def test_second_derivatives_raise(calls):
    """A gradient penalty on the loss is refused: it would add nothing."""
    h, w, t = inputs()
    (dh,) = torch.autograd.grad(L.head_cross_entropy(h, w, t), h, create_graph=True)
    with pytest.raises(RuntimeError):
        dh.square().sum().backward()
    # first derivatives are what they were
    ref = torch.autograd.grad(torch.nn.functional.cross_entropy(h @ w.T, t), (h, w))
    got = torch.autograd.grad(L.head_cross_entropy(h, w, t), (h, w))
    for a, b in zip(got, ref):
        assert torch.allclose(a, b, rtol=1e-4, atol=1e-6)


def test_an_unused_output_takes_no_gradient(calls):
    """A plain loss hands no gradient of the log-sum-exp to the device (not zeros), and the
    log-sum-exp alone has zeros for the loss; frozen inputs are not asked for."""
    h, w, t = inputs()
    L.head_cross_entropy(h, w, t).backward()
    assert calls[-1]["grad_lse"] is None and calls[-1]["want_hidden"] and calls[-1]["want_lm_head"]
    L.head_loss(h, w.detach(), t)[1].sum().backward()
    assert bool((calls[-1]["grad_loss"] == 0).all()) and bool((calls[-1]["grad_lse"] == 1).all())
    assert calls[-1]["want_hidden"] and not calls[-1]["want_lm_head"]
    loss, lse, _ = L.head_loss(h.detach(), w, t)
    (2 * loss.sum() + 3 * lse.sum()).backward()
    assert bool((calls[-1]["grad_loss"] == 2).all()) and bool((calls[-1]["grad_lse"] == 3).all())
    assert not calls[-1]["want_hidden"] and calls[-1]["want_lm_head"]


@pytest.mark.parametrize("ignore", [2 ** 31, -2 ** 31 - 1, 2 ** 40])
def test_ignore_index_past_32_bits_is_refused(calls, ignore):
    """It would be cut to 32 bits, 2^40 to token 0."""
    h, w, t = inputs()
    for ids in (t, t.int()):
        with pytest.raises(ValueError, match="ignore_index"):
            L.head_loss(h, w, ids, ignore_index=ignore)
        with pytest.raises(ValueError, match="ignore_index"):
            L.head_cross_entropy(h, w, ids, ignore_index=ignore)


@pytest.mark.parametrize("ignore", [2 ** 31, -2 ** 31 - 1])
def test_device_calls_refuse_it_too(ignore):
    h, w, t = inputs()
    with pytest.raises(ValueError, match="ignore_index"):
        ops.head_loss(h, w, t, ignore)
    with pytest.raises(ValueError, match="ignore_index"):
        ops.head_loss_grad(h, w, t, t, t, ignore_index=ignore)


@pytest.mark.parametrize("ignore", [-100, 20, 21, -1, 7, 2 ** 31 - 1, -2 ** 31])
def test_ids_outside_the_vocabulary_stay_outside(ignore):
    """Whatever the ignored id is, and however large the others are: ids of the vocabulary as they
    are, the ignored id as it is, any other id neither."""
    V = 20
    t = torch.tensor([0, 5, 19, 20, 21, 25, -1, -7, 2 ** 40, 2 ** 40 + 5, -2 ** 40, 2 ** 32 + 7, ignore])
    got = L._ids(t, V, ignore).long()
    inside = (t >= 0) & (t < V)
    assert torch.equal(got[inside], t[inside]) and torch.equal(got == ignore, t == ignore)
    outside = ~inside & (t != ignore)
    assert bool(((got < 0) | (got >= V))[outside].all())
