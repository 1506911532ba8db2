"""The differentiable distillation without a GPU: what is made where no gradient is wanted, and what is
refused; plain torch stands in the device calls' place."""
import pytest
import torch

from strim_amd import loss as L
from test_scores_cpu import plain  # noqa: F401  (a fixture)


def rows():
    g = torch.Generator().manual_seed(1)
    return torch.randn(5, 30, generator=g).requires_grad_(), torch.arange(20).reshape(5, 4), torch.randn(5, 4, generator=g)


@pytest.mark.parametrize("reduction", ["mean", "sum"])
@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
def test_no_gradient_is_made_where_none_is_recorded(plain, mode, reduction):  # noqa: F811
    """Logits of a trained head in an evaluation: the loss alone, no pass that writes a gradient."""
    x, ids, lp = rows()
    with mode():
        value = L.distill_loss(x, ids, lp, reduction=reduction)
    assert plain == [] and not value.requires_grad
    again = L.distill_loss(x, ids, lp, reduction=reduction)
    assert plain == ["step"] and torch.equal(again.detach(), value.clone())
    again.backward()
    assert x.grad is not None


def test_nothing_to_lay_out_is_refused_by_the_call_itself():
    """Empty vocabularies, lists and widths get the calls' own errors, with and without rows."""
    from strim_amd import norm

    for lead in ((3,), (2, 3), (0,), ()):
        none = torch.empty(*lead, 0)
        for call in (lambda: L.token_scores(none), lambda: L.distill_loss(none, none.int(), none),
                     lambda: L.distill_loss(torch.zeros(*lead, 8), none.int(), none),
                     lambda: L.distill_loss(torch.zeros(*lead, 8), none.int(), none, reduction="none"),
                     lambda: norm.rms_norm(none)):
            with pytest.raises(ValueError):
                call()
