"""Temperatures that the scores and the distillation refuse, at their C entries, before any launch."""
import ctypes

import pytest

from strim_amd import _native as N
from test_scores_cpu import distill, distill_grad, scores, scores_grad, step

LEAST = 2.0 ** -126


@pytest.mark.parametrize("T", [LEAST / 2, 1e-39, 1e-45, 0.0, -1e-39])
def test_without_a_reciprocal(T):
    """log2(e) / T of a temperature below float32's normal numbers is infinite, and every product with it."""
    for call in (scores, scores_grad):
        assert call(T=T) == N.EINVAL
    for call in (distill, distill_grad, step):
        assert call(T=T) == N.EINVAL


def test_the_least():
    assert scores(T=LEAST, R=0) == scores_grad(T=LEAST, R=0) == N.OK
    assert distill(T=LEAST, N=0) == distill_grad(T=LEAST, N=0) == step(T=LEAST, N=0) == N.OK
    assert ctypes.c_float(LEAST).value == LEAST
