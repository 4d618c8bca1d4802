"""The loss of distillation on the GPU where its terms need the 64 bits that they are computed in: probabilities smaller than 32
bits hold, and losses of hundreds.  The loss alone and the call that also gives the gradient agree on it."""
import numpy as np
import pytest

from gpu_util import F32
from test_gpu_class_rows import TYPES, check_distill, logits, rounded, slots

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("mode", ["fused", "apart"])
@pytest.mark.parametrize("n,rows", [(100, 8), (900, 8), (1700, 8), (5000, 8), (12000, 8), (30000, 8), (70001, 8), (140000, 40)])
def test_classes_that_the_student_rules_out(kind, mode, n, rows):
    g = np.random.default_rng(n)
    x = logits(g, rows, n, kind)
    index = np.broadcast_to(np.array([3, n // 2, n - 1, 7], np.uint32), (rows, 4)).copy()
    value = np.broadcast_to(np.array([2.0, 1.0, 0.5, 0.25], F32), (rows, 4)).copy()
    for r, low in enumerate((-60.0, -95.0, -110.0, -300.0, -735.0, -800.0, -3e38)):
        value[r, 2] = low                       # e^-95 is a denormal of 32 bits, e^-110 none, e^-800 none of 64 either
        x[r, n - 1] = -np.inf                   # the loss is infinite while 64 bits hold the probability
    value[7, 2:] = -120.0, -130.0
    x[7, 7] = -np.inf
    dy = g.standard_normal(rows).astype(F32)
    check_distill(kind, x, value, index, 1.0, dy, None, mode, what="ruled out")
    check_distill(kind, x, value, index, 1.0, dy, np.full(rows, 3.0, F32), mode, what="ruled out, norm")
    check_distill(kind, x, value, index, 0.5, dy, None, mode, n + 3, 1, what="ruled out, sharp")


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("mode", ["fused", "apart"])
@pytest.mark.parametrize("n,k", [(13, 8), (40, 9), (700, 64), (3000, 30)])
def test_large_losses(kind, mode, n, k):
    # logits far apart: a loss of hundreds to thousands, of which the bound leaves little more than its own rounding
    g = np.random.default_rng(n + k)
    rows = 60
    x = rounded(800.0 * g.standard_normal((rows, n)), kind)
    value, index = slots(g, rows, n, k, absent=0.1)
    dy = g.standard_normal(rows).astype(F32)
    for t in (1.0, 0.5):
        check_distill(kind, x, value, index, t, dy, None, mode, what="large losses")
