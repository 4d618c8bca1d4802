"""The loss of distillation where a slot's probability is smaller than 32 bits hold, on the GPU: the loss alone and the call that
also gives the gradient agree on it."""
import numpy as np
import pytest

from gpu_util import F32
from test_gpu_class_rows import TYPES, check_distill, logits

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
