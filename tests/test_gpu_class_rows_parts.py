"""Rows of many classes that are cut into parts on the GPU (few rows of more than 65536 classes): parts that hold nothing, and
rows that the fast form of the sums does not measure."""
import numpy as np
import pytest
import torch

import class_rows_ref as ref
from gpu_util import F32, call
from test_gpu_class_rows import TYPES, U, check_results, logits, rounded, run_distill, slots

pytestmark = pytest.mark.gpu


def check_wide(kind, x, value, index, t, dy, log_norm, mode, stride, offset, what):
    """As check_distill(), of rows whose loss may lie near the end of the range of 32 bits or beyond it.

    The probabilities of the call that also gives the gradient are rounded three times to 32 bits (exponential, scale, product): a
    loss is off by 3 U of its terms' sizes besides what check_results() counts.  That is far below the row's sum's share, but
    for losses of 1e30 and more, whose terms of that size have one sign: 3 U of the loss itself, and U for its own rounding.
    Beyond the range (a number from the largest one and half its step, 2^-25 of it, on rounds to infinity) as a whole it has to be
    infinite, and may be where part of want +- 3 U lies there."""
    old = rounded(np.random.default_rng(9).standard_normal(x.shape), kind) if mode == "accumulate" else None
    loss, top, total, dx = run_distill(kind, x, value, index, t, dy, log_norm, mode, stride, offset, False, old)
    want = ref.distill(x, value, index, t, log_norm)[0]
    loss = loss.astype(np.float64)
    edge = float(np.finfo(F32).max) * (1 + 2.0 ** -25)
    for r in np.flatnonzero(np.isfinite(want) & (want > 1e30)):
        good = loss[r] == np.inf if want[r] * (1 + 3 * U) >= edge else False
        if want[r] * (1 - 3 * U) < edge:
            good = good or abs(loss[r] - want[r]) <= 4.1 * U * want[r]
        assert good, (what, r, loss[r], want[r])
        loss[r] = want[r]
    check_results(kind, x, value, index, t, dy, log_norm, mode, old, what, (loss, top, total, dx))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("mode", ["fused", "apart", "accumulate"])
@pytest.mark.parametrize("n", [131077, 65537, 65536])
def test_distill_masks_and_special_values_of_long_rows(kind, mode, n):
    g = np.random.default_rng(11)
    k = 6
    low, high = float(torch.finfo(TYPES[kind]).min), float(torch.finfo(TYPES[kind]).max)
    x = logits(g, 14, n, kind)
    value, index = slots(g, 14, n, k, absent=0.0)
    x[0, g.random(n) < 0.9] = -np.inf
    x[0, index[0]] = 0.5
    x[1] = low
    x[2, :] = -np.inf
    x[3, 17] = np.nan
    x[4, 60017] = np.inf
    x[5] = np.nan
    index[5] = ref.NONE
    x[6] = -np.inf
    index[6] = n + 3
    value[6] = np.nan
    x[7, :40000] = -np.inf                           # whole parts that a mask leaves empty
    x[7, index[7]] = 0.25
    x[8, 1000:] = low                                # ... or at the lowest value
    x[9, ::3], x[9, 1::3] = low, high
    x[10, :] = 0.0
    index[11] = index[11, 0]
    x[12, n // 2:] = np.nan                          # a NaN in some of the parts
    x[13] = high                                     # nothing but the largest value
    dy = g.standard_normal(14).astype(F32)
    dy[6] = np.nan
    check_wide(kind, x, value, index, 1.0, dy, None, mode, 0, 0, "long special")
    check_wide(kind, x[:3], value[:3], index[:3], 4.0, dy[:3], np.full(3, 7.0, F32), mode, n + 5, 1, "long special, norm")


def test_rows_of_one_value_beyond_what_32_bits_count():
    # 2^31 classes that all weigh the same, at a value outside the fast form's range: the sum is their number
    n = 2 ** 31 + 1003
    low = -65504.0
    x = torch.full((n,), low, dtype=torch.float16, device="cuda")
    value, index = torch.zeros(1, device="cuda"), torch.full((1,), 77, dtype=torch.int32, device="cuda")
    loss, top, total, norm = (torch.empty(1, device="cuda") for _ in range(4))
    print("large: loss", flush=True)
    call("anode_gpu_softmax_distill_rows_f16", n, 1, 0, 1, 1.0, x, value, index, None, loss, top, total)
    # (each part's sum is exact but for its threads' and waves' meeting in 32 bits, and so are the parts': 22 half steps)
    assert float(top) == low and abs(float(total) - n) <= 24 * U * n
    assert abs(float(loss) - np.log(float(n))) <= 24 * U + U * np.log(float(n))
    print("large: norm", flush=True)
    call("anode_gpu_top_k_rows_f16", n, 1, 0, 0, 1.0, x, None, None, norm)
    want = low + np.log(float(n))
    assert abs(float(norm) - want) <= 24 * U + U * abs(want)
