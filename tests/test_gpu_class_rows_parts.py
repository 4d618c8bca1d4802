"""Rows of many classes that are cut into parts on the GPU (few rows of more than 65536 classes): what meets at the parts'
borders, parts that hold nothing, and rows that the fast form of the sums does not measure."""
import numpy as np
import pytest
import torch

import class_rows_ref as ref
from gpu_util import F32, call
from test_gpu_class_rows import (TYPES, U, check_distill, check_results, check_top_k, check_verify, drafts, logits, rounded, run_distill,
                                 slots)

pytestmark = pytest.mark.gpu


def ordered_rows(g, n, kind):
    """Rows of orders, ties and masks; `per` classes of a row are a part where it is cut into four."""
    per = (-(-n // 4) + 1023) // 1024 * 1024
    at = np.arange(n)
    lowest = float(torch.finfo(TYPES[kind]).min)
    up = np.sort(g.standard_normal(n)).astype(F32) * 10
    rows = [up, up[::-1], np.zeros(n), np.full(n, -3.0), np.where(at % 2 == 0, 0.0, -0.0), (at // 100 % 7).astype(F32),
            np.where(np.abs(at - per) < 300, 2.0, -1.0),           # ties across a border between parts
            np.where(at < per, np.where(at >= per - 150, 1.0, -1.0), np.where(at < per + 60, 1.0, 0.0)),
            np.where(at // per == 2, 5.0 + at % 50, 0.0),          # the largest all in one part
            np.where(at // per == 1, -np.inf, 0.5 * (at % 11)),    # a part that a mask leaves empty
            np.where(at % per < 3, 1.0 * (at % 5), -np.inf),       # parts of three classes each
            np.where(at == n - 1, 7.0, -np.inf), np.where(at == per, -7.0, -np.inf), np.full(n, -np.inf),
            np.full(n, lowest), np.where(at % 9973 == 5, 1.0 * at / n, lowest),
            np.where(at // per == 3, np.nan, 1.0 * (at % 13)), np.where(at == per - 1, np.nan, 1.0 * (at % 17)), np.full(n, np.nan),
            np.where(at % per == per - 1, np.inf, 1.0 * (at % 3)), np.where(at // per == 0, np.inf, 0.0)]
    return rounded(np.stack([np.asarray(r, F32) for r in rows]), kind)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("k", [1, 33, 64, 200, 256, 341, 600, 1024])
def test_top_k_orders_ties_and_masks_in_parts(kind, k):
    n = 131077
    x = ordered_rows(np.random.default_rng(k), n, kind)
    for r in range(0, x.shape[0], 3):                # three rows a call: four parts each
        print("top_k in parts", kind, k, r, flush=True)
        check_top_k(kind, x[r:r + 3], k, 1.0, 0 if r % 2 else n + 7, r % 2, f"{kind} k={k} rows from {r}")


@pytest.mark.parametrize("kind", TYPES)
def test_top_k_of_a_row_of_many_parts(kind):
    n = 2 ** 21 + 5
    per = (-(-n // 64) + 1023) // 1024 * 1024
    at = np.arange(n)
    some = np.where((at % per) % 500 == 3, np.where(at % per < 30000, 2.0, 0.0), 0.0)   # sixty ties in each of the parts
    few = np.where((at % per) % 16000 == 9, 1.0 + at // per % 5, -np.inf)               # fewer than k a part
    g = np.random.default_rng(8)
    for name, row in (("some", some), ("few", few), ("zeros", np.zeros(n)), ("random", g.standard_normal(n)),
                      ("lowest", np.full(n, float(torch.finfo(TYPES[kind]).min)))):
        x = rounded(np.asarray(row, F32)[None], kind)
        for k in (1, 20, 21, 64, 300):
            print("top_k of many parts", kind, name, k, flush=True)
            check_top_k(kind, x, k, 1.0, what=f"{kind} {name} k={k}")


def check_wide(kind, x, value, index, t, dy, log_norm, mode, stride, offset, what):
    """As check_distill(), of rows whose loss may lie beyond the range of 32 bits: a number from the largest one and half its step
    (2^-25 of it) on rounds to infinity."""
    old = rounded(np.random.default_rng(9).standard_normal(x.shape), kind) if mode == "accumulate" else None
    loss, top, total, dx = run_distill(kind, x, value, index, t, dy, log_norm, mode, stride, offset, False, old)
    want = ref.distill(x, value, index, t, log_norm)[0]
    loss = loss.astype(np.float64)
    beyond = np.isfinite(want) & (want >= float(np.finfo(F32).max) * (1 + 2.0 ** -25))
    assert np.all(loss[beyond] == np.inf), what
    loss[beyond] = want[beyond]
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


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n", [65535, 65536, 65537])
def test_rows_at_the_border_of_one_launch(kind, n):
    g = np.random.default_rng(n)
    x = logits(g, 3, n, kind)
    check_top_k(kind, x, 50, 2.0, what="border")
    value, index = slots(g, 3, n, 20)
    index[:, 0] = n - 1
    check_distill(kind, x, value, index, 1.0, np.ones(3, F32), None, "apart", what="border")


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


# ---- verification ----


@pytest.mark.parametrize("n", [65536, 65537, 70001, 131072])
@pytest.mark.parametrize("point", [False, True])
def test_verify_long_rows(n, point):
    g = np.random.default_rng(n)
    target, draft, token = drafts(g, n, 2, 6)
    if point:
        token = target[:, :2].argmax(-1).astype(np.uint32)
    for offset, length in ((0, None), (1, np.array([0, 1, 2, 3, 2, 1], np.uint32))):
        check_verify(target, None if point else draft, token, length, g.random((6, 2)).astype(F32), g.random(6).astype(F32),
                     f"long {n} {point}", offset)


@pytest.mark.parametrize("n", [65536, 65537, 70001])
def test_verify_borders_of_long_rows(n):
    # dyadic weights at the ends of blocks: every sum is exact, the random numbers lie on the borders
    places = [0, 2047, 2048, 4095, 32768, 63487, 65535, n - 1] if n - 1 != 65535 else [0, 2047, 2048, 4095, 32768, 63487, 65534, 65535]
    picks = np.concatenate([np.arange(8) / 8.0, np.arange(8) / 8.0 + 1 / 16, [1.0, 1.5, np.nan, -1.0]]).astype(F32)
    B = picks.size
    target, draft = np.zeros((B, 2, n), F32), np.zeros((B, 1, n), F32)
    target[:, :, places] = 0.125
    token = np.full((B, 1), 5, np.uint32)             # of no probability: never taken
    # what is left is the target; as a point mass, too; and the row after a draft of nothing
    for d in (draft, None):
        got, count = check_verify(target, d, token, None, np.zeros((B, 1), F32), picks, "borders")
        assert not count.any() and list(got[:8, 0]) == places and list(got[8:16, 0]) == places
    draft[:, 0, places[::2]] = 0.125                  # every other weight goes
    check_verify(target, draft, token, None, np.zeros((B, 1), F32), picks, "every other")
    draft[:, 0, places] = 0.125                       # all go: the target's row itself
    check_verify(target, draft, token, None, np.zeros((B, 1), F32), picks, "nothing left")
    check_verify(target, None, token, np.zeros(B, np.uint32), np.zeros((B, 1), F32), picks, "no drafts")


@pytest.mark.parametrize("n", [65536, 70001])
def test_verify_degenerate_long_rows(n):
    g = np.random.default_rng(21)
    B = 8
    target, draft, token = drafts(g, n, 2, B)
    accept, pick = np.ones((B, 2), F32), g.random(B).astype(F32)
    draft[0] = target[0, :2]
    target[1, 0] = 0.0
    draft[1, 0] = 0.0
    target[2, 0, :] = np.nan
    target[2, 0, 60077] = 0.5
    draft[2, 0, 60077] = 0.25
    token[2, 0] = 3
    pick[3], pick[4], pick[5] = 1.0, np.nan, -1.0
    target[6, 0] = 0.0
    target[6, 0, n - 1] = 1.0
    draft[6, 0, n - 1] = 0.0
    target[7] = np.nan
    length = np.array([2, 2, 2, 0, 0, 0, 1, 0], np.uint32)
    got, _ = check_verify(target, draft, token, length, accept, pick, "degenerate")
    assert got[1, 0] == ref.NONE and got[7, 0] == ref.NONE and got[2, 0] == 60077 and got[6, 0] == n - 1
