"""The operators over rows of many classes on the GPU, against the plain 64-bit implementations of class_rows_ref.py:
top-k rows, distillation from top logits (loss, gradient, both at once) and the verification of drafted tokens.

Bars.  Classes, tokens and counts are equal, and so are the values that top-k hands on.  Sums, losses and gradients are
within the bounds that class_rows_ref.sum_bound derives, plus half a step of the type they are stored in."""
import numpy as np
import pytest
import torch

import class_rows_ref as ref
from gpu_util import F32, call, dev, host

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
# half a step relative to the value, and half of the smallest step
HALF_STEP = {"f32": (2.0 ** -24, 2.0 ** -150), "bf16": (2.0 ** -8, 2.0 ** -134), "f16": (2.0 ** -11, 2.0 ** -25)}
U = ref.U


class Rows:
    """A [rows, stride] array on the GPU, `offset` elements into an allocation, whose padding and surroundings hold
    a mark that must stay."""

    def __init__(self, values, kind, stride=0, offset=0, mark=77.0):
        rows, n = values.shape
        self.kind, self.rows, self.n, self.stride, self.offset = kind, rows, n, stride or n, offset
        self.buf = torch.full((offset + rows * self.stride + 32,), mark, dtype=TYPES[kind], device="cuda")
        self.view = self.buf[offset:offset + rows * self.stride]
        self.inner = self.view.view(rows, self.stride)[:, :n] if rows * n else None
        if rows * n:
            self.inner.copy_(torch.from_numpy(np.ascontiguousarray(values)).to(TYPES[kind]))
        self.mark = float(torch.tensor(mark, dtype=TYPES[kind]))

    def get(self):
        torch.cuda.synchronize()
        return self.inner.float().cpu().numpy() if self.rows * self.n else np.zeros((self.rows, self.n), F32)

    def check_surroundings(self, what):
        keep = torch.ones_like(self.buf, dtype=torch.bool)
        if self.rows * self.n:
            keep[self.offset:self.offset + self.rows * self.stride].view(self.rows, self.stride)[:, :self.n] = False
        assert bool((self.buf[keep] == self.mark).all()), f"{what}: wrote outside its rows"


def guarded(n, dtype=torch.float32):
    """An output of n elements between marks; returns it and a check."""
    mark = 77 if dtype != torch.float32 else 77.0
    buf = torch.full((n + 64,), mark, dtype=dtype, device="cuda")

    def check(what):
        assert bool((buf[:32] == mark).all()) and bool((buf[32 + n:] == mark).all()), f"{what}: wrote outside its array"

    return buf[32:32 + n], check


def u32(a):
    return dev(np.ascontiguousarray(a, np.uint32).view(np.int32))


def got_u32(t):
    return host(t).view(np.uint32)


def logits(g, rows, n, kind, masked=0.0):
    x = (3.0 * g.standard_normal((rows, n))).astype(F32)
    if masked:
        x[g.random((rows, n)) < masked] = -np.inf
    return rounded(x, kind)


def rounded(x, kind):
    return torch.from_numpy(np.asarray(x, F32)).to(TYPES[kind]).float().numpy()


def slots(g, rows, n, k, absent=0.2, same=0.0):
    """A teacher's slots: classes of the row, some slots absent in either way, some classes named twice."""
    index = np.zeros((rows, k), np.uint32)
    for r in range(rows):
        index[r] = g.permutation(max(n, k))[:k] if n <= 4096 else g.choice(n, k, replace=False)
    if same and k > 1:
        twice = g.random((rows, k)) < same
        index = np.where(twice, index[:, :1], index)
    value = (4.0 + 2.0 * g.standard_normal((rows, k))).astype(F32)
    out = g.random((rows, k)) < absent
    index = np.where(out & (g.random((rows, k)) < 0.5), np.uint32(ref.NONE), index).astype(np.uint32)
    value = np.where(out & (index != ref.NONE), F32(-np.inf), value).astype(F32)
    value = np.where(index == ref.NONE, F32(np.nan), value).astype(F32)  # what an absent slot holds is not looked at
    return value, index


# ---- top-k ----


def run_top_k(kind, x, k, t=1.0, stride=0, offset=0, norm=True):
    rows, n = x.shape
    xd = Rows(x, kind, stride, offset)
    value, check_v = guarded(rows * k)
    index, check_i = guarded(rows * k, torch.int32)
    log_norm, check_n = guarded(rows)
    call("anode_gpu_top_k_rows_" + kind, n, rows, stride, k, t, xd.view, value, index, log_norm if norm else None)
    for c in (check_v, check_i, check_n):
        c(f"top_k [{n}, {rows}] k={k}")
    xd.check_surroundings("top_k")
    return host(value).reshape(rows, k), got_u32(index).reshape(rows, k), host(log_norm)


def check_top_k(kind, x, k, t=1.0, stride=0, offset=0, what=""):
    t = float(F32(t))
    value, index, log_norm = run_top_k(kind, x, k, t, stride, offset)
    want_v, want_i = ref.top_k(x, k)
    assert np.array_equal(index, want_i), (what, np.argwhere(index != want_i)[:5])
    assert np.array_equal(value, want_v), what
    top, total = ref.stats(x, t)
    for r in range(x.shape[0]):
        with np.errstate(all="ignore"):
            want = top[r] / t + np.log(total[r])
        if not np.isfinite(want):
            assert np.array_equal(F32(log_norm[r]), F32(want), equal_nan=True), (what, r, log_norm[r], want)
        else:
            assert abs(log_norm[r] - want) <= ref.sum_bound(x[r], t) + U * abs(want), (what, r, log_norm[r], want)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n,rows,k", [(1, 3, 1), (2, 5, 3), (7, 4, 7), (8, 3, 2), (9, 2, 20), (63, 5, 10), (255, 3, 64), (256, 2, 256),
                                      (1000, 9, 10), (1000, 3, 1000), (2047, 3, 1024), (4099, 4, 50), (8191, 2, 65), (8200, 3, 129),
                                      (16384, 2, 1), (32768, 3, 50), (50257, 2, 300), (65537, 2, 1024), (131072, 2, 64),
                                      (262147, 1, 128)])
def test_top_k(kind, n, rows, k):
    print(f"top_k {kind} n={n} rows={rows} k={k}", flush=True)
    g = np.random.default_rng(n * 7 + k)
    for stride, offset in ((0, 0), (n + 13, 3)):
        check_top_k(kind, logits(g, rows, n, kind), k, 2.0, stride, offset, f"{kind} [{n}, {rows}] k={k} {stride} {offset}")


@pytest.mark.parametrize("kind", TYPES)
def test_top_k_orders_and_ties(kind):
    g = np.random.default_rng(3)
    n = 20011
    up = np.sort(g.standard_normal(n)).astype(F32) * 10
    lowest = float(torch.finfo(TYPES[kind]).min)
    rows = [up, up[::-1], np.zeros(n), np.full(n, -3.0), np.where(np.arange(n) % 2 == 0, 0.0, -0.0),
            (np.arange(n) // 100 % 7).astype(F32),               # thousands of ties
            np.where(np.arange(n) < 40, 5.0, np.where(np.arange(n) < n - 30, 1.0, 2.0)),
            np.full(n, lowest), np.where(np.arange(n) % 997 == 5, 1.0 * np.arange(n) / n, lowest),
            np.where(np.arange(n) % 1024 == 7, 3.0, -1.0),      # the largest all in one lane's places
            np.concatenate([np.full(n - 70, -1.0), np.arange(70)])]
    x = rounded(np.stack([np.asarray(r, F32) for r in rows]), kind)
    for k in (1, 33, 64, 200, 256, 1024):
        print("top_k orders", kind, k, flush=True)
        check_top_k(kind, x, k, 1.0, what=f"{kind} k={k}")


@pytest.mark.parametrize("kind", TYPES)
def test_top_k_masks(kind):
    g = np.random.default_rng(4)
    for n in (5, 1000, 30000):
        x = logits(g, 9, n, kind)
        x[0] = -np.inf                                       # a mask that leaves nothing
        x[1, :] = -np.inf
        x[1, n // 2] = 1.0                                   # and one that leaves one class
        x[2, ::2] = -np.inf
        x[3, 1:] = np.nan                                    # NaN is not taken; the row's norm is NaN
        x[4] = np.nan
        x[5, n // 3] = np.inf
        x[6, g.random(n) < 0.99] = -np.inf
        x[7, :3] = float(torch.finfo(TYPES[kind]).max)
        x[8, g.random(n) < 0.5] = float(torch.finfo(TYPES[kind]).min)
        for k in (1, 4, 100):
            check_top_k(kind, x, k, what=f"{kind} n={n} k={k}")


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("row", [4096, 8192, 16384, 32768, 65536])
@pytest.mark.parametrize("k", [32, 33, 64, 65, 256, 257])
def test_top_k_rows_at_the_borders(kind, row, k):
    # where the number of threads and of groups in a segment changes
    g = np.random.default_rng(row + k)
    for n in (row // TYPES[kind].itemsize + more for more in (-1, 0, 1)):
        x = logits(g, 4, n, kind)
        x[1] = np.sort(x[1])
        x[2, g.random(n) < 0.9] = -np.inf
        x[3] = 0.5
        check_top_k(kind, x, k, 1.0, n + 1, 1, what=f"border {n}")


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("k", [1, 64, 200, 1000])
def test_top_k_of_large_arrays(kind, k):
    # more than the last cache holds: 800 rows (400 of floats) of an odd length, and rows in order, of ties and of masks
    n, stride = 131071, 131075
    rows = 800 if kind != "f32" else 400
    g = torch.Generator("cuda").manual_seed(k)
    buf = torch.randn(1 + rows * stride, generator=g, device="cuda").mul_(3.0).to(TYPES[kind])
    grid = buf[1:].view(rows, stride)
    ramp = torch.arange(n, device="cuda") / 1024.0 - 60.0
    grid[0, :n], grid[1, :n] = ramp.to(TYPES[kind]), ramp.flip(0).to(TYPES[kind])
    grid[2], grid[3] = 0.0, torch.finfo(TYPES[kind]).min
    grid[3, 5::9001] = 1.0
    grid[4] = -float("inf")
    grid[4, 7::30011] = -2.0
    grid[5, ::256] += 20.0                         # the largest all in a few threads' places
    grid[6, 1000:1300] += 20.0                     # ... and all in one place
    x = grid[:, :n].float()
    grid[:, n:] = float("inf")                     # what lies behind a row is not looked at
    value, check_v = guarded(rows * k)
    index, check_i = guarded(rows * k, torch.int32)
    norm, check_n = guarded(rows)
    call("anode_gpu_top_k_rows_" + kind, n, rows, stride, k, 2.0, buf[1:], value, index, norm)
    for c in (check_v, check_i, check_n):
        c("top_k of a large array")
    v, i = value.view(rows, k), index.view(rows, k)
    want, _ = torch.sort(x, dim=1, descending=True)
    want = want[:, :k]
    assert bool((v == want).all())
    found = want > -float("inf")
    assert bool((x.gather(1, i.long().clamp(0, n - 1))[found] == want[found]).all()) and bool((i[~found] == -1).all())
    tied = (v[:, 1:] == v[:, :-1]) & found[:, 1:]
    assert bool((i[:, 1:] > i[:, :-1])[tied].all())  # of equal values the lower class first: so all differ
    for r in (0, 2, 3, 4, 5, 6, rows - 1):
        row = x[r:r + 1].cpu().numpy()
        assert np.array_equal(host(i[r]).view(np.uint32), ref.top_k(row, k)[1][0]), r
        top, total = ref.stats(row, 2.0)
        norm_want = top[0] / 2.0 + np.log(total[0])
        assert abs(float(norm[r]) - norm_want) <= ref.sum_bound(row[0], 2.0) + U * abs(norm_want), r


def test_top_k_without_norm_and_with_norm_alone():
    g = np.random.default_rng(5)
    x = logits(g, 4, 3000, "f32")
    value, index, norm = run_top_k("f32", x, 5, norm=False)
    want_v, want_i = ref.top_k(x, 5)
    assert np.array_equal(index, want_i) and np.array_equal(value, want_v) and np.all(norm == 77.0)
    xd = dev(x)
    out, check = guarded(4)
    call("anode_gpu_top_k_rows_f32", 3000, 4, 0, 0, 0.5, xd, None, None, out)
    check("norm alone")
    want = ref.stats(x, 0.5)
    assert np.allclose(host(out), want[0] / 0.5 + np.log(want[1]), rtol=1e-5)


def test_top_k_of_one_is_arg_max():
    g = np.random.default_rng(6)
    x = logits(g, 50, 1999, "f32")
    x[:, 700] = x.max(1)
    value, index, _ = run_top_k("f32", x, 1)
    arg = torch.empty(50, dtype=torch.int32, device="cuda")
    call("anode_gpu_arg_max_packed_u32", 1999, 50, dev(x), arg)
    assert np.array_equal(index[:, 0], got_u32(arg))


# ---- distillation ----


def run_distill(kind, x, value, index, t, dy, log_norm, mode, stride=0, offset=0, in_place=False, old=None, apart=0):
    """loss, row_max, row_sum, dx of one of the ways to get them."""
    rows, n = x.shape
    k = value.shape[1]
    xd = Rows(x, kind, stride, offset + apart)
    tv, ti = dev(value) if value.size else torch.zeros(1, device="cuda"), u32(index) if index.size else torch.zeros(
        1, dtype=torch.int32, device="cuda")
    tn = None if log_norm is None else dev(np.asarray(log_norm, F32))
    loss, top, total = guarded(rows), guarded(rows), guarded(rows)
    head = (n, rows, stride, k, t)
    if mode == "fused":
        dx = xd if in_place else Rows(np.full((rows, n), 5.0, F32), kind, stride, offset)
        call("anode_gpu_softmax_distill_fused_fwd_bwd_rows_" + kind, *head, xd.view, tv, ti, tn, dev(dy), loss[0], top[0], total[0],
             dx.view)
    else:
        call("anode_gpu_softmax_distill_rows_" + kind, *head, xd.view, tv, ti, tn, loss[0], top[0], total[0])
        if not in_place:
            assert np.array_equal(xd.get(), x, equal_nan=True)
        if mode == "accumulate":
            dx = Rows(old, kind, stride, offset)
            call("anode_gpu_softmax_distill_bwd_rows_accumulate_" + kind, *head, dev(dy), xd.view, tv, ti, tn, top[0], total[0],
                 dx.view)
        else:
            dx = xd if in_place else Rows(np.full((rows, n), 5.0, F32), kind, stride, offset)
            call("anode_gpu_softmax_distill_bwd_rows_" + kind, *head, dev(dy), xd.view, tv, ti, tn, top[0], total[0], dx.view)
    for o in (loss, top, total):
        o[1]("distill")
    xd.check_surroundings("distill x")
    dx.check_surroundings("distill dx")
    return host(loss[0]), host(top[0]), host(total[0]), dx.get()


def check_distill(kind, x, value, index, t, dy, log_norm, mode, stride=0, offset=0, in_place=False, what="", apart=0):
    rows, n = x.shape
    t = float(F32(t))  # the entry point's argument has 32 bits
    old = rounded(np.random.default_rng(9).standard_normal((rows, n)), kind) if mode == "accumulate" else None
    check_results(kind, x, value, index, t, dy, log_norm, mode, old, what,
                  run_distill(kind, x, value, index, t, dy, log_norm, mode, stride, offset, in_place, old, apart))


def check_results(kind, x, value, index, t, dy, log_norm, mode, old, what, got):
    """Loss, row_max, row_sum and dx against the plain forms, within their bounds."""
    rows, n = x.shape
    loss, top, total, dx = got
    want_loss, want_top, want_total = ref.distill(x, value, index, t, log_norm)
    want_dx, q, p = ref.distill_grad(x, value, index, t, dy, log_norm)
    assert np.array_equal(top.astype(np.float64), want_top), what
    half, least = HALF_STEP[kind]
    for r in range(rows):
        s = ref.sum_bound(x[r], t)
        mass = p[r].sum()
        where = f"{what} {kind} [{n}, {rows}] {mode} row {r}"
        # 64-bit terms on the row's 32-bit sum: its error times the mass, and the rounding of the result
        if np.isfinite(want_loss[r]):
            bound = mass * s + U * abs(want_loss[r]) + 1e-11
            assert abs(loss[r] - want_loss[r]) <= bound, (where, loss[r], want_loss[r], bound)
        else:
            assert np.array_equal(F32(want_loss[r]), loss[r], equal_nan=True), (where, loss[r], want_loss[r])
        if np.isfinite(want_total[r]):
            assert abs(total[r] - want_total[r]) <= (s + U) * want_total[r], (where, total[r], want_total[r])
        else:
            assert np.isnan(total[r]), where
        if not n:
            continue
        want = want_dx[r] + (0.0 if old is None else old[r].astype(np.float64))
        nan = np.isnan(want)
        assert np.array_equal(nan, np.isnan(dx[r])), (where, "NaN pattern")
        if nan.all():
            continue
        if not ((index[r] < n) & (value[r] > -np.inf)).any():  # a row without a slot: exact, whatever dy and x hold
            assert np.array_equal(dx[r], np.zeros(n, F32) if old is None else old[r]), where
            continue
        w = abs(float(dy[r])) / t
        m = 1.0 if log_norm is None else mass
        with np.errstate(all="ignore"):
            a = np.where(x[r] > -np.inf, (want_top[r] - x[r].astype(np.float64)) / t * 1.4427, 0.0)
        # the exponential's own error (as in sum_bound), the scale's and the product's rounding, the row's sum; the slots'
        # probabilities are rounded to 32 bits; results below 2^-126 may be flushed
        mine = np.zeros(n)
        ok = (index[r] < n) & (value[r] > -np.inf)
        np.add.at(mine, index[r][ok].astype(np.int64), p[r][ok])
        bound = w * m * np.nan_to_num(q[r]) * (s + (8 + 3 * np.log(2) * a) * U) + 2 * U * w * mine + w * 2.0 ** -120
        if old is not None:
            bound = bound + U * (np.abs(want) + np.abs(want_dx[r]))
        bound = bound + (half + U) * np.abs(want) + least
        # beyond the type's range rounding gives an infinity: so where the whole interval want +- bound lies beyond it
        # (from the largest value and half a step on), and either that or a number within the bound where part of it does
        largest = float(torch.finfo(TYPES[kind]).max)
        edge = largest * (1 + HALF_STEP[kind][0])
        good = np.abs(dx[r] - want) <= bound
        good = np.where(np.abs(want) + bound >= edge, good | (dx[r] == np.copysign(np.inf, want)), good)
        bad = np.flatnonzero(~good)
        assert bad.size == 0, (where, bad[:5], dx[r][bad[:5]], want[bad[:5]], bound[bad[:5]])


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("apart", [1, 2, 5])
def test_distill_of_arrays_that_lie_unlike_each_other(kind, apart):
    g = np.random.default_rng(apart)
    for n in (130, 9001):
        x = logits(g, 5, n, kind)
        value, index = slots(g, 5, n, 9)
        for mode in ("fused", "apart", "accumulate"):
            check_distill(kind, x, value, index, 1.0, g.standard_normal(5).astype(F32), None, mode, n + 3, 1, what="unlike", apart=apart)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n,stride", [(130, 261), (130, 260), (9001, 20001)])
def test_distill_of_a_gradient_between_the_rows_of_the_logits(kind, n, stride):
    # one array of rows twice as long: the logits and the gradient lie beside each other in it
    g = np.random.default_rng(n + stride)
    rows, k = 5, 9
    x = logits(g, rows, n, kind)
    value, index = slots(g, rows, n, k)
    dy = g.standard_normal(rows).astype(F32)
    for first in (0, stride - n):                  # the gradient before the logits' rows, and behind them
        both = torch.full((rows * stride + n,), 3.0, dtype=TYPES[kind], device="cuda")
        grid = both[:rows * stride].view(rows, stride)
        at = stride - n - first
        grid[:, at:at + n] = torch.from_numpy(x).to("cuda").to(TYPES[kind])
        out = [torch.empty(rows, device="cuda") for _ in range(3)]
        call("anode_gpu_softmax_distill_fused_fwd_bwd_rows_" + kind, n, rows, stride, k, 1.0, both[at:], dev(value), u32(index), None,
             dev(dy), *out, both[first:])
        got = grid.float().cpu().numpy()
        assert np.array_equal(got[:, at:at + n], x)
        check_results(kind, x, value, index, 1.0, dy, None, "fused", None, f"between {first}",
                      (*map(host, out), got[:, first:first + n]))
        left = np.delete(got, np.r_[at:at + n, first:first + n], 1)
        assert np.all(left == 3.0) and bool((both[rows * stride:] == 3.0).all())


@pytest.mark.parametrize("kind", TYPES)
def test_distill_accumulates_onto_the_logits_themselves(kind):
    g = np.random.default_rng(15)
    for n in (77, 4100, 40000):
        x = logits(g, 6, n, kind)
        value, index = slots(g, 6, n, 12)
        dy = g.standard_normal(6).astype(F32)
        teacher = (dev(value), u32(index), None)
        stats = [torch.empty(6, device="cuda") for _ in range(3)]
        rows = Rows(x, kind)
        call("anode_gpu_softmax_distill_rows_" + kind, n, 6, 0, 12, 1.0, rows.view, *teacher, *stats)
        apart = Rows(x, kind)
        call("anode_gpu_softmax_distill_bwd_rows_accumulate_" + kind, n, 6, 0, 12, 1.0, dev(dy), rows.view, *teacher, *stats[1:], apart.view)
        call("anode_gpu_softmax_distill_bwd_rows_accumulate_" + kind, n, 6, 0, 12, 1.0, dev(dy), rows.view, *teacher, *stats[1:], rows.view)
        assert np.array_equal(rows.get(), apart.get())
        rows.check_surroundings("accumulate in place")


# rows that fill the registers they are held in to the last value, and one value more; and the next workgroup's
HELD = [2048, 4096, 12288, 18432, 43008, 71680, 143360, 276480]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("row", HELD)
@pytest.mark.parametrize("more", [-1, 0, 1])
def test_distill_rows_at_the_borders(kind, row, more):
    n = row // TYPES[kind].itemsize + more
    rows = 34                                      # (more than are cut into parts)
    g = np.random.default_rng(n)
    x = np.broadcast_to(logits(g, 1, n, kind), (rows, n)).copy()
    x[:, :3] = rounded(g.standard_normal((rows, 3)), kind)
    value, index = slots(g, rows, n, 7)
    for r in range(rows):
        index[r, :2] = n - 1, (r * 64 + r) % n     # the row's last value, and places of every kind
    index[:, 2:] = np.where(index[:, 2:] == index[:, :1], ref.NONE, index[:, 2:])
    dy = g.standard_normal(rows).astype(F32)
    for stride, offset, in_place in ((0, 0, False), (n + 1, 1, True)):
        check_distill(kind, x, value, index, 1.0, dy, None, "fused", stride, offset, in_place, "border")


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("mode", ["fused", "apart"])
@pytest.mark.parametrize("n", [1001, 2600, 4095])
def test_distill_of_many_short_rows(kind, mode, n):
    g = np.random.default_rng(n)
    rows = 1030
    x = logits(g, rows, n, kind)
    value, index = slots(g, rows, n, 20)
    check_distill(kind, x, value, index, 1.5, g.standard_normal(rows).astype(F32), None, mode, what="many")


SHAPES = [(1, 3, 1), (2, 5, 3), (7, 4, 7), (8, 3, 2), (9, 2, 9), (63, 5, 10), (255, 3, 64), (257, 2, 0), (1000, 40, 10), (1000, 2, 700),
          (2047, 3, 33), (4099, 4, 50), (8191, 2, 65), (16385, 2, 1), (32768, 3, 32), (50257, 2, 1024), (65541, 2, 128), (131072, 2, 64),
          (262147, 1, 200)]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n,rows,k", SHAPES)
def test_distill(kind, n, rows, k):
    print(f"distill {kind} n={n} rows={rows} k={k}", flush=True)
    g = np.random.default_rng(n * 3 + k)
    x = logits(g, rows, n, kind)
    value, index = slots(g, rows, n, k, same=0.1 if rows > 2 else 0.0)
    dy = (g.standard_normal(rows) * 100).astype(F32)
    norm = (6.0 + g.standard_normal(rows)).astype(F32)
    for mode, log_norm, t, stride, offset, in_place in (
            ("fused", None, 1.0, 0, 0, False), ("apart", norm, 2.0, 0, 0, False), ("accumulate", norm, 0.7, n + 13, 3, False),
            ("fused", norm, 3.0, n + 13, 5, True), ("apart", None, 1.0, n + 64, 1, True), ("accumulate", None, 1.0, 0, 0, False)):
        check_distill(kind, x, value, index, t, dy, log_norm, mode, stride, offset, in_place, f"t={t} stride={stride} offset={offset}")


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("mode", ["fused", "apart", "accumulate"])
@pytest.mark.parametrize("n,k", [(30, 64), (3, 200), (700, 333), (5000, 1024), (40000, 1024)])
def test_distill_of_classes_named_many_times(kind, mode, n, k):
    g = np.random.default_rng(n + k)
    rows = 6
    x = logits(g, rows, n, kind)
    index = g.integers(0, n, (rows, k)).astype(np.uint32)      # drawn with replacement
    index[1] = index[1, 0]                                     # one class in every slot
    index[2] = g.integers(0, 2, k) * (n - 1)                   # the row's ends in turn
    index[3, ::2] = index[3, 1]
    index[4] = (np.arange(k) * 2048 % n).astype(np.uint32)     # classes that lie alike
    value = (4.0 + 2.0 * g.standard_normal((rows, k))).astype(F32)
    value[5, g.random(k) < 0.9] = -np.inf
    norm = np.array([np.logaddexp.reduce(v.astype(np.float64)) + 0.1 for v in value], F32)
    dy = g.standard_normal(rows).astype(F32)
    check_distill(kind, x, value, index, 1.0, dy, None, mode, what="repeated")
    check_distill(kind, x, value, index, 1.0, dy, norm, mode, n + 3, 1, what="repeated, norm")


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("mode", ["fused", "apart", "accumulate"])
def test_distill_masks_and_special_values(kind, mode):
    g = np.random.default_rng(11)
    n, k = 5000, 6
    low, high = float(torch.finfo(TYPES[kind]).min), float(torch.finfo(TYPES[kind]).max)
    x = logits(g, 14, n, kind)
    value, index = slots(g, 14, n, k, absent=0.0)
    x[0, g.random(n) < 0.9] = -np.inf
    x[0, index[0]] = 0.5
    x[1] = low                                     # a mask of the lowest value everywhere: uniform
    x[2, :] = -np.inf                              # nothing is left: NaN, as the row's softmax
    x[3, 17] = np.nan
    x[4, 17] = np.inf
    x[5] = np.nan                                  # an ignored row may hold anything
    index[5] = ref.NONE
    x[6] = -np.inf                                 # a padded position on both sides
    index[6] = n + 3
    value[6] = np.nan
    x[7, index[7, 2]] = -np.inf                    # the student rules out what the teacher holds likely
    x[8, index[8, 1]] = -np.inf                    # ... and what it does not (mass 0 by underflow)
    value[8, 1] = -3e38
    x[9, ::3], x[9, 1::3] = low, high              # the widest differences
    x[10, :] = 0.0
    index[11] = index[11, 0]                       # one class in every slot
    value[12, 1:] = -np.inf                        # one slot left
    value[13] = low                                # a teacher's row of lowest values: uniform over its slots
    dy = g.standard_normal(14).astype(F32)
    dy[6] = np.nan                                 # nothing of an ignored row shows
    check_distill(kind, x, value, index, 1.0, dy, None, mode, what="special")
    check_distill(kind, x, value, index, 4.0, dy, np.where(np.arange(14) == 13, low / 4.0, 7.0).astype(F32), mode, what="special, norm")


def test_distill_of_one_slot_is_the_categorical_nll():
    # one slot with all of the mass: the loss and gradient of softmax_cat_nll, within the bounds of the two
    g = np.random.default_rng(12)
    K, R = 1000, 64
    x = logits(g, R, K, "f32")
    label = g.integers(0, K, R).astype(np.uint32)
    dy = g.standard_normal(R).astype(F32)
    loss, _, _, dx = run_distill("f32", x, np.zeros((R, 1), F32), label[:, None], 1.0, dy, None, "fused")
    p, nll, want = (torch.empty(s, device="cuda") for s in (K * R, R, K * R))
    call("anode_gpu_softmax_cat_nll_fused_fwd_bwd_packed_f32", K, R, dev(x), u32(label), dev(dy), p, nll, want)
    assert np.all(np.abs(loss - host(nll)) <= 2e-6 * (1 + np.abs(loss)))
    assert np.all(np.abs(dx - host(want).reshape(R, K)) <= 4e-6 * np.abs(dy)[:, None])


def test_distill_gradient_against_differences():
    # central differences of the loss in 64 bits at the logits that differ most; their own error is h^2/6 of the third
    # derivative (each at most 1/t^3 in size here) and the rounding of two losses over 2 h
    g = np.random.default_rng(13)
    n, rows, k, t = 40, 3, 5, 1.5
    x = logits(g, rows, n, "f32")
    value, index = slots(g, rows, n, k, absent=0.0)
    dy = np.ones(rows, F32)
    _, _, _, dx = run_distill("f32", x, value, index, t, dy, None, "fused")
    h = 1e-4
    x64 = x.astype(np.float64)
    for r in range(rows):
        for j in range(n):
            lo, hi = x64.copy(), x64.copy()
            lo[r, j] -= h
            hi[r, j] += h
            d = (ref.distill(hi, value, index, t)[0][r] - ref.distill(lo, value, index, t)[0][r]) / (2 * h)
            assert abs(d - dx[r, j]) <= h * h / 6 + 1e-11 + 40 * U, (r, j, d, dx[r, j])


def test_distill_reads_what_top_k_wrote():
    g = np.random.default_rng(14)
    for kind in TYPES:
        n, rows, k, t = 3001, 20, 16, 2.0
        teacher = logits(g, rows, n, kind, masked=0.3)
        teacher[4] = -np.inf                       # a position without a teacher: its slots come out absent
        teacher[5, 3:] = -np.inf                   # fewer classes than slots
        td = Rows(teacher, kind)
        value, index = torch.empty(rows * k, device="cuda"), torch.empty(rows * k, dtype=torch.int32, device="cuda")
        norm = torch.empty(rows, device="cuda")
        call("anode_gpu_top_k_rows_" + kind, n, rows, 0, k, t, td.view, value, index, norm)
        x = logits(g, rows, n, kind)
        v, i, ln = host(value).reshape(rows, k), got_u32(index).reshape(rows, k), host(norm)
        assert np.all(i[4] == ref.NONE) and ln[4] == -np.inf and np.all(i[5, 3:] == ref.NONE)
        for mode in ("fused", "apart"):
            check_distill(kind, x, v, i, t, np.full(rows, 0.05, F32), ln, mode, what="record")


# ---- verification of drafted tokens ----


def probabilities(g, *shape, sharp=2.0):
    z = sharp * g.standard_normal(shape)
    z = np.exp(z - z.max(-1, keepdims=True))
    return (z / z.sum(-1, keepdims=True)).astype(F32)


def drafts(g, n, G, B, near=0.5):
    target = probabilities(g, B, G + 1, n)
    noisy = target[:, :G].astype(np.float64) * np.exp(near * g.standard_normal((B, G, n)))
    draft = (noisy / noisy.sum(-1, keepdims=True)).astype(F32)
    token = np.zeros((B, G), np.uint32)
    for b in range(B):
        for i in range(G):
            c = np.cumsum(draft[b, i].astype(np.float64))
            token[b, i] = min(n - 1, np.searchsorted(c, g.random() * c[-1], side="right"))
    return target, draft, token


def run_verify(target, draft, token, length, accept, pick, offset=0):
    B, G1, n = target.shape
    out, check_o = guarded(B * G1, torch.int32)
    accepted, check_a = guarded(B, torch.int32)
    one = torch.zeros(1, device="cuda")
    call("anode_gpu_verify_draft_packed_f32", n, G1 - 1, B, dev(target, offset) if target.size else one,
         None if draft is None else dev(draft, offset) if draft.size else one,
         u32(token) if token.size else one, None if length is None else u32(length),
         dev(np.asarray(accept, F32)) if np.size(accept) else one, dev(np.asarray(pick, F32)), out, accepted)
    check_o("verify tokens")
    check_a("verify counts")
    return got_u32(out).reshape(B, G1), got_u32(accepted)


def check_verify(target, draft, token, length, accept, pick, what="", offset=0):
    got, n_got = run_verify(target, draft, token, length, accept, pick, offset)
    want, n_want = ref.verify(target, draft, token, length, accept, pick)
    assert np.array_equal(n_got, n_want), (what, n_got, n_want)
    assert np.array_equal(got, want), (what, got[(got != want).any(1)], want[(got != want).any(1)])
    return got, n_got


@pytest.mark.parametrize("n,G,B", [(1, 1, 2), (2, 3, 9), (3, 0, 5), (5, 2, 7), (63, 4, 20), (64, 1, 3), (257, 70, 3), (1000, 5, 30),
                                   (4097, 3, 5), (16391, 2, 6), (50257, 4, 4), (131072, 3, 3), (300007, 1, 2)])
@pytest.mark.parametrize("point", [False, True])
def test_verify(n, G, B, point):
    print(f"verify n={n} G={G} B={B} point={point}", flush=True)
    g = np.random.default_rng(n + G)
    target, draft, token = drafts(g, n, G, B)
    if point and G:
        token = target[:, :G].argmax(-1).astype(np.uint32)
    for offset, length in ((0, None), (1, g.integers(0, G + 3, B).astype(np.uint32))):
        accept, pick = g.random((B, G)).astype(F32), g.random(B).astype(F32)
        check_verify(target, None if point else draft, token, length, accept, pick, f"[{n}, {G}, {B}] {point} {offset}", offset)


@pytest.mark.parametrize("B", [200, 300, 600])
@pytest.mark.parametrize("n", [500, 8195])
def test_verify_many_sequences(n, B):
    g = np.random.default_rng(n + B)
    target, draft, token = drafts(g, n, 1, B)
    accept, pick = g.random((B, 1)).astype(F32), g.random(B).astype(F32)
    check_verify(target, draft, token, None, accept, pick, f"[{n}, 1, {B}]")


def test_verify_borders():
    # dyadic probabilities: every sum is exact, and the random numbers lie on the borders
    target = np.zeros((8, 2, 8), F32)
    target[:, 0, :4] = [0.5, 0.25, 0.125, 0.125]
    target[:, 1, 2:6] = [0.25, 0.25, 0.25, 0.25]
    draft = np.zeros((8, 1, 8), F32)
    draft[:, 0, :4] = [0.25, 0.25, 0.25, 0.25]
    token = np.array([0, 2, 2, 2, 2, 5, 8, 2], np.uint32)[:, None]
    accept = np.array([0.999, 0.5, 0.4999, 0.5, 0.0, 0.0, 0.0, 0.5], F32)[:, None]
    pick = np.array([0.0, 0.0, 0.25, 0.999, 0.5, 0.0, 0.3, 1.0], F32)
    got, n = check_verify(target, draft, token, None, accept, pick, "borders")
    assert list(n) == [1, 0, 1, 0, 1, 0, 0, 0]    # 0.5 * 0.25 < 0.125 is false; a class outside is never taken
    assert list(got[0]) == [0, 2] and list(got[1]) == [0, ref.NONE] and list(got[2]) == [2, 3] and list(got[4]) == [2, 4]
    # as a point mass: what is left is the target without the token
    check_verify(target, None, token, None, accept, pick, "borders, point")


def test_verify_degenerate_rows():
    g = np.random.default_rng(21)
    n, B = 1500, 10
    target, draft, token = drafts(g, n, 2, B)
    accept, pick = np.ones((B, 2), F32), g.random(B).astype(F32)   # u = 1: taken only if p > q
    draft[0] = target[0, :2]                        # nothing is left of the difference: the target's row
    accept[0] = 1.0
    target[1, 0] = 0.0                              # nothing to draw from
    draft[1, 0] = 0.0
    target[2, 0, :] = np.nan                        # NaN weighs nothing
    target[2, 0, 77] = 0.5
    draft[2, 0, 77] = 0.25
    token[2, 0] = 3
    pick[3], pick[4], pick[5], pick[6] = 1.0, np.nan, -1.0, 1.5
    target[7, 0] = 0.0
    target[7, 0, n - 1] = 1.0                       # the last class holds everything
    draft[7, 0, n - 1] = 0.0
    target[8] = np.nan
    length = np.array([2, 2, 2, 0, 0, 0, 0, 1, 0, 2], np.uint32)
    got, _ = check_verify(target, draft, token, length, accept, pick, "degenerate")
    assert got[1, 0] == ref.NONE and got[8, 0] == ref.NONE and got[2, 0] == 77 and got[7, 0] == n - 1


def test_verify_without_classes_draws_nothing():
    out, accepted = run_verify(np.zeros((3, 3, 0), F32), np.zeros((3, 2, 0), F32), np.zeros((3, 2), np.uint32), None,
                               np.zeros((3, 2), F32), np.zeros(3, F32))
    assert np.all(out == ref.NONE) and np.all(accepted == 0)


def test_drawing_follows_the_probabilities():
    # one token of each row for many evenly spaced numbers: the counts are the probabilities to within one
    g = np.random.default_rng(22)
    n, B = 37, 4096
    p = probabilities(g, 1, 1, n)
    pick = ((np.arange(B) + 0.5) / B).astype(F32)
    got, _ = run_verify(np.broadcast_to(p, (B, 1, n)).copy(), None, np.zeros((B, 0), np.uint32), None, np.zeros((B, 0), F32), pick)
    counts = np.bincount(got[:, 0].astype(np.int64), minlength=n)
    assert np.all(np.abs(counts - B * p[0, 0]) <= 1.0 + 1e-3)


# ---- all of them together ----


def test_a_draft_model_is_distilled_and_its_tokens_verified():
    """The chain as it is used: the target's rows give a record, the draft model's head takes gradient steps on it, and
    its tokens are then verified."""
    g = np.random.default_rng(30)
    n, B, G, k, t = 2000, 64, 2, 64, 1.0
    rows = B * (G + 1)
    z = rounded(3.0 * g.standard_normal((rows, n)), "bf16")
    teacher = Rows(z, "bf16")
    value, index = torch.empty(rows * k, device="cuda"), torch.empty(rows * k, dtype=torch.int32, device="cuda")
    norm, ones = torch.empty(rows, device="cuda"), torch.ones(rows, device="cuda")
    call("anode_gpu_top_k_rows_bf16", n, rows, 0, k, t, teacher.view, value, index, norm)
    student = dev(np.zeros((rows, n), F32))
    dx = torch.empty_like(student)
    loss, top, total = (torch.empty(rows, device="cuda") for _ in range(3))
    losses = []
    for step in range(3):
        call("anode_gpu_softmax_distill_fused_fwd_bwd_rows_f32", n, rows, 0, k, t, student, value, index, norm, ones, loss, top, total, dx)
        losses.append(host(loss).copy())
        want = ref.distill(host(student).reshape(rows, n), host(value).reshape(rows, k), got_u32(index).reshape(rows, k), t, host(norm))
        assert np.all(np.abs(losses[-1] - want[0]) <= 1e-5 * (1 + np.abs(want[0])))
        call("anode_gpu_online_add_packed_f32", rows * n, -100.0, dx, student)     # student -= 100 dx
    p, q = torch.empty(rows * n, device="cuda"), torch.empty(rows * n, device="cuda")
    call("anode_gpu_softmax_packed_deterministic_f32", n, rows, dev(z), p)
    call("anode_gpu_softmax_packed_deterministic_f32", n, rows, student, q)
    target = host(p).reshape(B, G + 1, n)
    draft = np.ascontiguousarray(host(q).reshape(B, G + 1, n)[:, :G])
    tokens = []
    for i in range(G):                              # the draft's tokens, drawn from its rows
        got, _ = run_verify(draft[:, i:i + 1], None, np.zeros((B, 0), np.uint32), None, np.zeros((B, 0), F32), g.random(B).astype(F32))
        tokens.append(got[:, 0])
    token = np.stack(tokens, 1)
    got, accepted = check_verify(target, draft, token, None, g.random((B, G)).astype(F32), g.random(B).astype(F32), "chain")
    assert np.all(got[np.arange(B), accepted.astype(np.int64)] < n)
