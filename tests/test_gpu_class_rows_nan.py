"""Rows that hold NaN of either kind on the GPU: top-k never takes one and loses nothing beside it, and row_max of the
distillation entry points passes over it.

A quiet NaN is what arithmetic gives; a signalling one (the top mantissa bit clear) is what memory that was never
written, or a mask made of bits, can hold.  A hardware maximum treats the two differently, so both are looked at, at
every place of a thread's groups."""
import numpy as np
import pytest
import torch

import class_rows_ref as ref
from gpu_util import F32, call, dev, host
from test_gpu_class_rows import TYPES, got_u32, guarded, logits, slots, u32

pytestmark = pytest.mark.gpu

# bits of NaN: signalling of either sign, quiet
BITS = {"f32": (0x7F800001, 0xFF800001, 0x7FBFFFFF, 0x7FC00000), "bf16": (0x7F81, 0xFF81, 0x7FBF, 0x7FC0),
        "f16": (0x7C01, 0xFC01, 0x7DFF, 0x7E00)}
WORD = {"f32": (torch.int32, np.uint32, np.int32), "bf16": (torch.int16, np.uint16, np.int16), "f16": (torch.int16, np.uint16, np.int16)}


def with_nans(x, kind, where, bits):
    """x on the GPU in its type, with these bits where `where` is true (moved as whole numbers, so that nothing quiets them)."""
    word, unsigned, signed = WORD[kind]
    t = torch.from_numpy(np.ascontiguousarray(x)).to(TYPES[kind])
    b = t.view(word).numpy().view(unsigned).copy()
    b[where] = bits if np.isscalar(bits) else np.asarray(bits, unsigned)[where]
    return torch.from_numpy(b.view(signed)).cuda().view(TYPES[kind])


def check(kind, x, where, bits, want, k, what, norm=True):
    """`want` is what the plain form gives for k slots or more."""
    rows, n = x.shape
    xd = with_nans(x, kind, where, bits)
    value, check_v = guarded(rows * k)
    index, check_i = guarded(rows * k, torch.int32)
    log_norm, check_n = guarded(rows)
    call("anode_gpu_top_k_rows_" + kind, n, rows, 0, k, 1.0, xd, value, index, log_norm if norm else None)
    for c in (check_v, check_i, check_n):
        c(what)
    want_v, want_i = want[0][:, :k], want[1][:, :k]
    got_v, got_i = host(value).reshape(rows, k), got_u32(index).reshape(rows, k)
    bad = np.flatnonzero((got_i != want_i).any(1))
    assert bad.size == 0, (what, bad[:5], got_i[bad[:2]], want_i[bad[:2]])
    assert np.array_equal(got_v, want_v), what
    if norm:
        has = where.any(1)
        assert np.array_equal(np.isnan(host(log_norm)), has), what


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n", [24, 200, 1500, 9000, 20000, 50000, 70001])
def test_top_k_beside_one_nan(kind, n):
    # the row's largest values all before the NaN, all behind it, and round it, in one thread's groups and in others'
    g = np.random.default_rng(n)
    places = sorted({0, 1, 3, 4, 5, 7, 8, 11, n // 3, n // 2, n // 2 + 1, n - 9, n - 8, n - 3, n - 2, n - 1})
    rows = [(p, d) for p in places for d in (-12, 12)]
    x = logits(g, len(rows), n, kind)
    where = np.zeros(x.shape, bool)
    for r, (p, d) in enumerate(rows):
        lo, hi = sorted((p + d, p))
        x[r, max(0, lo):min(n, hi + 1)] = 30.0
        where[r, p] = True
    want = ref.top_k(np.where(where, np.nan, x).astype(F32), 300)
    for bits in BITS[kind]:
        for k in (1, 6, 40, 300):
            check(kind, x, where, bits, want, k, f"one NaN {bits:x} n={n} k={k}", norm=k != 6)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n", [500, 5000, 30011, 70001])
@pytest.mark.parametrize("share", [0.01, 0.3, 0.999, 1.0])
def test_top_k_among_many_nans(kind, n, share):
    g = np.random.default_rng(n)
    x = logits(g, 6, n, kind)
    x[4] = 0.25
    x[5] = -np.inf
    where = g.random(x.shape) < share
    bits = g.choice(np.array(BITS[kind], np.uint64), x.shape)
    want = ref.top_k(np.where(where, np.nan, x).astype(F32), 1000)
    for k in (1, 20, 64, 200, 256, 1000):
        check(kind, x, where, bits, want, k, f"many NaNs n={n} share={share} k={k}")


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n,rows", [(100, 4), (1000, 300), (3000, 1100), (9000, 8), (40000, 4), (140000, 3), (140000, 40)])
def test_distill_row_max_passes_over_nans(kind, n, rows):
    # loss, sum and gradient of such a row are NaN; its largest value is that of the numbers in it
    g = np.random.default_rng(n + rows)
    x = np.broadcast_to(logits(g, 4, n, kind)[None], (-(-rows // 4), 4, n)).reshape(-1, n)[:rows].copy()
    k = 5
    value, index = slots(g, rows, n, k, absent=0.0)
    where = np.zeros(x.shape, bool)
    for r in range(rows):
        if r % 4 == 3:
            continue                                   # a row without a NaN among them
        p = int(g.integers(0, n))
        if r % 4 == 2:
            where[r] = True                            # nothing but NaN and one number
            where[r, p] = False
        else:
            where[r, p] = True
            x[r, max(0, p - 9):p] = 30.0
            x[r, p + 1:p + 10] = 29.0 if r % 4 else 31.0
    want = np.where(where, -np.inf, x).max(1)
    has = where.any(1)
    for bits in BITS[kind]:
        for fused in (False, True):
            xd = with_nans(x, kind, where, bits)
            (loss, c0), (top, c1), (total, c2) = guarded(rows), guarded(rows), guarded(rows)
            if fused:
                dx = torch.zeros_like(xd)
                call("anode_gpu_softmax_distill_fused_fwd_bwd_rows_" + kind, n, rows, 0, k, 1.0, xd, dev(value), u32(index), None,
                     torch.ones(rows, device="cuda"), loss, top, total, dx)
                assert np.array_equal(torch.isnan(dx).all(1).cpu().numpy(), has) and np.array_equal(torch.isnan(dx).any(1).cpu().numpy(), has)
            else:
                call("anode_gpu_softmax_distill_rows_" + kind, n, rows, 0, k, 1.0, xd, dev(value), u32(index), None, loss, top, total)
            for c in (c0, c1, c2):
                c("distill")
            what = f"{kind} [{n}, {rows}] {bits:x} fused={fused}"
            bad = np.flatnonzero(host(top) != want)
            assert bad.size == 0, (what, bad[:4], host(top)[bad[:4]], want[bad[:4]])
            assert np.array_equal(np.isnan(host(loss)), has) and np.array_equal(np.isnan(host(total)), has), what


@pytest.mark.parametrize("kind", TYPES)
def test_top_k_beside_nans_of_large_arrays(kind):
    # more than the last cache holds: a thread's groups lie side by side there
    n, rows, k = 131071, 800 if kind != "f32" else 400, 64
    g = torch.Generator("cuda").manual_seed(5)
    x = torch.randn(rows, n, generator=g, device="cuda").mul_(3.0).to(TYPES[kind])
    seen = x.float().clone()                          # (float() of a float array is the array itself)
    word, unsigned, _ = WORD[kind]
    bits = x.view(word)
    place = torch.randint(100, n - 100, (rows,), generator=g, device="cuda")
    row = torch.arange(rows, device="cuda")
    for d in (-12, -5, -1, 1, 4, 12):                 # the largest values round the NaN
        seen[row, place + d] = 30.0 + d
    x.copy_(seen.to(TYPES[kind]))
    seen.copy_(x)
    for i, b in enumerate(BITS[kind]):
        at = row[i::len(BITS[kind]) + 1]              # (every fifth row has none)
        bits[at, place[at]] = torch.from_numpy(np.array([b], unsigned).view(WORD[kind][2])).cuda()
        seen[at, place[at]] = -float("inf")
    value, check_v = guarded(rows * k)
    index, check_i = guarded(rows * k, torch.int32)
    norm, check_n = guarded(rows)
    call("anode_gpu_top_k_rows_" + kind, n, rows, 0, k, 1.0, x, value, index, norm)
    for c in (check_v, check_i, check_n):
        c("large array with NaN")
    v, i = value.view(rows, k), index.view(rows, k)
    assert bool((v == torch.sort(seen, dim=1, descending=True)[0][:, :k]).all())
    assert bool((seen.gather(1, i.long()) == v).all())
    has = row % (len(BITS[kind]) + 1) < len(BITS[kind])
    assert bool((torch.isnan(norm) == has).all())
