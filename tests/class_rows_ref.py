"""Plain 64-bit implementations of the operators over rows of many classes, and the error bounds of their 32-bit
kernels.  Arrays are numpy; logits come as the float32 values that the element type holds."""
import numpy as np

NONE = 0xFFFFFFFF
U = 2.0 ** -24  # half a step of fp32, relative


def top_k(x, k):
    """x [rows, classes] -> value float32 [rows, k], index uint32 [rows, k]."""
    rows, n = x.shape
    value = np.full((rows, k), -np.inf, np.float32)
    index = np.full((rows, k), NONE, np.uint32)
    for r in range(rows):
        ok = np.flatnonzero(x[r] > -np.inf)  # NaN compares false
        order = ok[np.argsort(-x[r, ok].astype(np.float64), kind="stable")][:k]
        value[r, :order.size] = x[r, order]
        index[r, :order.size] = order
    return value, index


def stats(x, t):
    """row_max, row_sum in 64 bits; -inf rows give (-inf, 0), NaN and +inf a NaN sum."""
    rows, n = x.shape
    top = np.full(rows, -np.inf)
    total = np.zeros(rows)
    for r in range(rows):
        v = x[r].astype(np.float64)
        seen = v[~np.isnan(v)]
        if seen.size:
            top[r] = seen.max()
        if np.isnan(v).any() or top[r] == np.inf:
            total[r] = np.nan
        elif top[r] > -np.inf:
            total[r] = np.exp((v - top[r]) / t).sum()
    return top, total


def sum_bound(x, t, lanes=256, width=4):
    """Relative error bound of a row's 32-bit sum of exponentials.

    A term exp2((x - m) c): the difference, c and the product are rounded once each (three half steps of |a| = |x - m|
    / t log2 e, which the exponential turns into 3 ln 2 |a| u), the hardware exponential is off by at most a step (2 u).
    The mean of |a| over the weights bounds the first part.  A thread adds its groups in turn (a group's `width` terms,
    then the group to the running sum), rescales it when the maximum moves (five half steps each time, counted for
    every group: a rescale is an exponential of its own), and the merge of wave and workgroup has at most 6 + 16
    levels of five half steps."""
    v = x.astype(np.float64)
    v = v[v > -np.inf]
    if v.size == 0 or not np.isfinite(v).all():
        return 0.0
    a = (v.max() - v) / t * 1.4426950408889634
    w = np.exp2(-a)
    groups = -(-x.size // (lanes * 4)) + 1
    return U * (2 + 3 * np.log(2) * float((a * w).sum() / w.sum()) + (1 + 5) * groups + 8 + 5 * 22)


def teacher(value, index, n, t, log_norm=None):
    """p [rows, k] in 64 bits; log p; which slots count."""
    value, index = value.astype(np.float64), index.astype(np.int64)
    there = (index < n) & (value > -np.inf)
    p = np.zeros(value.shape)
    log_p = np.full(value.shape, -np.inf)
    for r in range(value.shape[0]):
        ok = there[r]
        if not ok.any():
            continue
        z = value[r, ok] / t
        if log_norm is None:
            z = z - z.max()
            z = z - np.log(np.exp(z).sum())
        else:
            z = z - np.float64(log_norm[r])
        log_p[r, ok] = z
        p[r, ok] = np.exp(z)
    return p, log_p, there


def distill(x, value, index, t, log_norm=None):
    rows, n = x.shape
    top, total = stats(x, t)
    p, log_p, there = teacher(value, index, n, t, log_norm)
    loss = np.zeros(rows)
    with np.errstate(all="ignore"):
        for r in range(rows):
            for j in np.flatnonzero(there[r]):
                if p[r, j] == 0.0:
                    continue
                log_q = (np.float64(x[r, index[r, j]]) - top[r]) / t - np.log(total[r])
                loss[r] += p[r, j] * (log_p[r, j] - log_q)
    return loss, top, total


def distill_grad(x, value, index, t, dy, log_norm=None):
    """dx in 64 bits, q in 64 bits, p summed by class."""
    rows, n = x.shape
    top, total = stats(x, t)
    p, _, there = teacher(value, index, n, t, log_norm)
    dx = np.zeros((rows, n))
    q = np.zeros((rows, n))
    with np.errstate(all="ignore"):
        for r in range(rows):
            if not there[r].any():
                continue
            q[r] = np.exp((x[r].astype(np.float64) - top[r]) / t) / total[r]
            mass = 1.0 if log_norm is None else p[r].sum()
            g = mass * q[r]
            np.subtract.at(g, index[r, there[r]].astype(np.int64), p[r, there[r]])
            dx[r] = float(dy[r]) / t * g
    return dx, q, p


def verify(target, draft, token, length, accept, pick):
    """target [B, G + 1, n] float32, draft [B, G, n] or None, token [B, G], length [B] or None -> token [B, G + 1], accepted [B]."""
    B, G1, n = target.shape
    G = G1 - 1
    out = np.full((B, G1), NONE, np.uint32)
    accepted = np.zeros(B, np.uint32)
    for b in range(B):
        most = G if length is None else min(int(length[b]), G)
        i = 0
        while i < most:
            d = int(token[b, i])
            if d >= n:
                break
            q = 1.0 if draft is None else float(draft[b, i, d])
            if not float(accept[b, i]) * q < float(target[b, i, d]):
                break
            out[b, i] = d
            i += 1
        accepted[b] = i
        w = target[b, i].astype(np.float64)
        if i < most:
            rest = w.copy()
            if draft is None:
                if int(token[b, i]) < n:
                    rest[int(token[b, i])] = 0.0
            else:
                rest = rest - draft[b, i].astype(np.float64)
            if (rest > 0).any():
                w = rest
        w = np.where(w > 0, w, 0.0)
        if not (w > 0).any():
            continue
        upto = np.cumsum(w)
        with np.errstate(all="ignore"):
            over = np.flatnonzero((upto > float(pick[b]) * upto[-1]) & (w > 0))
        out[b, i] = over[0] if over.size else np.flatnonzero(w > 0)[-1]
    return out, accepted
