"""Operators on rows of logits in 64 bits, row by row from their definitions, for the tests of gan_amd.logits."""
import math

import numpy as np

UNIT = 2.0 ** 36


def sample_row(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Places drawn from one row's valid logits (float64 array); -1 where nothing is left."""
    at = np.array([i for i in range(len(x)) if x[i] > -math.inf], dtype=np.int64)        # (NaN compares false)
    if len(at) == 0:
        return [-1] * len(u)
    at = at[np.lexsort((at, -x[at]))]
    temperature, top_p, min_p = (float(np.float32(v)) for v in (temperature, top_p, min_p))
    if not temperature > 0:
        return [int(at[d]) if d < len(at) else -1 for d in range(len(u))]
    same = x[at] == x[at[0]]
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(same, 1.0, np.exp((x[at] - x[at[0]]) / temperature))
    q = np.rint(np.where(np.isnan(w), 0.0, w) * UNIT)
    if top_k > 0:
        at, q = at[:top_k], q[:top_k]
    if top_p < 1:
        total, front, keep = math.fsum(q), 0.0, []
        for j in range(len(q)):
            if j and not front < top_p * total:
                break
            keep.append(j)
            front += q[j]
        at, q = at[keep], q[keep]
    if min_p > 0:
        stays = q >= min(min_p, 1.0) * UNIT
        at, q = at[stays], q[stays]
    at, q = at[q > 0], q[q > 0]
    order = np.argsort(at)
    at, q = list(at[order]), list(q[order])
    picks = []
    for v in u:
        if not at:
            picks.append(-1)
            continue
        v = 0.0 if math.isnan(v) else min(max(float(v), 0.0), 1.0 - 2.0 ** -24)
        t, upto, j = v * math.fsum(q), 0.0, 0
        while upto + q[j] <= t:
            upto += q[j]
            j += 1
        picks.append(int(at.pop(j)))
        q.pop(j)
    return picks


def top_row(x, m, temperature):
    at = np.array([i for i in range(len(x)) if x[i] > -math.inf], dtype=np.int64)
    order = at[np.lexsort((at, -x[at]))] if len(at) else at
    values, index = np.full(m, -np.inf), np.full(m, -1, dtype=np.int32)
    k = min(m, len(order))
    values[:k], index[:k] = x[order[:k]], order[:k]
    if not len(at):
        return values, index, -math.inf
    y = x[at] / temperature
    top = y.max()
    return values, index, top if math.isinf(top) else top + math.log(math.fsum(np.exp(y - top)))


def distill_row(x, values, index, lse, temperature, weight=1.0):
    """(loss, gradient, bound of the loss's error, bounds of the gradient's) of one row's valid logits.

    The bounds count the roundings of 32-bit arithmetic, each half a step (2^-24 of its result).  Y bounds the numbers
    that are subtracted (y, the log-sum-exps): a difference of two of them, each rounded up to three times, is off by at
    most 8 Y half steps, and an exponential of one relatively by as much (plus 16 for its own and for the sum it is
    divided by)."""
    n, h = len(x), 2.0 ** -24
    grad, none = np.zeros(n), np.zeros(n)
    named = [j for j in range(len(index)) if 0 <= index[j] < n and values[j] != -math.inf]
    if not named or not n or np.all(x == -math.inf):
        return 0.0, grad, 0.0, none
    y = x / temperature
    top = y.max()
    logz = top + math.log(math.fsum(np.exp(y - top)))
    t = np.array([values[j] for j in named]) / temperature
    at = np.array([index[j] for j in named])
    with_rest = lse is not None
    if not with_rest:
        lse = t.max() + math.log(math.fsum(np.exp(t - t.max())))
    lq = t - lse
    q = np.minimum(np.exp(lq), 1.0)
    listed = np.zeros(n, dtype=bool)
    listed[at] = True
    with np.errstate(invalid="ignore", over="ignore"):
        terms = np.where(q > 0, q * (lq - (y[at] - logz)), 0.0)
    loss = math.fsum(terms) if np.all(np.isfinite(terms)) else float(np.sum(terms))
    rest = ~listed & (x > -math.inf)
    full, rest_q, share = q.sum(), 0.0, np.zeros(n)
    finite = [abs(v) for v in (*y, *t, lse, logz) if math.isfinite(v)]
    big = max(finite)
    D = math.fsum(q * np.abs(np.where(np.isfinite(y[at]), lq - (y[at] - logz), 0.0)))
    if with_rest and rest.any():
        rest_q = max(1.0 - q.sum(), 0.0)
        full += rest_q
        if rest_q > 0:
            rtop = y[rest].max()
            log_rest = rtop + math.log(math.fsum(np.exp(y[rest] - rtop)))
            loss += rest_q * (math.log(rest_q) - (log_rest - logz))
            share[rest] = np.exp(y[rest] - log_rest)
            D += abs(math.log(rest_q)) + abs(log_rest - logz) + 1
    p = np.exp(y - logz)
    grad = p * full - share * rest_q
    sums = np.zeros(n)
    np.add.at(sums, at, q)
    grad -= sums
    step = h * (8 * big + 16)
    scale = weight * temperature
    loss_err = abs(scale) * temperature * step * (2 + 2 * D)
    grad_err = abs(scale) * (step * (2 * p * full + 2 * share * rest_q + sums + share) + len(named) * 2.0 ** -31)
    return scale * temperature * loss, scale * grad, loss_err, grad_err
