"""Plain implementations in 64 bits of the operators over rows of logits, and their tolerances."""
from __future__ import annotations

import numpy as np

NAN, INF = float("nan"), float("inf")


def ref_top_k(x: np.ndarray, k: int, temperature: float = 1.0):
    """(indices, lse): larger first, NaN last, equal values by ascending index."""
    x = x.astype(np.float64)
    nan = np.isnan(x)
    clean = np.where(nan, 0.0, x)
    place = np.broadcast_to(np.arange(x.shape[1]), x.shape)
    order = np.lexsort((place, -clean, nan), axis=1)[:, :k]
    with np.errstate(all="ignore"):
        m = x.max(axis=1, keepdims=True, initial=-INF)
        safe = np.where(np.isfinite(m), m, 0.0)
        lse = np.log(np.exp((x - safe) / temperature).sum(axis=1)) + safe[:, 0] / temperature
    lse = np.where(nan.any(1), NAN, lse)
    return order.astype(np.int32), lse


def lse_error(n: int) -> float:
    """Bound on the absolute error of a row's log-sum-exp in fp32.  The sum of n terms is taken by 256
    threads or more, in order, so it is off by at most n / 256 half steps (2^-24 each) and those of
    the few merges; every term is off by one step of exp2 (2^-23) and by what its argument a is
    off, 2^-24 |a| ln 2 twice (the constant, the product): below 40 half steps for |a| < 28, and terms beyond
    weigh less than 2^-28."""
    return (n / 256 + 60) * 2.0 ** -24


def ref_distill(z, t, idx, temperature, scale, t_lse=None, row_grad=None):
    """(loss, gradient, probabilities q, teacher mass) in 64 bits."""
    z, t = z.astype(np.float64), t.astype(np.float64)
    rows, n = z.shape
    with np.errstate(all="ignore"):
        m = z.max(axis=1, keepdims=True, initial=-INF)
        safe = np.where(np.isfinite(m), m, 0.0)
        e = np.exp((z - safe) / temperature)
        s = e.sum(axis=1, keepdims=True)
        q = np.where(s == 0, 0.0, e / np.where(s == 0, 1.0, s))
        log_q = (z - safe) / temperature - np.log(s)
    loss, grad, mass = np.zeros(rows), np.zeros(z.shape), np.zeros(rows)
    for i in range(rows):
        used = [j for j in range(t.shape[1]) if 0 <= idx[i, j] < n]
        if not used:
            continue
        y = t[i, used] / temperature
        with np.errstate(all="ignore"):
            top = y.max()
            norm = (np.log(np.exp(y - (top if np.isfinite(top) else 0.0)).sum()) + (top if np.isfinite(top) else 0.0)
                    if t_lse is None else float(t_lse[i]))
            p = np.exp(y - norm) if norm != -INF else np.zeros(len(used))
        for pj, yj, v in zip(p, y, idx[i, used]):
            if pj != 0:
                loss[i] += pj * (yj - norm - log_q[i, v])
        mass[i] = p.sum()
        if mass[i] == 0:
            continue
        d = mass[i] * q[i]
        if np.isnan(s[i, 0]):
            d = np.full(n, NAN)
            loss[i] = NAN
        for pj, v in zip(p, idx[i, used]):
            d[v] -= pj
        grad[i] = d * (scale / temperature) * (1.0 if row_grad is None else float(row_grad[i]))
    return loss * scale, grad, q, mass


def weight_step(n: int) -> float:
    """What the weights of a row of n logits are whole multiples of, where the largest is 1."""
    return 2.0 ** -min(50, 62 - max(0, n - 1).bit_length())


def ref_sample(x, u, temperature=None, top_k=None, top_p=None, min_p=None, allowed=None):
    """(token, logprob, the token's weight beside the largest) of every row in 64 bits; allowed: a
    matrix of truth values."""
    x = x.astype(np.longdouble)
    tokens, logprobs, weights = [], [], []
    least = weight_step(x.shape[1]) / 2
    for i, row in enumerate(x):
        ok = row > -INF
        if allowed is not None:
            ok &= allowed[i]
        where = np.flatnonzero(ok)
        if len(where) == 0:
            tokens.append(-1)
            logprobs.append(-INF)
            weights.append(1.0)
            continue
        t = 1.0 if temperature is None else float(temperature[i])
        greedy = not t > 0
        rank = where[np.lexsort((where, -row[where]))]
        m = row[rank[0]]
        with np.errstate(all="ignore"):
            w = np.where(row[rank] == m, np.longdouble(1),
                         np.exp((row[rank] - m) / np.longdouble(1.0 if greedy else t)))
        w = np.where(w >= least, w, 0)  # NaN (an infinity over an infinity) is nothing, too
        limit = 1 if greedy else (0 if top_k is None else int(top_k[i]))
        if limit > 0:
            w, rank = w[:limit], rank[:limit]
        p = 1.0 if greedy or top_p is None else float(top_p[i])
        if p < 1:
            before = np.cumsum(w) - w
            keep = before < np.longdouble(p) * w.sum()
            keep[0] = True
            w, rank = w[keep], rank[keep]
        lo = 0.0 if greedy or min_p is None else float(min_p[i])
        if lo > 0:
            keep = w >= min(lo, 1.0)
            w, rank = w[keep], rank[keep]
        order = np.argsort(rank)
        w, rank = w[order], rank[order]
        c = np.cumsum(w)
        ui = float(u[i])
        goal = (ui if ui > 0 else 0.0) * c[-1]
        at = int(np.searchsorted(c, goal, side="right"))
        at = min(at, int(np.flatnonzero(w > 0)[-1]))
        tokens.append(int(rank[at]))
        logprobs.append(float(np.log(w[at] / c[-1])))
        weights.append(float(w[at]))
    return np.array(tokens, dtype=np.int32), np.array(logprobs), np.array(weights)


def pack_bits(allowed: np.ndarray) -> np.ndarray:
    """Truth values [rows, n] as 32-bit words, token v in bit v % 32 of word v // 32."""
    rows, n = allowed.shape
    words = (n + 31) // 32
    bits = np.zeros((rows, words * 32), dtype=np.uint64)
    bits[:, :n] = allowed
    return (bits.reshape(rows, words, 32) << np.arange(32, dtype=np.uint64)).sum(axis=2).astype(np.uint32).view(np.int32)
