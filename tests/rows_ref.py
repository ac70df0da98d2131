"""Plain 64-bit forms of the operators for rows of tokens, on the CPU, row by
row as their definitions read. Used by test_gpu_rows*.py."""
import math

import numpy as np

EPS32 = 2.0 ** -24  # half a step of fp32, relative


def plan(parents, row_start, cache_len, max_seq, max_rows, words, delta=None):
    rows = len(parents)
    mask = np.zeros((rows, words), np.uint64)
    pos, slots = np.full(rows, -1, np.int64), np.full(rows, -1, np.int64)
    for b in range(len(cache_len)):
        s, e = row_start[b], row_start[b + 1]
        sets = []
        for t in range(e - s):
            p = int(parents[s + t])
            good = -1 <= p < t and t < max_rows and (p < 0 or sets[p] is not None)
            sets.append((set() if p < 0 else sets[p]) | {t} if good else None)
            at = int(cache_len[b]) + t
            base = int(cache_len[b]) + (int(delta[b]) if delta is not None else 0)
            if sets[t] is None or cache_len[b] < 0 or at >= max_seq or not 0 <= base + len(sets[t]) - 1 < 2 ** 31:
                pos[s + t] = -2
                continue
            pos[s + t] = base + len(sets[t]) - 1
            slots[s + t] = b * max_seq + at
            for j in sets[t]:
                mask[s + t, j // 64] |= np.uint64(1) << np.uint64(j % 64)
    return mask, pos, slots


def axis_of(half, sections, interleaved):
    if sections is None:
        return [0] * half
    if not interleaved:
        return [0] * sections[0] + [1] * sections[1] + [2] * sections[2]
    out = [0] * half
    for a in (1, 2):
        for n in range(sections[a]):
            out[3 * n + a] = a
    return out


def norm_rope(x, w, s, gs, eps, cos, sin, pos, axis):
    """x [heads, D] of one row at positions pos (one per axis): the result, and
    the sum of its two terms' sizes, which a tolerance is made of."""
    x = x.astype(np.float64)
    D = x.shape[1]
    y = x / np.sqrt((x * x).mean(1, keepdims=True) + np.float64(np.float32(eps))) * (w.astype(np.float64) * np.repeat(s, gs))
    c = np.array([cos[pos[axis[i]], i] for i in range(D // 2)], np.float64)
    n = np.array([sin[pos[axis[i]], i] for i in range(D // 2)], np.float64)
    a, b = y[:, :D // 2], y[:, D // 2:]
    return (np.concatenate([a * c - b * n, b * c + a * n], 1),
            np.concatenate([np.abs(a * c) + np.abs(b * n), np.abs(b * c) + np.abs(a * n)], 1))


def seen_by(t, n, length, mask_row):
    """Positions that row t of n sees."""
    out = list(range(length))
    for i in range(n):
        if (mask_row is None and i <= t) or (mask_row is not None and i < 64 * len(mask_row)
                                             and int(mask_row[i // 64]) >> (i % 64) & 1):
            out.append(length + i)
    return out


def attention(q, k, v, seen, scale):
    """q [heads, D] over k, v [kv_heads, S, D]: (out, and sum p |v| and the
    largest scale * sum |q k|, which the tolerances are made of)."""
    H, D = q.shape
    g = H // k.shape[0]
    out, absv, qk = np.zeros((H, D)), np.zeros((H, D)), np.zeros(H)
    if not seen:
        return out, absv, qk
    q = q.astype(np.float64)
    with np.errstate(all="ignore"):
        for h in range(H):
            kk, vv = k[h // g][seen].astype(np.float64), v[h // g][seen].astype(np.float64)
            s = scale * (kk @ q[h])
            p = np.exp(s - s.max())
            p /= p.sum()
            out[h], absv[h] = p @ vv, p @ np.abs(vv)
            qk[h] = abs(scale) * (np.abs(kk) @ np.abs(q[h])).max()
    return out, absv, qk


def attention_tolerance(absv, qk, D, keys, half):
    """Bound of |computed - exact| for each output, to first order.

    Scores: a D-term fp32 sum of exact products is off by at most (D - 1) 2^-23
    sum |q k| (half a step a term, doubled for adders that truncate); fp32
    queries are two fp16 terms, off by 2^-21. Scaling and the exponent add 2^-23
    of the score each and 2^-22 of 2^x. p then is off by twice the score's
    error, relatively (it and the sum it is divided by). Sums over the keys:
    keys 2^-23; p as two fp16 terms 2^-21, as one 2^-10 (rounded either way,
    against a sum of the unrounded). fp16 outputs: half a step, 2^-11."""
    ds = qk * (D * 2.0 ** -23 + (0 if half else 2.0 ** -21) + 2.0 ** -22) + 2.0 ** -22
    rel = 2 * ds + (keys + 16) * 2.0 ** -23 + (2.0 ** -10 if half else 2.0 ** -21)
    return absv * rel[:, None] * 1.01 + (absv * 2.0 ** -11 + 2.0 ** -25 if half else 1e-30)


def logprobs(x, token, k):
    """(logprob, rank, entropy, ids, top logprobs) of one row."""
    x = x.astype(np.float64)
    V = x.size
    key = np.where(np.isnan(x), -np.inf, x)
    order = np.lexsort((np.arange(V), -key))
    ids = order[:k]
    m = key.max()
    bad = np.isnan(x).any() or not np.isfinite(m)
    if bad:
        logs = lp = np.full(V, np.nan)
        ent = math.nan
    else:
        e = np.exp(x - m)
        rest = e.copy()
        rest[order[0]] = 0
        logs = np.log1p(rest.sum())
        lp = (x - m) - logs
        with np.errstate(invalid="ignore"):
            ent = logs - np.where(e > 0, e * (x - m), 0).sum() / e.sum()
    if not 0 <= token < V:
        return math.nan, -1, ent, ids, lp[ids]
    rank = int((key > key[token]).sum() + (key[:token] == key[token]).sum())
    return lp[token], rank, ent, ids, lp[ids]
