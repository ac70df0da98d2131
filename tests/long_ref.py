"""Plain 64-bit forms of the operators for long contexts and for judged drafts,
on the CPU, as their definitions read. Used by test_gpu_long*.py and
test_gpu_verify.py."""
import math

import numpy as np

BLOCK = 32


def key_order(D):
    """order[byte] = (position, value) of a block's keys."""
    a, c, g, i, s, e = np.indices((2, D // 64, 4, 16, 2, 8)).reshape(6, -1)
    return 16 * a + i, 64 * c + 32 * s + 8 * g + e


def value_order(D):
    c, g, i, s, a, e = np.indices((D // 32, 4, 16, 2, 2, 4)).reshape(6, -1)
    return 16 * a + 4 * g + e, 32 * c + 16 * s + i


def to_bytes(n, order):
    """Integers [..., 32, D] in a block's order."""
    p, d = order(n.shape[-1])
    return n[..., p, d].astype(np.int8)


def from_bytes(b, order):
    D = b.shape[-1] // BLOCK
    p, d = order(D)
    out = np.empty(b.shape[:-1] + (BLOCK, D), np.int8)
    out[..., p, d] = b
    return out


def quantise(x):
    """fp16 blocks [..., 32, D]: (integers, scales)."""
    x = x.astype(np.float32)
    with np.errstate(invalid="ignore"):
        top = np.abs(x).max((-1, -2))
        s = (top / np.float32(127)).astype(np.float32)
        fine = np.isfinite(x).all((-1, -2))
        n = np.rint(x / np.where(s > 0, s, 1)[..., None, None])
    n = np.where(fine[..., None, None], n, 0).astype(np.int64)
    return n, np.where(fine, s, np.nan).astype(np.float32)


def fills(cached, packed, max_seq, blocks):
    """Blocks that a sequence's lengths let be packed."""
    if not 0 <= cached <= max_seq or packed < 0 or packed % BLOCK or packed // BLOCK + cached // BLOCK > blocks:
        return 0
    return cached // BLOCK


def pack(k, v, k8, v8, ks, vs, cached, packed):
    """kv_pack on numpy arrays, in place (k, v fp16 [B, H, S, D])."""
    for b, (n, at) in enumerate(zip(cached, packed)):
        whole = fills(n, at, k.shape[2], k8.shape[2])
        for x, x8, s, order in ((k, k8, ks, key_order), (v, v8, vs, value_order)):
            for j in range(whole):
                q, sc = quantise(x[b, :, j * BLOCK:(j + 1) * BLOCK])
                x8[b, :, at // BLOCK + j], s[b, :, at // BLOCK + j] = to_bytes(q, order), sc
            if whole:
                x[b, :, :n - whole * BLOCK] = x[b, :, whole * BLOCK:n].copy()


def seen_by(t, n, before, mask_row, window, sinks):
    """Positions that row t of n sees, behind `before` cached ones."""
    out = list(range(before))
    for i in range(n):
        if (mask_row is None and i <= t) or (mask_row is not None and i < 64 * len(mask_row)
                                             and int(mask_row[i // 64]) >> (i % 64) & 1):
            out.append(before + i)
    if not window:
        return out
    return [j for r, j in enumerate(out) if r < sinks or r >= len(out) - window]


def attention_tolerance(absv, qk, D, keys, half, vmax):
    """rows_ref.attention_tolerance with what 8-bit blocks add: the product of
    the score's factor with the block's scale (2^-22 of the score, and once more
    where the largest is taken), the probability's with the value's (2^-23), and
    the least that a weight is held to, 2^-31 of the largest times the largest
    value of the blocks, for every key."""
    ds = qk * (D * 2.0 ** -23 + (0 if half else 2.0 ** -21) + 2.0 ** -21) + 2.0 ** -22
    rel = 2 * ds + (keys + 16) * 2.0 ** -23 + (2.0 ** -10 if half else 2.0 ** -21) + 2.0 ** -23
    return absv * rel[:, None] * 1.01 + keys * vmax * 2.0 ** -31 + (absv * 2.0 ** -11 + 2.0 ** -25 if half else 1e-30)


# ------------------------------------------------------------------- drafts
def _first_over(w, u):
    s = np.cumsum(w)
    over = np.nonzero((s > u * s[-1]) & (w > 0))[0]
    return int(over[0]) if len(over) else int(np.nonzero(w > 0)[0][-1])


def verify(x, tokens, parents, row_start, accept_u, sample_u, max_rows, draft=None, temperature=1.0):
    """(accepted, path, next) by following each path row by row."""
    B, V = len(row_start) - 1, x.shape[1]
    accepted, nxt = np.zeros(B, np.int64), np.full(B, -1)
    path = np.full((B, max_rows), -1)
    for b in range(B):
        s, n = int(row_start[b]), min(int(row_start[b + 1]) - int(row_start[b]), max_rows)
        at = 0 if n > 0 else -1
        while at >= 0:
            path[b, accepted[b]] = at
            accepted[b] += 1
            row = x[s + at].astype(np.float64)
            nxt[b] = -1
            if np.isnan(row).any() or not np.isfinite(row.max()):
                break
            with np.errstate(under="ignore"):
                p = np.exp((row - row.max()) / temperature)
            p /= p.sum()
            kids = [t for t in range(at + 1, n) if parents[s + t] == at]
            go = -1
            if draft is None:
                nxt[b] = _first_over(p, float(sample_u[s + at]))
                go = next((t for t in kids if tokens[s + t] == nxt[b]), -1)
            else:
                with np.errstate(invalid="ignore"):
                    q = np.where(draft[s + at] > 0, draft[s + at], 0).astype(np.float64)
                c, w = 0.0, p
                for t in kids:
                    k = int(tokens[s + t])
                    if not 0 <= k < V:
                        continue
                    z = w.sum()
                    if float(accept_u[s + t]) * q[k] * z < w[k]:
                        go = t
                        break
                    c += z
                    w = np.maximum(p - c * q, 0)
                if go < 0:
                    nxt[b] = _first_over(w if w.sum() > 0 else p, float(sample_u[s + at]))
            at = go
    return accepted, path, nxt


def within(got, want, tol, what):
    off = np.abs(got.astype(np.float64) - want)
    bad = ~(off <= tol)
    if bad.any():
        at = tuple(np.argwhere(bad)[0])
        raise AssertionError(f"{what}: {bad.sum()} of {bad.size} off, first at {at}: {got[at]} for {want[at]}, tolerance "
                             f"{tol[at] if np.ndim(tol) else tol}")


__all__ = [n for n in dir() if not n.startswith("_") and n not in ("math", "np")]
