"""GPU tests of attention over 8-bit blocks whose value scales lie far apart,
against 64 bits: what a row does not see, or sees with next to no weight, costs
the rest of it no bits.

A weight p vs is held to 2^-31 of the largest p |vs| that its row sees, a fp16
row's p to 2^-31 of the largest p; each key's integer is at most 127."""
import numpy as np
import pytest

import long_ref as ref
import rows_ref
from long_ref import within
from test_gpu_long import HALF, Long

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def tolerance(P, scales, rows_v, absv, qk, D, keys, half):
    """Of one row [H, D]: long_ref.attention_tolerance, the least that a weight is
    held to taken from what the row sees: P [H, keys] its probabilities, scales
    [H, keys] |vs| (0 for fp16 rows), rows_v [H] the largest |v| of fp16 rows."""
    ds = qk * (D * 2.0 ** -23 + (0 if half else 2.0 ** -21) + 2.0 ** -21) + 2.0 ** -22
    rel = 2 * ds + (keys + 16) * 2.0 ** -23 + (2.0 ** -10 if half else 2.0 ** -21) + 2.0 ** -23
    least = 127 * (P * scales).max(1) + P.max(1) * rows_v  # of the packed ones and of the others
    return absv * rel[:, None] * 1.01 + keys * 1.01 * 2.0 ** -31 * least[:, None] + (absv * 2.0 ** -11 + 2.0 ** -25 if half else 1e-30)


def check(B, got):
    g = B.H // B.Hk
    for b, n in enumerate(B.rows):
        k, v, p = B.positions(b)
        vs = np.concatenate([np.repeat(np.abs(B.vs[b].astype(np.float64)), 32, 1)[:, :p], np.zeros((B.Hk, B.S))], 1)
        for t in range(n):
            r = int(B.st[b]) + t
            seen = ref.seen_by(t, n, p + B.lens[b], None if B.mask is None else B.mask[r], B.window, B.sinks)
            want, absv, qk = rows_ref.attention(B.q[r].reshape(B.H, B.D), k, v, seen, B.D ** -0.5)
            P, sc, rv = np.zeros((B.H, len(seen))), np.zeros((B.H, len(seen))), np.zeros(B.H)
            for h in range(B.H):
                s = B.D ** -0.5 * (k[h // g][seen] @ B.q[r].reshape(B.H, B.D)[h].astype(np.float64))
                e = np.exp(s - s.max())
                P[h], sc[h] = e / e.sum(), vs[h // g][seen]
                rv[h] = np.abs(v[h // g][[j for j in seen if j >= p]]).max(initial=0.0)
            within(got[r].reshape(B.H, B.D), want, tolerance(P, sc, rv, absv, qk, B.D, len(seen), B.half), f"seq {b} row {t}")


RATIOS = pytest.mark.parametrize("ratio", [10, 20, 30])
ROWS = pytest.mark.parametrize("T", [1, 6, 80])


def small(B, level):
    """Value scales of one size everywhere, and fp16 rows to match."""
    B.vs[:] = (2.0 ** level * (1 + B.rng.random(B.vs.shape))).astype(np.float32)
    B.v[:] = (B.v.astype(np.float64) * 127 * 2.0 ** level).astype(np.float16)


@HALF
@ROWS
@RATIOS
def test_unseen_blocks_of_large_scales(T, half, ratio):
    """Beside the first positions, and before the window in its first turn."""
    for D in (64, 128):
        B = Long(T + ratio, [T, 2], [4, 9], [960, 640], 4, 2, D, half, T == 6, window=200, sinks=4)
        small(B, -8 if half else -18)
        for b, p in enumerate(B.packed):
            first = (p + B.lens[b] + 1 - 200) // 32  # that a window may reach
            B.vs[b, :, 1:first - 1] *= np.float32(2.0 ** ratio)
        check(B, B.run())


@HALF
@ROWS
@RATIOS
def test_seen_blocks_of_large_scales_and_no_weight(T, half, ratio):
    """One block, early, in the middle or last, whose positions all score 40 less
    (as powers of e) than the others could."""
    for block in (0, 7, 15):
        B = Long(T + ratio + block, [T], [5], [512], 4, 2, 64, half, False)
        small(B, -8 if half else -18)
        q = B.q.reshape(-1, B.H, B.D)
        q[:] *= 0.25
        q[..., 3] = 8.0
        B.kn[..., 3], B.k[..., 3] = 0, 0
        B.kn[:, :, block] = 0
        B.kn[:, :, block, :, 3] = -100
        B.ks[:, :, block] = 0.4  # a score of -100 0.4 8 / 8
        B.vs[:, :, block] *= np.float32(2.0 ** ratio)
        check(B, B.run())


@HALF
@ROWS
@pytest.mark.parametrize("way", ["falling", "rising", "any"])
def test_scales_against_scores(T, half, way):
    """Scores that rise block by block while the scales fall, so that weights stay
    alike; the reverse; and both at random."""
    B = Long(T + len(way), [T, 1], [7, 3], [640, 320], 4, 2, 128, half, False)
    n = B.vs.shape[2]
    step = np.arange(n) if way == "falling" else np.arange(n)[::-1] if way == "rising" else B.rng.integers(0, n, n)
    q = B.q.reshape(-1, B.H, B.D)
    q[:] *= 0.25
    q[..., 3] = 4.0
    B.k[..., 3] = 0
    for j in range(n):  # 1.5 a step: 2^2.2
        B.kn[:, :, j] = B.rng.integers(-30, 31, B.kn[:, :, j].shape)
        B.kn[:, :, j, :, 3] = 100
        B.ks[:, :, j] = 1.5 * step[j] * 128 ** 0.5 / 4 / 100
        B.vs[:, :, j] = 2.0 ** ((-8 if half else -18) + 2.2 * (n - step[j]) / (2 if half else 1)) * (1 + B.rng.random(B.vs[:, :, j].shape))
    B.v[:] = (B.v.astype(np.float64) * 0.5).astype(np.float16)
    check(B, B.run())


@pytest.mark.parametrize("T", [1, 80])
def test_scales_at_the_ends_of_their_type(T):
    """Blocks that a caller wrote: scales of 2^-120 beside ones of 2^100 that no
    row sees, zeros, and scales below the normal numbers."""
    for level in (-120, -60, 60):
        B = Long(T, [T], [0], [320], 4, 2, 64, False, False, window=100, sinks=3)
        B.vs[:] = (2.0 ** level * (1 + B.rng.random(B.vs.shape))).astype(np.float32)
        B.v[:] = 0
        B.vs[:, :, 1:4] = 2.0 ** 100
        B.vs[:, :, 8] = 0.0 if level < 0 else 2.0 ** -140
        check(B, B.run())
