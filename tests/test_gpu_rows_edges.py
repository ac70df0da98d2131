"""GPU tests of the operators for rows of tokens at calls that the other files
leave out: many query heads of one kv head, large batches, wide cache rows,
infinite scores, very long rows of logits."""
import math

import numpy as np
import pytest

import rows_ref as ref
from test_gpu_rows import Batch, dev, i32, qa, q, within

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("half", [False, True], ids=["fp32", "fp16"])
@pytest.mark.parametrize("H,Hk,D,T", [(64, 1, 128, 1), (33, 1, 64, 1), (33, 1, 64, 2), (28, 4, 128, 3), (128, 1, 64, 5)], ids=str)
def test_many_heads_of_one_kv_head(H, Hk, D, T, half):
    """A token's query heads fill one tile, or pass it."""
    for lens in ([0, 70, 1], [2500, 9, 64]):
        B = Batch(H + T, [T, T, 1], lens, H, Hk, D, half, T > 1, pad=1)
        B.check(B.run())


@pytest.mark.parametrize("T", [1, 3])
def test_large_batches(T):
    """More sequences than the chip has places, many of them without rows."""
    rng = np.random.default_rng(T)
    rows = [int(n) for n in rng.integers(0, T + 1, 900)]
    rows[5] = T
    B = Batch(T, rows, [int(n) for n in rng.integers(0, 90, 900)], 4, 2, 64, False, T > 1, pad=2)
    B.check(B.run(), only=lambda b, t: b % 7 == 0 or b > 890)


def test_long_prompts():
    """Many tiles of one sequence, behind nothing and behind a cache."""
    for half in (False, True):
        B = Batch(3 + half, [2500], [700 * half], 4, 2, 64, half, False)
        B.check(B.run(), only=lambda b, t: t % 311 == 0 or t > 2495 or t in (31, 32, 63, 64, 127, 128))


@pytest.mark.parametrize("rows,lens", [([1, 1], [300, 77]), ([50, 2], [300, 77])], ids=str)
def test_wide_cache_rows(rows, lens):
    """Cache rows far apart in memory (2^16 values), NaN between them."""
    B = Batch(8, rows, lens, 4, 2, 128, False, True)
    want = B.run()
    B.check(want)
    wide = []
    for c in (B.k, B.v):
        t = torch.full((B.S, 2, 2, 16384), math.nan, dtype=torch.float16, device="cuda").permute(1, 2, 0, 3)[..., :128]
        t.copy_(dev(c))
        wide.append(t)
    np.testing.assert_array_equal(B.run(cache=qa.KVCache(*wide)), want)


@pytest.mark.parametrize("half", [False, True], ids=["fp32", "fp16"])
@pytest.mark.parametrize("T", [1, 40])
def test_infinite_keys(T, half):
    """A seen key of -inf has no weight where the query is positive there, and
    leaves nothing to compute where it is negative (a score of +inf)."""
    B = Batch(T, [T], [500], 4, 2, 128, half, False)
    B.k[0, :, 100, 3] = -np.inf
    B.q[:, 3::256] = np.abs(B.q[:, 3::256]) + np.asarray(0.5, B.q.dtype)
    B.q[:, 131::256] = -np.abs(B.q[:, 131::256]) - np.asarray(0.5, B.q.dtype)
    got = B.run()
    for t in {0, T // 2, T - 1}:
        g = got[t].reshape(4, 128)
        assert np.isnan(g[1::2]).all()
        seen = [j for j in range(500 + t + 1) if j != 100]
        want, absv, qk = ref.attention(B.q[t].reshape(4, 128), B.k[0], B.v[0], seen, 128 ** -0.5)
        tol = ref.attention_tolerance(absv, qk, 128, len(seen), half)
        within(g[0::2], want[0::2], tol[0::2], f"row {t}")


def test_half_queries_at_their_end():
    """fp16 queries of up to 6e4: one key takes all."""
    B = Batch(2, [5, 40], [100, 64], 4, 2, 64, True, True, qscale=1.0)
    B.q = (B.q.astype(np.float32) / np.abs(B.q).max() * 60000).astype(np.float16)
    got = B.run()
    for b, n in enumerate(B.rows):
        for t in range(n):
            r = int(B.st[b]) + t
            seen = ref.seen_by(t, n, B.lens[b], B.mask[r])
            for h in range(4):
                s = B.k[b, h // 2][seen].astype(np.float64) @ B.q[r, h * 64:(h + 1) * 64].astype(np.float64)
                first, second = np.sort(s)[::-1][:2] if len(s) > 1 else (s[0], -np.inf)
                if (first - second) / 8 > 20:  # e^-20 is below fp16's steps
                    np.testing.assert_allclose(got[r, h * 64:(h + 1) * 64], B.v[b, h // 2, seen[int(np.argmax(s))]], rtol=2.0 ** -10, atol=2.0 ** -20)


@pytest.mark.parametrize("V,half", [(5_000_003, False), (300_000_001, True)], ids=str)
def test_very_long_rows(V, half):
    """Rows of logits with more parts than a joining wave has lanes, and of
    more than 2^28 values."""
    x = torch.empty((1, V + 9), dtype=torch.float16 if half else torch.float32, device="cuda")
    x.normal_(0, 2, generator=torch.Generator(device="cuda").manual_seed(1))
    x = x[:, 1:V + 1]
    at = [V - 1, 0, V // 2, 12345]
    for n, i in enumerate(at):
        x[0, i] = 18.0 - n
    r = q.token_logprobs(x, i32([V // 2]), top_k=4)
    assert r.top_ids[0].tolist() == at and int(r.rank[0]) == 2
    s = t = 0.0
    for c in x[0].split(1 << 24):
        d = c.double() - 18.0
        e = d.exp()
        s, t = s + float(e.sum()), t + float((e * d).sum())
    # exponents and weights 21 2^-23 as elsewhere; a lane adds at most V / 16384
    # values in order (256 blocks of 256 lanes over 8 registers), half a step each
    e = 21 * 2.0 ** -23 + (V / 16384 + 64) * 2.0 ** -24
    for n in range(4):
        assert abs(float(r.top_logprobs[0, n]) - (-n - math.log(s))) <= e + 20 * 2.0 ** -22
    assert float(r.logprob[0]) == float(r.top_logprobs[0, 2])
    ent = math.log(s) - t / s
    assert abs(float(r.entropy[0]) - ent) <= 4 * e * ent
