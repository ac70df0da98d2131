"""GPU tests of the operators for rows of tokens over the caches against their
plain 64-bit forms (rows_ref.py): the draft plan, head norms with the rotary
position, attention over a cache, and log probabilities of given tokens; with
lengths of none and one, ragged batches, odd sizes and strides, rows that see
nothing, infinities and NaN in unseen places, untouched memory behind the
rows, and a step of them together against the decode step."""
import math

import numpy as np
import pytest

import rows_ref as ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import q3vl_int8 as q  # noqa: E402
from q3vl_int8 import attention as qa  # noqa: E402


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


def starts(rows):
    return np.concatenate([[0], np.cumsum(rows)]).astype(np.int64)


def random_parents(rng, rows):
    out = []
    for n in rows:
        out += [int(t - 1 - math.floor(rng.random() ** 2 * (t + 1))) for t in range(n)]
    return np.maximum(np.array(out, np.int64), -1) if out else np.zeros(0, np.int64)


def within(got, want, tol, what):
    off = np.abs(got.astype(np.float64) - want)
    bad = ~(off <= tol)
    if bad.any():
        at = tuple(np.argwhere(bad)[0])
        pytest.fail(f"{what}: {bad.sum()} of {bad.size} off, first at {at}: {got[at]} for {want[at]}, tolerance {tol[at]}", pytrace=False)


# ------------------------------------------------------------------ the plan
def check_plan(parents, rows, lens, max_seq, max_rows, pad=0, words=None, delta=None):
    st = starts(rows)
    total = int(st[-1]) + pad
    par = np.concatenate([parents, np.zeros(pad, np.int64)])
    words = words or max(1, -(-max_rows // 64))
    m = torch.full((total, words), -7, dtype=torch.int64, device="cuda")
    mask, pos, slots = qa.draft_plan(i32(par), i32(st), i32(lens), max_seq, max_rows, mask=m,
                                     pos_delta=None if delta is None else i32(delta))
    em, ep, es = ref.plan(par, st, lens, max_seq, max_rows, words, delta)
    np.testing.assert_array_equal(mask.cpu().numpy().view(np.uint64), em)
    np.testing.assert_array_equal(pos.cpu().numpy(), ep)
    np.testing.assert_array_equal(slots.cpu().numpy(), es)


@pytest.mark.parametrize("T", [1, 2, 3, 63, 64, 65, 200, 257, 513, 1024])
def test_plan_trees(T):
    rng = np.random.default_rng(T)
    rows = [T, 0, max(1, T // 3), T]
    check_plan(random_parents(rng, rows), rows, [5, 0, 77, 1000], 2100, T, pad=3, delta=[0, 3, -70, 11])


@pytest.mark.parametrize("T", [1, 64, 100, 1024])
def test_plan_chains_and_stars(T):
    """The deepest tree (a chain) and the flattest (all roots)."""
    check_plan(np.concatenate([np.arange(T) - 1, np.full(T, -1)]), [T, T], [3, 9], T + 9, T, words=T // 64 + 2)


def test_plan_refused_rows():
    """Parents out of place and their descendants, rows past max_rows and past
    the cache, negative lengths, positions below 0: position -2, nothing else."""
    par = np.array([-1, 0, 2, 2, 1, 5, 9, -2, 7, 3] + [-1, 0, 1, 2, 3, 4] + [-1, 0, 1] + [-1, -1] + [-1, 0, 1, 2])
    check_plan(par, [10, 6, 3, 2, 4], [4, 60, -1, 64, 2], 64, 5, pad=2, delta=[0, 0, 0, 0, -4])


def test_plan_many_sequences():
    rng = np.random.default_rng(3)
    rows = [int(n) for n in rng.integers(0, 9, 300)]
    check_plan(random_parents(rng, rows), rows, rng.integers(0, 50, 300), 64, 8, pad=40)


# ------------------------------------------------- head norms and the rotation
def norm_weights(rng, D, gs):
    w = rng.integers(-127, 128, D).astype(np.int8)
    return w, rng.uniform(0.002, 0.02, D // gs).astype(np.float32)


def tables(rows, D, theta=5e6):
    a = np.arange(rows)[:, None] * theta ** (-np.arange(0, D, 2) / D)
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


def bits(t):
    return t.cpu().numpy().view({2: np.uint16, 4: np.uint32}[t.element_size()])


@pytest.mark.parametrize("H,Hk,gs", [(16, 8, 64), (1, 1, 128), (7, 7, 32), (13, 1, 16)], ids=str)
@pytest.mark.parametrize("M", [1, 2, 5, 37])
def test_rope_is_the_decode_steps(orc, M, H, Hk, gs):
    """head_dim 128, one axis: the oracle's norm and rotation bit for bit, and
    its fp16 caches; nothing else of the cache changes."""
    rng = np.random.default_rng(M * 100 + H)
    D, S, B = 128, 64, 3
    (qw, qs), (kw, ks) = norm_weights(rng, D, gs), norm_weights(rng, D, gs)
    cos, sin = tables(70, D)
    x = [rng.standard_normal((M, n * D)).astype(np.float32) * 3 for n in (H, Hk, Hk)]
    x[0][0, :D] = 0.0
    x[1][M - 1, 3] = 1e20
    kc, vc = (rng.standard_normal((B, Hk, S, D)).astype(np.float16) for _ in range(2))
    slots = rng.permutation(B * S)[:M].astype(np.int64)
    pos = rng.integers(0, 70, M)
    kt, vt = dev(kc), dev(vc)
    out = qa.qk_norm_rope(dev(x[0]), dev(x[1]), dev(x[2]), qa.KVCache(kt, vt), dev(slots), i32(pos),
                          qa.QKNorm(dev(qw), dev(qs), dev(kw), dev(ks), gs, 1e-6), qa.Rope(dev(cos), dev(sin)))
    want = np.empty_like(x[0])
    with np.errstate(over="ignore"):
        for r in range(M):
            c, s = cos[pos[r]], sin[pos[r]]
            want[r] = orc.rope(orc.rms_norm_inplace_i8(x[0][r], qw, qs, gs, 1e-6, H), c, s, H, D)
            b, at = divmod(int(slots[r]), S)
            kc[b, :, at] = orc.rope(orc.rms_norm_inplace_i8(x[1][r], kw, ks, gs, 1e-6, Hk), c, s, Hk, D).reshape(Hk, D)
            vc[b, :, at] = x[2][r].reshape(Hk, D)
    np.testing.assert_array_equal(bits(out), want.view(np.uint32))
    np.testing.assert_array_equal(bits(kt), kc.view(np.uint16))
    np.testing.assert_array_equal(bits(vt), vc.view(np.uint16))


@pytest.mark.parametrize("D,sections,inter", [(128, (24, 20, 20), True), (128, (16, 24, 24), False), (64, (12, 10, 10), True),
                                              (64, (0, 32, 0), False), (64, None, False), (128, (64, 0, 0), True)], ids=str)
@pytest.mark.parametrize("half", [False, True], ids=["fp32", "fp16"])
def test_rope_axes_strides_and_left_out_rows(D, sections, inter, half):
    """Positions on three axes in both layouts, views of one wide projection,
    a cache laid out [batch, max_seq, kv_heads, head_dim], rows without a token
    or without a slot, and positions past the tables."""
    rng = np.random.default_rng(D + half)
    M, H, Hk, S, B, gs = 23, 6, 2, 16, 2, 16
    (qw, qs), (kw, ks) = norm_weights(rng, D, gs), norm_weights(rng, D, gs)
    cos, sin = tables(50, D)
    axes = 1 if sections is None else 3
    x = rng.standard_normal((M, (H + 2 * Hk) * D + 24)).astype(np.float32)
    xt = dev(x)
    parts = [(0, H), (H, Hk), (H + Hk, Hk)]
    views = [xt[:, a * D:(a + n) * D] for a, n in parts]
    pos = rng.integers(0, 50, (M, axes))
    slots = rng.permutation(B * S)[:M].astype(np.int64)
    pos[3, 0], pos[5, 0], pos[6, -1], pos[7, 0] = -1, -2, 50, 2 ** 31 - 1
    slots[8], slots[9], slots[10] = -1, B * S, 2 ** 40
    base = rng.standard_normal((2, B, S, Hk, D)).astype(np.float16)
    c = dev(base)
    wide = rng.standard_normal((M, H * D + 5)).astype(np.float16 if half else np.float32)
    out_w = dev(wide)
    out = out_w[:, :H * D]
    qa.qk_norm_rope(*views, qa.KVCache(c[0].transpose(1, 2), c[1].transpose(1, 2)), dev(slots), i32(pos),
                    qa.QKNorm(dev(qw), dev(qs), dev(kw), dev(ks), gs, 1e-5), qa.Rope(dev(cos), dev(sin), sections, inter), out=out)
    got, gc = out_w.cpu().numpy(), c.cpu().numpy()
    axis = ref.axis_of(D // 2, sections, inter)
    touched = np.zeros((B, S), bool)
    np.testing.assert_array_equal(got[:, H * D:], wide[:, H * D:])
    for r in range(M):
        if pos[r, 0] == -1:
            np.testing.assert_array_equal(got[r], wide[r])
            continue
        if not all(0 <= p < 50 for p in pos[r]):
            assert np.isnan(got[r, :H * D].astype(np.float32)).all()
            continue
        xs = [x[r, a * D:(a + n) * D].reshape(n, D) for a, n in parts]
        want, size = ref.norm_rope(xs[0], qw, qs, gs, 1e-5, cos, sin, pos[r], axis)
        # the mean of D squares: D half steps; root, reciprocal, three products
        # and the two-term rotation a few more; the output's own rounding
        tol = size * (D + 16) * ref.EPS32
        tol16 = tol + np.abs(want) * 2.0 ** -11 + 2.0 ** -25
        within(got[r, :H * D].reshape(H, D), want, tol16 if half else tol, f"row {r}")
        if 0 <= slots[r] < B * S:
            b, at = divmod(int(slots[r]), S)
            touched[b, at] = True
            want, size = ref.norm_rope(xs[1], kw, ks, gs, 1e-5, cos, sin, pos[r], axis)
            tol16 = size * (D + 16) * ref.EPS32 + np.abs(want) * 2.0 ** -11 + 2.0 ** -25
            within(gc[0, b, at], want, tol16, f"key {r}")
            np.testing.assert_array_equal(gc[1, b, at], xs[2].astype(np.float16))
    np.testing.assert_array_equal(gc[:, ~touched], base[:, ~touched])


def test_rope_in_place_and_many_rows():
    """q_out over q gives what a separate q_out gives; more rows than blocks run at once."""
    rng = np.random.default_rng(1)
    M, H, Hk, D, gs = 3001, 16, 8, 128, 64
    (qw, qs), (kw, ks) = norm_weights(rng, D, gs), norm_weights(rng, D, gs)
    cos, sin = tables(M, D)
    x = [dev(rng.standard_normal((M, n * D)).astype(np.float32)) for n in (H, Hk, Hk)]
    norm, rope = qa.QKNorm(dev(qw), dev(qs), dev(kw), dev(ks), gs, 1e-6), qa.Rope(dev(cos), dev(sin))
    slots, pos = torch.arange(M, device="cuda"), torch.arange(M, device="cuda", dtype=torch.int32)
    caches = [torch.zeros((2, 1, Hk, M, D), dtype=torch.float16, device="cuda") for _ in range(2)]
    a = qa.qk_norm_rope(*x, qa.KVCache(*caches[0]), slots, pos, norm, rope)
    qc = x[0].clone()
    b = qa.qk_norm_rope(qc, x[1], x[2], qa.KVCache(*caches[1]), slots, pos, norm, rope, out=qc)
    assert b.data_ptr() == qc.data_ptr()
    assert torch.equal(a.view(torch.int32), b.view(torch.int32)) and torch.equal(*[c.view(torch.int16) for c in caches])
    # the last row alone is what it is among the others
    one = torch.zeros_like(caches[0])
    c = qa.qk_norm_rope(*[t[M - 1:] for t in x], qa.KVCache(*one), slots[M - 1:], pos[M - 1:], norm, rope)
    assert torch.equal(c.view(torch.int32), a[M - 1:].view(torch.int32))


# ---------------------------------------------------------------- attention
class Batch:
    """A batch over random caches, with the 64-bit answer row by row."""

    def __init__(self, seed, rows, lens, H, Hk, D, half, tree, pad=0, slack=5, qscale=2.0, words=None):
        rng = self.rng = np.random.default_rng(seed)
        self.rows, self.lens, self.H, self.Hk, self.D, self.half = rows, lens, H, Hk, D, half
        self.S = max(n + c for n, c in zip(rows, lens)) + slack
        self.st, self.T = starts(rows), max(max(rows), 1)
        N = int(self.st[-1]) + pad
        dt = np.float16 if half else np.float32
        self.q = (rng.standard_normal((N, H * D)) * qscale).astype(dt)
        self.k, self.v = (rng.standard_normal((len(rows), Hk, self.S, D)).astype(np.float16) for _ in range(2))
        self.mask = None
        if tree:
            W = words or -(-self.T // 64)
            par = np.concatenate([random_parents(rng, rows), np.zeros(pad, np.int64)])
            self.mask = ref.plan(par, self.st, [0] * len(rows), 1 << 20, 1 << 20, max(W, -(-self.T // 64)))[0][:, :W].copy()
        self.out = rng.standard_normal((N, H * D)).astype(dt)  # what was in the buffer

    def tensors(self):
        k, v = dev(self.k), dev(self.v)
        return dict(q=dev(self.q), cache=qa.KVCache(k, v), row_start=i32(self.st), cache_len=i32(self.lens), max_rows=self.T,
                    mask=None if self.mask is None else dev(self.mask.view(np.int64)), out=dev(self.out))

    def run(self, **over):
        a = {**self.tensors(), **over}
        got = qa.tree_attention(**a)
        torch.cuda.synchronize()
        return got.cpu().numpy()

    def check(self, got, scale=None, only=None):
        scale = self.D ** -0.5 if scale is None else scale
        for b, n in enumerate(self.rows):
            for t in range(n):
                r = int(self.st[b]) + t
                if only is not None and not only(b, t):
                    continue
                seen = ref.seen_by(t, n, self.lens[b], None if self.mask is None else self.mask[r])
                want, absv, qk = ref.attention(self.q[r].reshape(self.H, self.D), self.k[b], self.v[b], seen, scale)
                tol = ref.attention_tolerance(absv, qk, self.D, len(seen), self.half)
                g = got[r].reshape(self.H, self.D).astype(np.float64)
                within(g, want, tol, f"seq {b} row {t}")
        np.testing.assert_array_equal(got[int(self.st[-1]):], self.out[int(self.st[-1]):])


HEADS = [(16, 8, 128), (4, 4, 64), (12, 2, 64), (5, 1, 128)]


@pytest.mark.parametrize("H,Hk,D", HEADS, ids=str)
@pytest.mark.parametrize("half", [False, True], ids=["fp32", "fp16"])
def test_attention_one_token(H, Hk, D, half):
    """One new token of each sequence, contexts of none, one and odd lengths;
    one sequence takes no part; the buffer behind the rows stays."""
    lens = [0, 1, 31, 32, 33, 63, 64, 100, 127, 128, 129, 300, 1000]
    B = Batch(H, [1] * 5 + [0] + [1] * 7, lens, H, Hk, D, half, False, pad=3)
    B.check(B.run())


@pytest.mark.parametrize("H,Hk,D", HEADS, ids=str)
@pytest.mark.parametrize("half", [False, True], ids=["fp32", "fp16"])
@pytest.mark.parametrize("tree", [False, True], ids=["chain", "tree"])
def test_attention_few_rows(H, Hk, D, half, tree):
    B = Batch(H + 1, [2, 7, 0, 16, 33, 5], [0, 90, 50, 515, 64, 31], H, Hk, D, half, tree, pad=2)
    B.check(B.run())


@pytest.mark.parametrize("half", [False, True], ids=["fp32", "fp16"])
@pytest.mark.parametrize("tree", [False, True], ids=["chain", "tree"])
@pytest.mark.parametrize("T", [64, 65, 128, 130, 259])
def test_attention_many_rows(T, half, tree):
    """Row tiles and mask words at their edges."""
    B = Batch(T, [T, 1, T - 1], [70, 3, 0], 4, 2, 128 if T % 2 else 64, half, tree, pad=1)
    B.check(B.run())


@pytest.mark.parametrize("half", [False, True], ids=["fp32", "fp16"])
@pytest.mark.parametrize("T,ctx", [(1, 5000), (1, 20011), (9, 9001), (70, 4099)], ids=str)
def test_attention_split(T, ctx, half):
    """Long contexts, split and joined; the hint about their length, right,
    absent or far too small, changes the split alone."""
    B = Batch(T, [T, 1], [ctx, 37], 8, 4, 128, half, T > 1)
    B.check(B.run())
    B.check(B.run(max_len=ctx + T))
    B.check(B.run(max_len=1))


@pytest.mark.parametrize("half", [False, True], ids=["fp32", "fp16"])
def test_attention_prompt(half):
    B = Batch(8, [500], [300], 4, 2, 128, half, False)
    B.check(B.run())


def test_attention_flat_probabilities():
    """Scores near zero over few keys: what the probabilities' two terms and
    the sums keep shows against a bound of a few steps."""
    B = Batch(5, [7, 3], [0, 11], 4, 2, 128, False, False, qscale=1e-6)
    B.check(B.run())


@pytest.mark.parametrize("qscale", [1e-30, 1e-5, 300.0, 1e15])
def test_attention_query_sizes(qscale):
    """Queries far from fp16's range: their two terms are taken relative to the
    row's largest value. The largest: one key takes all."""
    B = Batch(6, [5, 40], [100, 64], 4, 2, 64, False, True, qscale=qscale)
    if qscale < 1e10:
        B.check(B.run())
        return
    got = B.run()
    for b, n in enumerate(B.rows):
        for t in range(n):
            r = int(B.st[b]) + t
            seen = ref.seen_by(t, n, B.lens[b], B.mask[r])
            for h in range(4):
                s = B.k[b, h // 2][seen].astype(np.float64) @ B.q[r, h * 64:(h + 1) * 64].astype(np.float64)
                best = seen[int(np.argmax(s))]
                np.testing.assert_allclose(got[r, h * 64:(h + 1) * 64], B.v[b, h // 2, best], rtol=2.0 ** -20)


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.7])
def test_attention_scale(scale):
    B = Batch(7, [3, 20], [50, 7], 4, 2, 64, False, True)
    B.check(B.run(scale=scale), scale=scale)


@pytest.mark.parametrize("half", [False, True], ids=["fp32", "fp16"])
def test_attention_rows_that_see_nothing(half):
    """Empty mask lines: over no cache the answer is 0, over a cache it is the
    cache's; bits of rows that do not exist count for nothing."""
    B = Batch(9, [4, 40, 3], [0, 0, 45], 4, 2, 128, half, True)
    B.mask[:] = 0
    B.mask[5] = (1 << 64) - 1 - ((1 << 40) - 1)  # bits of rows 40 ..
    B.mask[7] = 1 << 39 | 1 << 45
    B.mask[46] = 1 << 2
    got = B.run()
    assert (got[:4] == 0).all() and (got[4:7] == 0).all()
    B.mask[5], B.mask[7] = 0, 1 << 39
    B.check(got)


def test_attention_mask_words():
    """A mask with fewer words than rows (the rest unseen), and with more."""
    B = Batch(10, [100, 3], [20, 5], 4, 2, 64, False, True, words=1)
    B.check(B.run())
    B = Batch(11, [100, 3], [20, 5], 4, 2, 64, False, True, words=5)
    B.mask[:, 4] = (1 << 64) - 1
    got = B.run()
    B.check(got)


@pytest.mark.parametrize("half", [False, True], ids=["fp32", "fp16"])
@pytest.mark.parametrize("T", [1, 6, 90])
@pytest.mark.parametrize("ctx", [3, 700])
def test_attention_unseen_infinities(half, T, ctx):
    """NaN and infinities in the cache behind the rows, in drafts that other
    rows see, and in another row's query: only rows that see them change."""
    B = Batch(T + ctx, [T, 2], [ctx, 10], 4, 2, 128, half, True)
    for b, n in enumerate(B.rows):
        for c in (B.k, B.v):
            c[b, :, B.lens[b] + n:] = np.nan
    bad = {}
    if T > 1:
        B.v[0, 0, ctx + 1, 5], B.k[0, 1, ctx + 2, 7] = np.inf, np.nan
        B.v[0, 1, ctx + T - 1] = np.nan
        bad = {1, 2, T - 1}
        B.q[0, 3] = np.nan  # head 0 of the first row
    got = B.run()

    def clean(b, t):
        r = int(B.st[b]) + t
        return b == 1 or (t > 0 and not any(int(B.mask[r, j // 64]) >> (j % 64) & 1 for j in bad)) or T == 1

    B.check(got, only=clean)
    if T > 1:
        assert np.isnan(got[0, :128]).all()
        for t in range(1, T):
            see = [j for j in (1, 2, T - 1) if int(B.mask[t, j // 64]) >> (j % 64) & 1]
            o = got[t].reshape(4, 128).astype(np.float64)
            if 1 in see and T - 1 != 1:
                assert (o[:2, 5] == np.inf).all() and np.isfinite(np.delete(o[:2], 5, 1)).all()
            if 2 in see or T - 1 in see:
                assert np.isnan(o[2:]).all()
            else:
                assert np.isfinite(o[2:]).all()


def test_attention_sequences_that_do_not_fit():
    """A negative length, or rows past the cache: NaN, and the others whole."""
    B = Batch(12, [2, 3, 2, 1], [10, 20, 5, 8], 4, 2, 64, False, False, slack=0)
    lens = [10, B.S - 2, -1, 8]
    got = B.run(cache_len=i32(lens))
    assert np.isnan(got[2:7]).all()
    B.check(got, only=lambda b, t: b in (0, 3))


def test_attention_max_rows_and_broken_starts():
    """Rows past max_rows stay as they were; starts outside of the rows are
    taken as the nearest row there is."""
    B = Batch(13, [6, 2], [10, 20], 4, 2, 64, False, False)
    got = B.run(max_rows=4)
    B.check(got, only=lambda b, t: t < 4)
    np.testing.assert_array_equal(got[4:6], B.out[4:6])
    got = B.run(row_start=i32([-5, 6, 1 << 30]))
    B.check(got)
    got = B.run(row_start=i32([0, 6, 3]))
    np.testing.assert_array_equal(got[6:], B.out[6:])
    B.check(np.concatenate([got[:6], B.run()[6:]]))


def test_attention_layouts():
    """The cache as [batch, max_seq, kv_heads, head_dim], one layer of the
    decode step's caches, and q and out as views of wider rows."""
    B = Batch(14, [4, 1], [66, 130], 6, 3, 128, False, True)
    want = B.run()
    B.check(want)
    c = [dev(x.transpose(0, 2, 1, 3)).transpose(1, 2) for x in (B.k, B.v)]
    np.testing.assert_array_equal(B.run(cache=qa.KVCache(*c)), want)
    N = B.q.shape[0]
    wide = torch.zeros((N, 2 * B.q.shape[1] + 4), device="cuda")
    wide[:, 4:4 + B.q.shape[1]] = dev(B.q)
    ow = torch.full_like(wide, 7.0)
    got = B.run(q=wide[:, 4:4 + B.q.shape[1]], out=ow[:, :B.q.shape[1]])
    np.testing.assert_array_equal(got, want)
    assert (ow[:, B.q.shape[1]:] == 7).all()
    layers = torch.randn((3, 3, B.S, 128), device="cuda").half(), torch.randn((3, 3, B.S, 128), device="cuda").half()
    one = Batch(15, [4], [66], 6, 3, 128, False, True)
    one.S = B.S
    one.k, one.v = (x[1][None].cpu().numpy() for x in layers)
    one.check(one.run(cache=qa.KVCache(layers[0][1][None], layers[1][1][None])))


@pytest.mark.parametrize("rows,lens", [([1, 1], [900, 5]), ([40, 7], [700, 3]), ([150, 20], [64, 40])], ids=str)
def test_attention_in_place(rows, lens):
    """out over q gives what a separate out gives."""
    for half in (False, True):
        B = Batch(16, rows, lens, 8, 4, 128, half, True)
        x = dev(B.q)
        np.testing.assert_array_equal(B.run(q=x, out=x), B.run())


def test_attention_offsets_past_32_bits():
    """A cache of over 2^32 bytes a head and 2^33 in all: the last positions."""
    S, D = (1 << 25) + 1024, 64
    k, v = (torch.zeros((1, 2, S, D), dtype=torch.float16, device="cuda") for _ in range(2))
    lens, n = S - 70, 70
    g = torch.Generator(device="cuda").manual_seed(1)
    for c in (k, v):
        c[:, :, lens - 100:] = torch.randn((1, 2, n + 100, D), device="cuda", generator=g).half()
    k[:, :, :lens - 100] = -50.0  # weightless against the rest for positive queries
    x = torch.rand((n, 2 * D), device="cuda", generator=g) + 0.5
    got = qa.tree_attention(x, qa.KVCache(k, v), i32([0, n]), i32([lens]), n)
    tail = [t[0, :, lens - 100:].double().cpu().numpy() for t in (k, v)]
    got = got.cpu().numpy()
    for t in (0, 1, 35, 69):
        want, absv, qk = ref.attention(x[t].cpu().numpy().reshape(2, D), *tail, list(range(101 + t)), D ** -0.5)
        tol = ref.attention_tolerance(absv, qk + 300.0, D, 4096, False)
        within(got[t].reshape(2, D), want, tol, f"row {t}")


# --------------------------------------------------------- log probabilities
def check_logprobs(x, tokens, k, t=None):
    r = q.token_logprobs(dev(x) if t is None else t, i32(tokens), top_k=k)
    lp, rank, ent, ids, top = (a.cpu().numpy() for a in r)
    V = x.shape[1]
    for m in range(x.shape[0]):
        elp, erank, eent, eids, etop = ref.logprobs(x[m], int(tokens[m]), k)
        np.testing.assert_array_equal(ids[m], eids)
        assert rank[m] == erank
        # 2^y with y = (x - m) log2 e rounded twice: an error of |x - m| 2^-23
        # and the exponential's own 2^-23, for weights that count (|x - m| < 20)
        # at most 21 2^-23 of the rest's sum, and V half steps in it; log1p
        # shrinks both. x - m and the last difference round once each.
        e = 21 * 2.0 ** -23 + V ** 0.5 * 2.0 ** -22
        fin = x[m][np.isfinite(x[m])].astype(np.float64)
        rest = max(1e-30, np.exp(-ref.logprobs(x[m], int(eids[0] if k else np.argmax(np.nan_to_num(x[m], nan=-np.inf))), 0)[0]) - 1) if fin.size else 1
        logs = math.log1p(rest) if rest == rest else 1.0
        for got, want in [(lp[m], elp)] + list(zip(top[m], etop)):
            if not np.isfinite(want):
                assert (np.isnan(want) and np.isnan(got)) or got == want, (m, got, want)
                continue
            tol = e * min(rest / (1 + rest), 1.0) + abs(want) * 2.0 ** -22 + logs * 2.0 ** -22
            assert abs(got - want) <= tol, (m, got, want, tol)
        if not np.isfinite(eent):
            assert np.isnan(ent[m])
        else:
            assert abs(ent[m] - eent) <= 4 * e * max(eent, logs) + 1e-30, (m, ent[m], eent)


@pytest.mark.parametrize("V", [1, 2, 3, 63, 64, 255, 256, 257, 1000, 1023, 4099, 32000, 151936])
@pytest.mark.parametrize("half", [False, True], ids=["fp32", "fp16"])
def test_logprobs_sizes(V, half):
    rng = np.random.default_rng(V)
    M = 3
    x = (rng.standard_normal((M, V)) * 3).astype(np.float16 if half else np.float32)
    x[1, rng.integers(V)] += 9
    tokens = [0, V - 1, int(rng.integers(V))]
    for k in sorted({0, 1, min(5, V), min(20, V), min(64, V)}):
        check_logprobs(x, tokens, k)


@pytest.mark.parametrize("M,V", [(1, 151936), (70, 2000), (300, 515)], ids=str)
def test_logprobs_rows(M, V):
    rng = np.random.default_rng(M)
    x = (rng.standard_normal((M, V)) * 4).astype(np.float32)
    check_logprobs(x, rng.integers(0, V, M), 20)


@pytest.mark.parametrize("half", [False, True], ids=["fp32", "fp16"])
@pytest.mark.parametrize("off,pad", [(0, 1), (1, 0), (3, 6), (2, 2)], ids=str)
def test_logprobs_strides(off, pad, half):
    """Rows that start anywhere, in a wider buffer of NaN."""
    rng = np.random.default_rng(off)
    M, V = 5, 3001
    buf = np.full((M, V + off + pad), np.nan, np.float16 if half else np.float32)
    buf[:, off:off + V] = rng.standard_normal((M, V)) * 3
    t = dev(buf)[:, off:off + V]
    check_logprobs(buf[:, off:off + V], [0, 1, V - 1, V - 2, 77], 9, t)


def test_logprobs_ties():
    """Equal values by their place, zeros of both signs among them, in rows of
    few values and in constant ones."""
    rng = np.random.default_rng(0)
    V = 5000
    x = np.stack([rng.integers(-2, 3, V), np.zeros(V), np.where(np.arange(V) % 2, -0.0, 0.0), rng.integers(0, 2, V) * 1.5,
                  np.sort(rng.standard_normal(V)), -np.sort(rng.standard_normal(V))]).astype(np.float32)
    check_logprobs(x, [17, 4999, 3, 2500, 4990, 0], 64)
    check_logprobs(x.astype(np.float16), [4000, 0, 4, 2501, 0, 64], 64)


@pytest.mark.parametrize("k", [1, 31, 32, 33, 40, 63, 64])
def test_logprobs_rising_rows(k):
    """Rows whose values rise, so that each one read is among the best so far:
    the lists of alternatives are full at every turn."""
    for V, n in ((1500, 1), (9000, 3), (34000, 2)):
        x = np.stack([np.linspace(-9, 9, V), -np.linspace(-9, 9, V), np.roll(np.linspace(-9, 9, V), V // 2)])[:n].astype(np.float32)
        check_logprobs(x, [V - 1, 0, V // 3][:n], k)


def test_logprobs_ruled_out_values():
    """-inf beside few finite values, a row of nothing else, NaN, +inf, tokens
    outside of the row, the type's lowest value."""
    rng = np.random.default_rng(2)
    V = 2600
    x = rng.standard_normal((10, V)).astype(np.float32)
    x[0, 5:] = -np.inf
    x[1, :] = -np.inf
    x[1, 2000] = 3.0
    x[2, :] = -np.inf
    x[3, 100] = np.nan
    x[4, 7] = np.inf
    x[5, :] = np.finfo(np.float32).min
    x[6, 1:] = np.finfo(np.float32).min
    x[9, ::2] = -np.inf
    tokens = [3, 2000, 8, 5, 7, 9, 0, V, -1, 1]
    check_logprobs(x, tokens, 20)
    check_logprobs(x, [9, 0, 0, 100, 8, 0, 1, 2 ** 31 - 1, -2 ** 31, 0], 3)


def test_logprobs_of_the_certain_token():
    """One value far above: the log probability is that of the rest, to its
    last digits, and not 0."""
    V = 4096
    for gap in (9.0, 20.0, 40.0):
        x = np.zeros((2, V), np.float32)
        x[:, 1234] = gap
        x[1, 77] = gap - 12.0
        r = q.token_logprobs(dev(x), i32([1234, 1234]), top_k=1)
        for m in range(2):
            want = -math.log1p((V - 1 - m) * math.exp(-gap) + m * math.exp(-12.0))
            # |x - m| 2^-23 and the exponential's 2^-23, V half steps
            assert abs(float(r.logprob[m]) - want) <= abs(want) * (45 + V) * 2.0 ** -23
            assert r.top_ids[m, 0] == 1234 and r.rank[m] == 0 and r.top_logprobs[m, 0] == r.logprob[m]


@pytest.mark.parametrize("half", [False, True], ids=["fp32", "fp16"])
@pytest.mark.parametrize("T,ctx", [(7, 30), (40, 30), (150, 64), (40, 5000)], ids=str)
def test_attention_redone_rows_in_place(T, ctx, half):
    """A row whose result one lane alone finds not finite (an infinity in a
    single column of an unseen draft) is done again from its query: with out
    over q no lane of it may write before that. Unsplit and split tiles, few
    rows and many; the answer is that without the infinity."""
    B = Batch(T + ctx + 1, [T, 3], [ctx, 9], 4, 2, 128, half, True)
    for col in (0, 37, 126):
        clean = B.run()
        kept = B.v.copy()
        B.v[0, :, ctx + T - 1, col] = np.inf  # the last draft: no other row sees it
        x = dev(B.q)
        got = B.run(q=x, out=x)
        unseen = [r for r in range(T - 1)]
        assert np.isfinite(got[unseen]).all()
        B.check(got, only=lambda b, t: b == 1 or t < T - 1)
        g = got[T - 1].reshape(4, 128)
        assert (g[:, col] == np.inf).all() and np.isfinite(np.delete(g, col, 1)).all()
        np.testing.assert_array_equal(got, B.run())
        B.v = kept
        np.testing.assert_array_equal(B.run(), clean)


def test_plans_of_two_threads():
    """Plans of different sizes, both past 64 KiB of LDS, from two threads at
    once: neither call changes what the other's launch may use."""
    import threading
    wrong = []

    def plans(T):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                par = random_parents(np.random.default_rng(T), [T, T])
                args = i32(par), i32([0, T, 2 * T]), i32([5, 70]), 2 * T, T
                want = ref.plan(par, [0, T, 2 * T], [5, 70], 2 * T, T, -(-T // 64))
                got = [qa.draft_plan(*args) for _ in range(100)]
                stream.synchronize()
                for mask, pos, slots in got:
                    np.testing.assert_array_equal(mask.cpu().numpy().view(np.uint64), want[0])
                    np.testing.assert_array_equal(pos.cpu().numpy(), want[1])
                    np.testing.assert_array_equal(slots.cpu().numpy(), want[2])
        except BaseException as e:  # noqa: BLE001  (for the main thread)
            wrong.append((T, e))

    threads = [threading.Thread(target=plans, args=(T,)) for T in (1024, 750)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong


@pytest.mark.parametrize("half", [False, True], ids=["fp32", "fp16"])
@pytest.mark.parametrize("T,ctx", [(1, 3000), (40, 900)], ids=str)
@pytest.mark.parametrize("gap", [5.0, 12.0, 17.0, 21.0, 25.0])
def test_attention_small_probabilities(gap, T, ctx, half):
    """One cached key ahead of all others by e^gap, its value 0: the answer is
    made of the others' probabilities, which are held no finer than 2^-31 of
    the row's largest (fp16 subnormals' half step, 2^-25, where the largest is
    2^6 at least). Over the values: 2^-31 sum |v|, beside the general bound."""
    B = Batch(T, [T], [ctx], 4, 2, 128, half, False)
    B.k[:] = 0
    B.k[0, :, 0, 0] = 8.0
    B.v[0, :, 0] = 0
    B.q[:, 0::128] = gap / 8.0 / 128 ** -0.5
    got = B.run()
    for t in {0, T // 2, T - 1}:
        seen = ref.seen_by(t, T, ctx, None)
        want, absv, qk = ref.attention(B.q[t].reshape(4, 128), B.k[0], B.v[0], seen, 128 ** -0.5)
        sums = np.repeat(np.abs(B.v[0][:, seen].astype(np.float64)).sum(1), 2, axis=0)
        tol = ref.attention_tolerance(absv, qk, 128, len(seen), half) + 2.0 ** -31 * 1.01 * sums
        within(got[t].reshape(4, 128), want, tol, f"row {t}")
