"""GPU tests of the operators for long contexts against their plain 64-bit forms
(long_ref.py): blocks of 32 positions packed to 8 bits and read back, attention
over them and the fp16 rows behind them, and through windows; with lengths of
none and one, ragged batches, odd sizes and strides, rows that see nothing,
infinities and NaN, broken lengths, and untouched memory."""
import numpy as np
import pytest

import long_ref as ref
import rows_ref
from long_ref import within

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import q3vl_int8 as q  # noqa: E402
from q3vl_int8 import attention as qa  # noqa: E402


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


# ------------------------------------------------------- packing and reading
class Store:
    """A cache and its blocks, random, on the host and the device."""

    def __init__(self, seed, B, Hk, D, S, blocks, by_row=False):
        rng = self.rng = np.random.default_rng(seed)
        self.k, self.v = (rng.standard_normal((B, Hk, S, D)).astype(np.float16) for _ in range(2))
        self.k8, self.v8 = (rng.integers(-127, 128, (B, Hk, blocks, 32 * D)).astype(np.int8) for _ in range(2))
        self.ks, self.vs = (rng.random((B, Hk, blocks)).astype(np.float32) for _ in range(2))
        self.by_row = by_row

    def device(self):
        """Tensors and descriptions; by_row: the cache as [batch, row, head, value]."""
        if self.by_row:
            kv = [dev(x.transpose(0, 2, 1, 3)).transpose(1, 2) for x in (self.k, self.v)]
        else:
            kv = [dev(x) for x in (self.k, self.v)]
        packed = [dev(x) for x in (self.k8, self.v8, self.ks, self.vs)]
        return kv, packed, qa.KVCache(*kv), qa.PackedKV(*packed)

    def pack(self, cached, at):
        kv, packed, cache, p = self.device()
        lens = i32(cached), i32(at)
        qa.kv_pack(cache, p, *lens)
        assert lens[0].tolist() == list(cached) and lens[1].tolist() == list(at)
        qa.kv_advance(cache, p, *lens)
        whole = [ref.fills(n, a, self.k.shape[2], self.k8.shape[2]) for n, a in zip(cached, at)]
        assert lens[0].tolist() == [n - 32 * w for n, w in zip(cached, whole)]
        assert lens[1].tolist() == [a + 32 * w for a, w in zip(at, whole)]
        ref.pack(self.k, self.v, self.k8, self.v8, self.ks, self.vs, cached, at)
        for got, want in zip([*kv, *packed], (self.k, self.v, self.k8, self.v8, self.ks, self.vs)):
            np.testing.assert_array_equal(got.cpu().numpy(), want)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("by_row", [False, True])
def test_pack(D, by_row):
    """Bit for bit what the definition gives, lengths at and about whole blocks;
    sequences that cannot be packed whole, or whose lengths are broken, are left
    alone, and so is everything else in memory."""
    cached = [0, 1, 31, 32, 33, 63, 64, 65, 100, 203, 200, 64, 64, 64, -1, 204, 64, -2 ** 31]
    at = [0, 32, 64, 0, 32, 320, 0, 160, 32, 0, 192, 33, -32, 320, 0, 0, 384, 0]
    Store(D, len(cached), 3, D, 203, 11, by_row).pack(cached, at)


def test_pack_special_values():
    """Blocks of zeros, of the largest and the smallest halves, ties, and blocks
    that hold an infinity or NaN (a NaN scale, for that head and part alone)."""
    s = Store(5, 1, 2, 128, 200, 8)
    s.k[0, 0, :32] = 0
    s.k[0, 1, :32] = -0.0
    s.v[0, 0, :32] = 65504
    s.v[0, 1, :32] = -(2.0 ** -24)
    s.k[0, 0, 32:64] = np.arange(32)[:, None] * 4.0  # halves of the step of 127 / 127 among them
    s.k[0, 0, 40, 3] = 127
    s.k[0, 0, 41, :100] = np.arange(100) + 0.5
    s.k[0, 1, 70, 5], s.v[0, 0, 97, 127], s.v[0, 1, 66, 0] = np.nan, np.inf, -np.inf
    s.pack([170], [32])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("by_row", [False, True])
def test_unpack(D, by_row):
    """Positions from anywhere on, as far as they are packed and asked for; the
    cache's other rows stay."""
    at = [0, 32, 64, 96, 320, 352, 64, 64, 1 << 30, -5, 96]
    first = [0, 0, 5, 64, 31, 33, 64, 200, 300, 0, -3]
    for f, count in [(first, 70), (first, 1), (None, 203), (first, 203), (None, 33)]:
        s = Store(D, len(at), 2, D, 203, 11, by_row)
        s.ks[1, 1, 0] = np.nan
        kv, packed, cache, p = s.device()
        qa.kv_unpack(p, i32(at), cache, first=None if f is None else i32(f), count=count)
        for x, x8, sc, got, order in ((s.k, s.k8, s.ks, kv[0], ref.key_order), (s.v, s.v8, s.vs, kv[1], ref.value_order)):
            n = (ref.from_bytes(x8, order).astype(np.float32) * sc[..., None, None]).reshape(len(at), 2, -1, D)
            for b, end in enumerate(at):
                a = 0 if f is None else f[b]
                m = max(0, min(a + count, end, 352) - a) if a >= 0 else 0
                x[b, :, :m] = n[b, :, a:a + m].astype(np.float16)
            np.testing.assert_array_equal(got.cpu().numpy(), x)
        for got, want in zip(packed, (s.k8, s.v8, s.ks, s.vs)):
            np.testing.assert_array_equal(got.cpu().numpy(), want)


def test_pack_and_unpack_within_half_a_step():
    """There and back: no value is further off than half a step of its block and
    the result's own rounding."""
    s = Store(9, 2, 2, 128, 160, 5)
    kv, _, cache, p = s.device()
    lens = i32([160, 97]), i32([0, 0])
    qa.kv_pack(cache, p, *lens)
    qa.kv_advance(cache, p, *lens)
    back = [torch.zeros_like(x) for x in kv]
    qa.kv_unpack(p, lens[1], qa.KVCache(*back))
    for x, got, sc in ((s.k, back[0], p.k_scale), (s.v, back[1], p.v_scale)):
        for b, n in enumerate((160, 96)):
            step = np.repeat(sc[b, :, :n // 32].cpu().numpy().astype(np.float64), 32, 1)[..., None]
            want = x[b, :, :n].astype(np.float64)
            # the scale and the quotient round too: 2^-23 of 127 steps each
            within(got[b, :, :n].cpu().numpy(), want, step * (0.5 + 127 * 2.0 ** -22) + np.abs(want) * 2.0 ** -10, b)


# ---------------------------------------------------------------- attention
class Long:
    """A batch over packed positions and fp16 rows, with the 64-bit answer row by
    row. packed None: fp16 rows alone."""

    def __init__(self, seed, rows, lens, packed, H, Hk, D, half, tree, pad=0, slack=5, window=0, sinks=0, qscale=2.0, vscale=1.0):
        rng = self.rng = np.random.default_rng(seed)
        self.rows, self.lens, self.packed, self.H, self.Hk, self.D, self.half = rows, lens, packed, H, Hk, D, half
        self.window, self.sinks = window, sinks
        B, self.S = len(rows), max(n + c for n, c in zip(rows, lens)) + slack
        self.st, self.T = np.concatenate([[0], np.cumsum(rows)]).astype(np.int64), max(max(rows), 1)
        N = int(self.st[-1]) + pad
        dt = np.float16 if half else np.float32
        self.q = (rng.standard_normal((N, H * D)) * qscale).astype(dt)
        self.k, self.v = (rng.standard_normal((B, Hk, self.S, D)).astype(np.float16) for _ in range(2))
        if packed is not None:
            n = max(packed) // 32 + 1  # one more than is used
            self.kn, self.vn = (rng.integers(-127, 128, (B, Hk, n, 32, D)) for _ in range(2))
            self.ks = (rng.random((B, Hk, n)) * 0.02 + 0.005).astype(np.float32)
            self.vs = (np.exp2(rng.uniform(-1, 1, (B, Hk, n)) * 3) * 0.01 * vscale).astype(np.float32)
        self.mask = None
        if tree:
            par = np.concatenate([np.maximum([int(t - 1 - np.floor(rng.random() ** 2 * (t + 1))) for n in rows for t in range(n)], -1),
                                  np.zeros(pad)]).astype(np.int64)
            self.mask = rows_ref.plan(par, self.st, [0] * B, 1 << 20, 1 << 20, -(-self.T // 64))[0].copy()
        self.out = rng.standard_normal((N, H * D)).astype(dt)  # what was in the buffer

    def tensors(self):
        self.cache = dev(self.k), dev(self.v)
        a = dict(q=dev(self.q), cache=qa.KVCache(*self.cache), row_start=i32(self.st), cache_len=i32(self.lens), max_rows=self.T,
                 mask=None if self.mask is None else dev(self.mask.view(np.int64)), out=dev(self.out), window=self.window,
                 sinks=self.sinks)
        if self.packed is not None:
            p = qa.PackedKV(dev(ref.to_bytes(self.kn, ref.key_order)), dev(ref.to_bytes(self.vn, ref.value_order)), dev(self.ks),
                            dev(self.vs))
            a |= dict(packed=p, packed_len=i32(self.packed))
        return a

    def run(self, **over):
        got = qa.long_attention(**{**self.tensors(), **over})
        torch.cuda.synchronize()
        return got.cpu().numpy()

    def positions(self, b):
        """A sequence's keys and values in 64 bits, in order; its packed positions."""
        k, v = self.k[b].astype(np.float64), self.v[b].astype(np.float64)
        n = self.packed[b] if self.packed is not None else 0
        if n:
            kv = [(x[b].astype(np.float64) * s[b].astype(np.float64)[..., None, None]).reshape(self.Hk, -1, self.D)[:, :n]
                  for x, s in ((self.kn, self.ks), (self.vn, self.vs))]
            k, v = np.concatenate([kv[0], k], 1), np.concatenate([kv[1], v], 1)
        return k, v, n

    def check(self, got, scale=None, only=None):
        scale = self.D ** -0.5 if scale is None else scale
        for b, n in enumerate(self.rows):
            k, v, p = self.positions(b)
            vmax = 127 * float(np.nanmax(np.abs(self.vs[b, :, :p // 32]))) if p else 0.0
            for t in range(n):
                r = int(self.st[b]) + t
                if only is not None and not only(b, t):
                    continue
                seen = ref.seen_by(t, n, p + self.lens[b], None if self.mask is None else self.mask[r], self.window, self.sinks)
                want, absv, qk = rows_ref.attention(self.q[r].reshape(self.H, self.D), k, v, seen, scale)
                tol = ref.attention_tolerance(absv, qk, self.D, len(seen), self.half, vmax)
                within(got[r].reshape(self.H, self.D), want, tol, f"seq {b} row {t}")
        np.testing.assert_array_equal(got[int(self.st[-1]):], self.out[int(self.st[-1]):])


HEADS = [(16, 8, 128), (4, 4, 64), (12, 2, 64), (5, 1, 128)]
HALF = pytest.mark.parametrize("half", [False, True], ids=["fp32", "fp16"])


@pytest.mark.parametrize("H,Hk,D", HEADS, ids=str)
@HALF
def test_one_token(H, Hk, D, half):
    """One new token of each sequence behind packed positions and fp16 rows of
    none, one and odd numbers; one sequence takes no part."""
    lens = [0, 1, 31, 32, 0, 63, 0, 5, 70, 0, 129, 3]
    packed = [0, 0, 32, 64, 96, 0, 128, 160, 256, 1024, 544, 2016]
    B = Long(H, [1] * 4 + [0] + [1] * 7, lens, packed, H, Hk, D, half, False, pad=3)
    B.check(B.run())


@pytest.mark.parametrize("H,Hk,D", HEADS, ids=str)
@HALF
@pytest.mark.parametrize("tree", [False, True], ids=["chain", "tree"])
def test_few_rows(H, Hk, D, half, tree):
    B = Long(H + 1, [2, 7, 0, 16, 33, 5], [0, 90, 50, 15, 64, 31], [32, 0, 64, 512, 96, 640], H, Hk, D, half, tree, pad=2)
    B.check(B.run())


@HALF
@pytest.mark.parametrize("tree", [False, True], ids=["chain", "tree"])
@pytest.mark.parametrize("T", [64, 65, 128, 130, 259])
def test_many_rows(T, half, tree):
    """Row tiles and mask words at their edges."""
    B = Long(T, [T, 1, T - 1], [70, 3, 0], [96, 0, 352], 4, 2, 128 if T % 2 else 64, half, tree, pad=1)
    B.check(B.run())


@HALF
@pytest.mark.parametrize("T,ctx", [(1, 4992), (1, 20000), (9, 8992), (70, 4096)], ids=str)
def test_split(T, ctx, half):
    """Long contexts, split and joined; the hint about their length, right,
    absent or far too small, changes the split alone."""
    B = Long(T, [T, 1], [11, 37], [ctx, 32], 8, 4, 128, half, T > 1)
    B.check(B.run())
    B.check(B.run(max_len=ctx + 11 + T))
    B.check(B.run(max_len=1))


WINDOWS = [(1, 0), (1, 1), (5, 0), (31, 4), (32, 32), (33, 1), (64, 0), (100, 70), (127, 130), (700, 3), (5000, 4)]


@pytest.mark.parametrize("window,sinks", WINDOWS, ids=str)
@pytest.mark.parametrize("held", [False, True], ids=["fp16 rows", "packed"])
def test_window_one_token(window, sinks, held):
    """Windows that start in packed positions, in fp16 rows and before either,
    with first positions in both."""
    lens = [0, 1, 31, 32, 33, 100, 257, 700, 3, 20]
    packed = [0, 32, 96, 0, 640, 64, 128, 0, 1024, 288] if held else None
    B = Long(window, [1] * 10, lens, packed, 8, 4, 128 if window % 2 else 64, window % 3 == 0, False, pad=1, window=window, sinks=sinks)
    B.check(B.run())


@pytest.mark.parametrize("window,sinks", WINDOWS, ids=str)
@pytest.mark.parametrize("T", [7, 75, 300])
@pytest.mark.parametrize("held", [False, True], ids=["fp16 rows", "packed"])
def test_window_chain(T, window, sinks, held):
    """A prompt's chunk through a window: rows of one tile see different
    positions, windows inside the chunk itself and before it."""
    B = Long(T + window, [T, 2, T // 2], [0, 300, 40], [0, 160, 512] if held else None, 4, 2, 128 if T % 2 else 64, T == 75, False, pad=1,
             window=window, sinks=sinks)
    B.check(B.run())


@pytest.mark.parametrize("window,sinks", [(40, 0), (40, 3), (64, 70), (200, 1), (5000, 4)], ids=str)
@pytest.mark.parametrize("T", [3, 12, 40])
@pytest.mark.parametrize("held", [False, True], ids=["fp16 rows", "packed"])
def test_window_tree(T, window, sinks, held):
    """A tree's rows have windows of their own length before the drafts."""
    B = Long(T + window, [T, 1, T], [0, 300, 140], [0, 160, 512] if held else None, 4, 2, 128, T == 12, True, pad=1, window=window,
             sinks=sinks)
    B.mask[0] = 0  # a row without drafts, itself neither
    B.check(B.run())


@HALF
def test_window_long(half):
    """Long contexts through a window, split and joined."""
    B = Long(1, [1, 1], [4000, 13], [9600, 16000], 8, 4, 128, half, False, window=4000, sinks=4)
    B.check(B.run())
    B.check(B.run(max_len=16014))
    B.check(B.run(max_len=1))


@HALF
@pytest.mark.parametrize("T", [1, 5, 90])
@pytest.mark.parametrize("window", [0, 50])
def test_rows_that_see_nothing(half, T, window):
    """No positions before the step and empty mask lines: 0."""
    B = Long(T, [T, 1], [0, 3], [0, 64], 4, 2, 128, half, True, window=max(window, T) if window else 0)
    B.mask[:T] = 0
    got = B.run()
    assert (got[:T] == 0).all()
    B.check(got)


@pytest.mark.parametrize("vscale", [2.0 ** -30, 2.0 ** -10, 2.0 ** 12])
@pytest.mark.parametrize("T", [1, 6, 80])
def test_value_scales(T, vscale):
    """Values far from one: what a weight is held to goes with the blocks' own
    scales."""
    B = Long(T, [T], [0], [640], 4, 2, 64, False, False, vscale=vscale)
    B.v[:] *= np.float16(min(vscale, 1.0))
    B.check(B.run())


def test_zero_blocks():
    """Blocks of zeros with scale 0: their scores are 0 and count."""
    B = Long(3, [1, 40], [4, 3], [128, 320], 4, 2, 128, False, False)
    B.ks[:, :, 1], B.vs[:, :, 2] = 0, 0
    B.kn[:, :, 1], B.vn[:, :, 2] = 0, 0
    B.check(B.run())


@pytest.mark.parametrize("window,sinks", [(0, 0), (150, 70)])
@pytest.mark.parametrize("T", [1, 6, 80])
def test_scales_of_any_sign(T, window, sinks):
    """Blocks that a caller wrote by its own rule: negative scales, and zeros where
    a window begins and its first part ends."""
    B = Long(T + window, [T, 2], [4, 9], [320, 96], 4, 2, 64, False, T > 1, window=window, sinks=sinks)
    B.ks[:, :, 1::2] *= -1
    B.vs[:, 0] *= -1
    B.vs[:, 1, ::3] *= -1
    B.ks[:, :, 2] = B.ks[:, 1, 5] = B.vs[:, 1, 5] = 0
    B.check(B.run())


@pytest.mark.parametrize("T", [1, 80])
def test_blocks_past_32_bits(T):
    """Blocks whose bytes lie more than 2^32 behind the first: seen through a
    window, packed to and read back."""
    D, n = 64, (1 << 20) + 3
    B = Long(T, [1, T], [3, 10], [64, 192], 4, 1, D, False, False, window=100, sinks=5)
    small = B.tensors()["packed"]
    k, v = (torch.empty((2, 1, n, 32 * D), dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros((2, 1, n), device="cuda") for _ in range(2))
    assert k[1, 0, -5].data_ptr() - k.data_ptr() > 2 ** 32 - 2 ** 15 and k[1, 0, -1].data_ptr() - k.data_ptr() >= 2 ** 32
    for to, x in ((k, small.k), (v, small.v), (ks, small.k_scale), (vs, small.v_scale)):
        to[0, 0, :2], to[1, 0, 0], to[1, 0, -5:] = x[0, 0, :2], x[1, 0, 0], x[1, 0, 1:6]
    big = qa.PackedKV(k, v, ks, vs)
    B.check(B.run(packed=big, packed_len=i32([64, 32 * n])))

    s = Store(T, 2, 1, D, 70, 3)
    kv, _, cache, few = s.device()
    qa.kv_pack(cache, few, i32([0, 64]), i32([0, 32]))
    qa.kv_pack(qa.KVCache(dev(s.k), dev(s.v)), big, i32([0, 64]), i32([0, 32 * (n - 2)]))
    for got, want in ((k, few.k), (v, few.v), (ks, few.k_scale), (vs, few.v_scale)):
        assert torch.equal(got[1, 0, -2:], want[1, 0, 1:])
    back = [[torch.zeros_like(x) for x in kv] for _ in range(2)]
    qa.kv_unpack(few, i32([0, 96]), qa.KVCache(*back[0]), first=i32([0, 37]), count=70)
    qa.kv_unpack(big, i32([0, 32 * n]), qa.KVCache(*back[1]), first=i32([0, 32 * (n - 3) + 37]), count=70)
    for got, want in zip(back[1], back[0]):
        assert want[1, :, :59].any() and torch.equal(got, want)


@pytest.mark.parametrize("qscale", [1e-30, 300.0])
@pytest.mark.parametrize("T", [1, 40])
def test_query_sizes(T, qscale):
    B = Long(6, [T], [9], [160], 4, 2, 64, False, False, qscale=qscale)
    B.check(B.run())


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.7])
@pytest.mark.parametrize("T", [1, 20, 70])
def test_scale(T, scale):
    B = Long(7, [3, T], [50, 7], [96, 128], 4, 2, 64, False, True)
    B.check(B.run(scale=scale), scale=scale)


@HALF
@pytest.mark.parametrize("T", [1, 6, 70])
@pytest.mark.parametrize("window", [0, 100])
def test_nan_blocks_and_unseen_rows(half, T, window):
    """A block with a NaN scale makes the rows NaN that see a position of it, of
    its own kv head, and no others; what lies behind the lengths counts for
    nothing."""
    B = Long(T + window, [T, 1, T], [40, 10, 0], [320, 96, 480], 4, 2, 128, half, False, window=window, sinks=1 if window else 0)
    B.ks[0, 0, 3], B.vs[2, 1, 11] = np.nan, np.nan
    for b, (n, c, p) in enumerate(zip(B.rows, B.lens, B.packed)):
        B.k[b, :, c + n:], B.v[b, :, c + n:] = np.nan, np.inf
        B.ks[b, :, p // 32:], B.vs[b, :, p // 32:] = np.nan, np.nan
    got = B.run()

    def bad(b, t):  # of each kv head
        out = [False, False]
        seen = ref.seen_by(t, B.rows[b], B.packed[b] + B.lens[b], None, window, B.sinks)
        if b == 0:
            out[0] = any(96 <= j < 128 for j in seen)
        if b == 2:
            out[1] = any(352 <= j < 384 for j in seen)
        return out

    for b, n in enumerate(B.rows):
        for t in range(n):
            o = got[int(B.st[b]) + t].reshape(2, 2, 128)
            for h, is_bad in enumerate(bad(b, t)):
                assert np.isnan(o[h]).all() if is_bad else np.isfinite(o[h]).all(), (b, t, h)
    B.ks[0, 0, 3] = B.vs[2, 1, 11] = 1.0
    B.check(got, only=lambda b, t: not any(bad(b, t)))


@HALF
@pytest.mark.parametrize("T", [6, 90])
def test_unseen_infinities(half, T):
    """NaN and infinities in drafts that other rows see, and in another row's
    query: only rows that see them change."""
    B = Long(T, [T, 2], [9, 10], [96, 64], 4, 2, 128, half, True, window=128, sinks=2)
    B.v[0, 0, 10, 5], B.k[0, 1, 11, 7] = np.inf, np.nan
    B.q[0, 3] = np.nan
    got = B.run()
    B.check(got, only=lambda b, t: b == 1 or (t > 0 and not int(B.mask[t, 0]) & 6))
    assert np.isnan(got[0, :128]).all()


@pytest.mark.parametrize("T", [1, 40])
def test_windows_of_any_size(T):
    """The largest windows and first parts there are: everything is seen."""
    for window, sinks in ((2 ** 31 - 1, 0), (2 ** 31 - 1, 2 ** 31 - 1), (100, 2 ** 31 - 1)):
        B = Long(T, [T, 1], [40, 3], [320, 64], 4, 2, 64, False, T > 1, window=window, sinks=sinks)
        B.check(B.run())


def test_windows_leave_infinities_unseen():
    """NaN in fp16 rows that a window passes over, beside ones it holds."""
    for T in (1, 4, 70):
        B = Long(T, [T], [600], None, 4, 2, 128, False, False, window=64, sinks=3)
        B.k[0, :, 3:536 - T], B.v[0, :, 3:536 - T] = np.nan, np.nan
        B.check(B.run())


def test_sequences_that_do_not_fit():
    """Lengths out of range: NaN, and the others whole."""
    B = Long(12, [2, 3, 2, 1, 1, 40, 1, 2], [10, 20, 5, 8, 2, 3, 4, 5], [64, 0, 32, 64, 96, 0, 32, 64], 4, 2, 64, False, False, slack=0)
    lens, packed = list(B.lens), list(B.packed)
    lens[1], lens[2], packed[3], packed[4], packed[5] = B.S - 2, -1, 33, -32, 1 << 20
    for window, sinks in ((0, 0), (50, 2)):
        B.window, B.sinks = window, sinks
        got = B.run(cache_len=i32(lens), packed_len=i32(packed))
        bad = [1, 2, 3, 4, 5]
        for b in bad:
            assert np.isnan(got[B.st[b]:B.st[b + 1]]).all()
        B.check(got, only=lambda b, t: b not in bad)


def test_max_rows_and_broken_starts():
    B = Long(13, [6, 2], [10, 20], [64, 32], 4, 2, 64, False, False)
    got = B.run(max_rows=4)
    B.check(got, only=lambda b, t: t < 4)
    np.testing.assert_array_equal(got[4:6], B.out[4:6])
    B.check(B.run(row_start=i32([-5, 6, 1 << 30])))
    got = B.run(row_start=i32([0, 6, 3]))
    np.testing.assert_array_equal(got[6:], B.out[6:])
    B.check(np.concatenate([got[:6], B.run()[6:]]))


def test_layouts():
    """The cache by rows, one layer of several, and q and out as views of wider
    rows; out over q."""
    for T in (4, 80):
        B = Long(14, [T, 1], [66, 30], [96, 160], 6, 3, 128, False, True, window=100, sinks=2)
        want = B.run()
        B.check(want)
        c = [dev(x.transpose(0, 2, 1, 3)).transpose(1, 2) for x in (B.k, B.v)]
        np.testing.assert_array_equal(B.run(cache=qa.KVCache(*c)), want)
        N, W = B.q.shape
        wide = torch.zeros((N, 2 * W + 4), device="cuda")
        wide[:, 4:4 + W] = dev(B.q)
        ow = torch.full_like(wide, 7.0)
        np.testing.assert_array_equal(B.run(q=wide[:, 4:4 + W], out=ow[:, :W]), want)
        assert (ow[:, W:] == 7).all()
        x = dev(B.q)
        np.testing.assert_array_equal(B.run(q=x, out=x), want)
        p = B.tensors()["packed"]
        layers = [torch.stack([torch.zeros_like(t), t]) for t in (p.k, p.v, p.k_scale, p.v_scale)]
        np.testing.assert_array_equal(B.run(packed=qa.PackedKV(*[t[1] for t in layers])), want)


def test_without_blocks_or_window_as_tree_attention():
    """Over fp16 rows alone and without a window: what tree_attention gives, to
    both operators' tolerance."""
    for T, tree in ((1, False), (9, True), (200, False)):
        B = Long(T, [T, 1], [300, 20], None, 8, 4, 128, False, tree, pad=1)
        got = B.run()
        B.check(got)
        a = {n: v for n, v in B.tensors().items() if n not in ("window", "sinks")}
        B.check(qa.tree_attention(**a).cpu().numpy())


@pytest.mark.parametrize("H,Hk,D,T", [(64, 1, 128, 1), (33, 1, 64, 2), (28, 4, 128, 3)], ids=str)
def test_many_heads_of_one_kv_head(H, Hk, D, T):
    for half in (False, True):
        B = Long(H + T, [T, T, 1], [2, 70, 1], [2496, 0, 64], H, Hk, D, half, T > 1, pad=1)
        B.check(B.run())


def test_large_batch():
    rng = np.random.default_rng(4)
    rows = [int(n) for n in rng.integers(0, 2, 700)]
    rows[5] = 1
    B = Long(4, rows, [int(n) for n in rng.integers(0, 40, 700)], [int(n) * 32 for n in rng.integers(0, 4, 700)], 4, 2, 64, False, False,
             pad=2, window=60, sinks=3)
    B.check(B.run(), only=lambda b, t: b % 7 == 0 or b > 690)


def test_prompt_behind_packed_positions():
    for half in (False, True):
        B = Long(3 + half, [1500], [20], [1984], 4, 2, 128, half, False)
        B.check(B.run(), only=lambda b, t: t % 211 == 0 or t > 1495 or t in (31, 32, 63, 64, 127, 128))


def test_refused_by_the_bindings():
    B = Long(1, [2], [3], [32], 4, 2, 64, False, False)
    a = B.tensors()
    with pytest.raises(ValueError, match="come together"):
        qa.long_attention(**{**a, "packed_len": None})
    with pytest.raises(ValueError, match="packed_len must hold"):
        qa.long_attention(**{**a, "packed_len": i32([1, 2])})
    with pytest.raises(q.Q3VLError, match="without a window"):
        qa.long_attention(**a | {"sinks": 3})
    with pytest.raises(q.Q3VLError, match="heads of 128"):
        qa.long_attention(**{**a, "packed": qa.alloc_packed_kv(1, 2, 64, 128)})
    with pytest.raises(ValueError, match="on the current device"):
        qa.kv_pack(a["cache"], type("X", (), {"dev": -1})(), i32([1]), i32([0]))
    with pytest.raises(TypeError, match="torch.int32"):
        qa.kv_pack(a["cache"], a["packed"], torch.zeros(1, device="cuda"), i32([0]))
    with pytest.raises(q.Q3VLError, match="one array"):
        x = i32([1])
        qa.kv_advance(a["cache"], a["packed"], x, x)
    with pytest.raises(ValueError, match="their scales"):
        qa.PackedKV(a["packed"].k, a["packed"].v, a["packed"].k_scale, a["packed"].v_scale.repeat(1, 1, 2))
