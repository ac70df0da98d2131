"""GPU tests of the judging of drafts against its plain 64-bit form
(long_ref.verify), choice for choice: chains and trees, drafts with and without
probabilities, odd sizes, ruled-out tokens, rows that cannot be judged, broken
trees; and that the tokens come out with the target's distribution."""
import numpy as np
import pytest

import long_ref as ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import q3vl_int8 as q  # noqa: E402
from q3vl_int8 import attention as qa  # noqa: E402


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


class Drafts:
    def __init__(self, seed, rows, V, tree, probs, half=False, pad=0, spread=3.0, near=0.5):
        rng = self.rng = np.random.default_rng(seed)
        self.rows, self.V, self.half = rows, V, half
        self.start = np.concatenate([[0], np.cumsum(rows)])
        N = int(self.start[-1]) + pad
        x = rng.standard_normal((N, V)) * spread
        x[np.arange(N), rng.integers(0, V, N)] += np.abs(rng.standard_normal(N)) * 8
        self.x = x.astype(np.float16 if half else np.float32)
        par = [(-1 if t == 0 else int(t - 1 - np.floor(rng.random() ** 2 * t)) if tree else t - 1) for n in rows for t in range(n)]
        self.parents = np.array(par + [-1] * pad)
        d = np.exp(self.x.astype(np.float64) - self.x.max(1, keepdims=True) + near * rng.standard_normal((N, V)))
        d /= d.sum(1, keepdims=True)
        self.draft = d.astype(np.float32) if probs else None
        self.tokens = rng.integers(0, V, N)
        for b, n in enumerate(rows):
            for t in range(1, n):
                r = int(self.start[b]) + t
                self.tokens[r] = min(V - 1, int(np.searchsorted(np.cumsum(d[self.start[b] + self.parents[r]]), rng.random())))
        self.ua, self.us = (rng.random(N).astype(np.float32) for _ in range(2))
        self.T = max(max(rows), 1)

    def run(self, **over):
        i32 = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")  # noqa: E731
        a = dict(logits=dev(self.x), tokens=i32(self.tokens), parents=i32(self.parents), row_start=i32(self.start), accept_u=dev(self.ua),
                 sample_u=dev(self.us), max_rows=self.T, draft_probs=None if self.draft is None else dev(self.draft))
        r = qa.verify_drafts(**{**a, **over})
        torch.cuda.synchronize()
        return [t.cpu().numpy() for t in r]

    def check(self, max_rows=None, temperature=1.0, **over):
        got = self.run(max_rows=max_rows or self.T, temperature=temperature, **over)
        want = ref.verify(self.x, self.tokens, self.parents, self.start, self.ua, self.us, max_rows or self.T, self.draft, temperature)
        for g, w, n in zip(got, want, ("accepted", "path", "next")):
            np.testing.assert_array_equal(g, w, err_msg=n)
        return want


KINDS = [(t, p) for t in (False, True) for p in (False, True)]


@pytest.mark.parametrize("tree,probs", KINDS, ids=["chain", "chain probs", "tree", "tree probs"])
@pytest.mark.parametrize("V", [1, 2, 3, 63, 64, 65, 1000, 1024, 4099, 32000, 151936])
def test_sizes(V, tree, probs):
    rows = [4, 1, 0, 7, 2] if V > 5000 else [4, 1, 0, 7, 2, 61, 30, 1, 65]
    for half in (False, True):
        Drafts(V + half, rows, V, tree, probs, half, pad=2).check(temperature=0.8 if half else 1.0)


@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("V,rows", [(400_001, [4, 2]), (700_003, [7, 7])], ids=str)
def test_more_chunks_than_a_lane_keeps(V, rows, probs):
    """Rows of more chunks than the sums held in registers, small and large ones;
    flat ones, so that tokens come from all over them."""
    Drafts(V, rows, V, True, probs, spread=0.3, near=1.5).check()


@pytest.mark.parametrize("tree,probs", KINDS, ids=["chain", "chain probs", "tree", "tree probs"])
def test_paths_of_all_lengths(tree, probs):
    """Many sequences whose drafts are good: paths end everywhere."""
    want = Drafts(11, [9] * 150, 40, tree, probs, spread=2.0, near=0.2).check()
    assert len(set(want[0].tolist())) >= (4 if tree else 8)


@pytest.mark.parametrize("probs", [False, True])
def test_many_sequences(probs):
    """More sequences than a workgroup has threads, some of none."""
    Drafts(12, [1, 3, 0, 2, 5] * 130, 70, True, probs, pad=3).check()


@pytest.mark.parametrize("temperature", [1e-30, 1e-3, 7.5, 1e30])
def test_temperatures(temperature):
    """The largest logit alone, and all that are not ruled out alike."""
    for probs in (False, True):
        d = Drafts(13, [5] * 20, 600, True, probs)
        d.x[:, 1::3] = -np.inf
        d.check(temperature=temperature)


def test_many_children():
    """Rows with many children, tokens that come twice among them, all rejected
    now and then."""
    for seed in range(3):
        d = Drafts(seed, [1000, 300, 64, 65], 50, True, True, near=2.0)
        for b, n in enumerate(d.rows):
            s = int(d.start[b])
            d.parents[s + 1:s + n] = np.where(np.arange(1, n) < n // 2, 0, np.maximum(0, d.parents[s + 1:s + n]))
        d.check()
        d.draft = None
        d.check()


def test_ruled_out_tokens():
    """-inf logits: tokens of no probability are neither kept nor drawn; numbers
    at the ends of their range."""
    for probs in (False, True):
        d = Drafts(21, [3] * 60, 500, False, probs)
        d.x[:, ::2] = -np.inf
        d.us[::3], d.ua[::4] = 0.0, 0.0
        d.us[1::3], d.ua[1::4] = 1 - 2.0 ** -24, 1 - 2.0 ** -24
        want = d.check()
        assert (want[2] % 2 == 1).all()


def test_rows_that_cannot_be_judged():
    """A NaN, a +inf or nothing but -inf: the path ends there without a token."""
    for probs in (False, True):
        d = Drafts(22, [4] * 40, 300, False, probs, near=0.05)
        d.x[1::4][::3, 7] = np.nan
        d.x[2::4][::3, 8] = np.inf
        d.x[0::4][::5] = -np.inf
        want = d.check()
        assert (want[2] == -1).any() and (want[2] >= 0).any()


def test_finite_masks():
    """Masks of the type's lowest value count as no probability."""
    for half in (False, True):
        d = Drafts(23, [4] * 20, 300, True, True, half)
        d.x[:, 5::2] = np.finfo(d.x.dtype).min
        d.check()
        d.x[:] = np.finfo(d.x.dtype).min  # all the same: each as likely
        d.check()


def test_broken_trees_and_tokens():
    """Parents that are no earlier rows, tokens outside of the vocabulary, draft
    probabilities that are none: those rows do not stay, nothing else changes."""
    d = Drafts(24, [12, 9, 30], 100, True, True)
    d.parents[[3, 15, 25]] = [7, -9, 2 ** 31 - 1]
    d.parents[5] = 5
    d.tokens[[2, 14, 22]] = [-1, 100, 2 ** 31 - 1]
    d.draft[0, :20], d.draft[12, ::3], d.draft[21, 4] = -1.0, np.nan, np.inf
    d.check()
    d.draft = None
    d.tokens[13] = -1
    d.check()
    # starts outside of the rows are taken as the nearest row there is
    got = d.run(row_start=torch.tensor([-7, 12, 21, 1 << 30], dtype=torch.int32, device="cuda"))
    for g, w in zip(got, d.check()):
        np.testing.assert_array_equal(g, w)
    got = d.run(row_start=torch.tensor([0, 40, 10, 51], dtype=torch.int32, device="cuda"))  # not ascending: nothing out of bounds
    assert (got[0] <= d.T).all() and (got[1] < d.T).all()


def test_max_rows_cuts_a_sequence():
    d = Drafts(25, [9] * 30, 40, False, True, spread=1.0, near=0.05)
    d.check(max_rows=3)
    got = d.run(max_rows=0)
    assert (got[0] == 0).all() and got[1].shape == (30, 0) and (got[2] == -1).all()


def test_no_rows():
    d = Drafts(26, [1, 2], 10, False, False)
    empty = {n: dev(np.zeros(0, np.float32)) for n in ("accept_u", "sample_u")}
    got = d.run(logits=torch.zeros((0, 10), device="cuda"), tokens=dev(np.zeros(0, np.int32)), parents=dev(np.zeros(0, np.int32)),
                row_start=dev(np.zeros(4, np.int32)), **empty)
    assert (got[0] == 0).all() and (got[1] == -1).all() and (got[2] == -1).all()


def test_strided_rows():
    d = Drafts(27, [5, 6], 1001, True, True)
    x, p = torch.full((11, 1100), float("nan"), device="cuda"), torch.full((11, 1003), float("nan"), device="cuda")
    x[:, 50:1051], p[:, 1:1002] = dev(d.x), dev(d.draft)
    want = d.check()
    for g, w in zip(d.run(logits=x[:, 50:1051], draft_probs=p[:, 1:1002]), want):
        np.testing.assert_array_equal(g, w)


def test_equal_distributions_always_stay():
    """A draft drawn from the target itself (in fp32) stays unless the numbers
    fall on the last bits."""
    d = Drafts(28, [8] * 20, 2000, False, True, near=0.0)
    assert (d.check()[0] >= 7).all()


@pytest.mark.parametrize("probs", [False, True])
def test_distribution(probs):
    """The first token after the root, kept or drawn, has the target's
    distribution: 40000 sequences of one tree, five sigma."""
    rng = np.random.default_rng(29)
    n, V, T = 40000, 7, 4
    x = rng.standard_normal((T, V)).astype(np.float32)
    p = np.exp(x[0] * 1.0) / np.exp(x[0]).sum()
    dr = np.exp(rng.standard_normal((T, V)))
    dr = (dr / dr.sum(1, keepdims=True)).astype(np.float32)
    tok = rng.integers(0, V, (n, T))
    if probs:  # three children, drawn one by one
        cum = np.cumsum(dr[0].astype(np.float64))
        tok[:, 1:] = np.minimum(np.searchsorted(cum / cum[-1], rng.random((n, 3)), side="right"), V - 1)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    u = [dev(rng.random(n * T).astype(np.float32)) for _ in range(2)]
    r = qa.verify_drafts(dev(np.tile(x, (n, 1))), i32(tok.reshape(-1)), i32(np.tile([-1, 0, 0, 0], n)), i32(np.arange(n + 1) * T), *u, T,
                         draft_probs=dev(np.tile(dr, (n, 1))) if probs else None)
    path, acc, nxt = (t.cpu().numpy() for t in (r.path, r.accepted, r.next))
    first = np.where(acc > 1, tok[np.arange(n), np.maximum(path[:, 1], 0)], nxt)
    f = np.bincount(first, minlength=V) / n
    assert (np.abs(f - p) < 5 * np.sqrt(p * (1 - p) / n)).all(), (f, p)


def test_captured_on_other_streams_and_twice():
    """Captured with its own workspace and replayed over other inputs; two calls
    at once on two streams; without a workspace the library's own."""
    sets = [Drafts(31, [6, 3, 8], 5000, True, True), Drafts(32, [9] * 4, 3000, False, False, True)]
    keep = []
    for d in sets:
        i32 = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")  # noqa: E731
        a = dict(logits=dev(d.x), tokens=i32(d.tokens), parents=i32(d.parents), row_start=i32(d.start), accept_u=dev(d.ua),
                 sample_u=dev(d.us), max_rows=d.T, draft_probs=None if d.draft is None else dev(d.draft),
                 workspace=qa.alloc_verify_drafts_workspace(*d.x.shape))
        keep.append(a)
        qa.verify_drafts(**a)
    torch.cuda.synchronize()
    graphs = []
    for a in keep:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            with pytest.raises(q.Q3VLError, match="needs a workspace of its own"):
                qa.verify_drafts(**{**a, "workspace": None})
            out = qa.verify_drafts(**a)
        graphs.append((g, out))
    for turn in range(3):
        for a in keep:
            a["accept_u"].copy_(a["accept_u"].roll(turn))
            a["sample_u"].copy_(a["sample_u"].flip(0))
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        got = [[t.clone() for t in out] for _, out in graphs]
        for a, have in zip(keep, got):
            for x, y in zip(have, qa.verify_drafts(**{**a, "workspace": None})):
                assert torch.equal(x, y)
    want = [[t.clone() for t in qa.verify_drafts(**a)] for a in keep]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in keep]
    runs = [[], []]
    for _ in range(10):
        for i, (a, s) in enumerate(zip(keep, streams)):
            runs[i].append(qa.verify_drafts(**a, stream=s))
    torch.cuda.synchronize()
    for r, w in zip(runs, want):
        for out in r:
            assert all(torch.equal(x, y) for x, y in zip(out, w))


def test_bindings_refuse():
    d = Drafts(33, [3], 10, False, True)
    with pytest.raises(ValueError, match="logits' shape"):
        d.run(draft_probs=dev(d.draft[:2]))
    with pytest.raises(TypeError, match="draft_probs"):
        d.run(draft_probs=dev(d.draft.astype(np.float64)))
    with pytest.raises(ValueError, match="accept_u must hold 3"):
        d.run(accept_u=dev(d.ua[:2]))
    with pytest.raises(ValueError, match="max_rows"):
        d.run(max_rows=-1)
    with pytest.raises(ValueError, match="at least one"):
        d.run(row_start=torch.zeros(0, dtype=torch.int32, device="cuda"))
    with pytest.raises(q.Q3VLError, match="temperature"):
        d.run(temperature=0.0)
    with pytest.raises(ValueError, match="workspace must be"):
        d.run(workspace=torch.zeros(4096, dtype=torch.uint8))
