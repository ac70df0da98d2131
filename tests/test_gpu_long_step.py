"""The operators for long contexts and judged drafts together, as a program uses
them: trees of drafts planned, written, attended to and judged, the rows that
stay moved, whole blocks packed, over many steps; a step captured into a graph
and replayed; two of them at once; calls on several streams."""
import numpy as np
import pytest

import long_ref as ref
import rows_ref
from long_ref import within

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import q3vl_int8 as q  # noqa: E402
from q3vl_int8 import attention as qa  # noqa: E402


def i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


class Stream:
    """One layer of a batch: its newest rows, its blocks, its lengths."""

    def __init__(self, seed, B=3, H=4, Hk=2, D=64, S=70, positions=256, V=50):
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        self.B, self.H, self.Hk, self.D, self.S, self.V = B, H, Hk, D, S, V
        self.k, self.v = (torch.zeros((B, Hk, S, D), dtype=torch.float16, device="cuda") for _ in range(2))
        self.cache, self.packed = qa.KVCache(self.k, self.v), qa.alloc_packed_kv(B, Hk, positions, D)
        self.cache_len, self.packed_len = i32([0] * B), i32([0] * B)
        w = lambda: torch.randint(50, 127, (D,), device="cuda", generator=self.g, dtype=torch.int8)  # noqa: E731
        s = lambda: torch.rand(D // 64, device="cuda", generator=self.g) * 0.01 + 0.005  # noqa: E731
        self.norm = qa.QKNorm(w(), s(), w(), s(), 64, 1e-6)
        a = torch.arange(positions + S, device="cuda")[:, None] * 0.1 * torch.rand((1, D // 2), device="cuda", generator=self.g)
        self.rope = qa.Rope(a.cos(), a.sin())

    def randn(self, *s):
        return torch.randn(s, device="cuda", generator=self.g)

    def inputs(self, N):
        return [self.randn(N, n * self.D) for n in (self.H, self.Hk, self.Hk)]

    def layer(self, qkv, parents, row_start, T, window=0, sinks=0, ws=None, stream=None):
        mask, pos, slots = qa.draft_plan(parents, row_start, self.cache_len, self.S, T, pos_delta=self.packed_len, stream=stream)
        qr = qa.qk_norm_rope(*qkv, self.cache, slots, pos, self.norm, self.rope, stream=stream)
        o = qa.long_attention(qr, self.cache, row_start, self.cache_len, T, packed=self.packed, packed_len=self.packed_len, window=window,
                              sinks=sinks, mask=mask, workspace=ws, stream=stream)
        return mask, pos, qr, o

    def settle(self, stream=None):
        qa.kv_pack(self.cache, self.packed, self.cache_len, self.packed_len, stream=stream)
        qa.kv_advance(self.cache, self.packed, self.cache_len, self.packed_len, stream=stream)


@pytest.mark.parametrize("window,sinks", [(0, 0), (48, 2)], ids=str)
def test_many_steps(window, sinks):
    """40 steps of trees: each row's attention is that over the history that the
    paths so far have left, rounded to 8 bits where its block was packed; at the
    end what is read back is that history."""
    st = Stream(1)
    rng = np.random.default_rng(2)
    B, T, N, V = st.B, 7, 3 * 7, st.V
    hist = [[np.zeros((st.Hk, 0, st.D)) for _ in range(2)] for _ in range(B)]  # 64-bit values of kept positions
    held = [0] * B
    row_start = i32([0, 7, 14, 21])
    for step in range(40):
        parents = np.concatenate([[-1] + [int(rng.integers(0, t)) for t in range(1, T)] for _ in range(B)])
        mask, pos, qr, o = st.layer(st.inputs(N), i32(parents), row_start, T, window, sinks)
        logits, tokens = st.randn(N, V) * 2, torch.randint(0, V, (N,), device="cuda", generator=st.g, dtype=torch.int32)
        u = [torch.rand(N, device="cuda", generator=st.g) for _ in range(2)]
        probs = torch.softmax(logits + st.randn(N, V), 1)
        r = qa.verify_drafts(logits, tokens, i32(parents), row_start, *u, T, draft_probs=probs)
        acc, path = r.accepted.tolist(), r.path.tolist()
        want = ref.verify(logits.cpu().numpy(), tokens.cpu().numpy(), parents, [0, 7, 14, 21], u[0].cpu().numpy(), u[1].cpu().numpy(), T,
                          probs.cpu().numpy())
        assert acc == want[0].tolist() and path == want[1].tolist() and r.next.tolist() == want[2].tolist()
        lens = st.cache_len.tolist()
        assert st.packed_len.tolist() == held
        new = [x.cpu().numpy().astype(np.float64) for x in (st.k, st.v)]
        got, qn, m = o.cpu().numpy(), qr.cpu().numpy(), mask.cpu().numpy().view(np.uint64)
        for b in range(B):
            assert held[b] + lens[b] == hist[b][0].shape[1]
            kv = [np.concatenate([hist[b][i], new[i][b, :, lens[b]:lens[b] + T]], 1) for i in range(2)]
            for t in range(T):
                row = b * T + t
                depth = bin(int(m[row, 0])).count("1") - 1
                assert int(pos[row]) == held[b] + lens[b] + depth
                seen = ref.seen_by(t, T, held[b] + lens[b], m[row], window, sinks)
                want_o, absv, qk = rows_ref.attention(qn[row].reshape(st.H, st.D), *kv, seen, st.D ** -0.5)
                vmax = float(np.abs(hist[b][1][:, :held[b]]).max()) if held[b] else 0.0
                within(got[row].reshape(st.H, st.D), want_o, ref.attention_tolerance(absv, qk, st.D, len(seen), False, vmax), (step, b, t))
        for b in range(B):  # the rows that stay, to their places
            rows = path[b][:acc[b]]
            for i, x in enumerate((st.k, st.v)):
                x[b, :, lens[b]:lens[b] + acc[b]] = x[b, :, [lens[b] + j for j in rows]].clone()
                hist[b][i] = np.concatenate([hist[b][i], new[i][b][:, [lens[b] + j for j in rows]]], 1)
        st.cache_len += r.accepted
        st.settle()
        for b in range(B):
            n = (lens[b] + acc[b]) // 32
            for i in range(2):
                for j in range(n):
                    at = held[b] + 32 * j
                    w, s = ref.quantise(hist[b][i][:, at:at + 32].astype(np.float16))
                    hist[b][i][:, at:at + 32] = w * s.astype(np.float64)[:, None, None]
            held[b] += 32 * n
        assert st.packed_len.tolist() == held and (st.cache_len < 32).all()
    assert min(held) >= 32
    back = [torch.zeros((B, st.Hk, 256, st.D), dtype=torch.float16, device="cuda") for _ in range(2)]
    qa.kv_unpack(st.packed, st.packed_len, qa.KVCache(*back))
    for b in range(B):
        for i in range(2):
            h = hist[b][i][:, :held[b]]
            np.testing.assert_array_equal(back[i][b, :, :held[b]].cpu().numpy(), h.astype(np.float32).astype(np.float16))
            assert (back[i][b, :, held[b]:] == 0).all()
            tail = (st.k, st.v)[i][b, :, :int(st.cache_len[b])].cpu().numpy()
            np.testing.assert_array_equal(tail, hist[b][i][:, held[b]:].astype(np.float16))


def one_step(st, qkv, row_start, parents, ws=None, window=0, sinks=0, stream=None):
    out = st.layer(qkv, parents, row_start, 1, window, sinks, ws, stream)
    st.cache_len.add_(1)
    st.settle(stream)
    return [out[1], out[2], out[3]]


def copy_state(to, frm):
    for n in ("k", "v", "cache_len", "packed_len"):
        getattr(to, n).copy_(getattr(frm, n))
    for n in ("k", "v", "k_scale", "v_scale"):
        getattr(to.packed, n).copy_(getattr(frm.packed, n))


def state_of(st):
    return [st.k, st.v, st.cache_len, st.packed_len, st.packed.k, st.packed.v, st.packed.k_scale, st.packed.v_scale]


def same(a, b):
    return all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a, b))


def test_captured_steps():
    """Two streams of different sizes, each a graph of one token's step with a
    workspace of its own, replayed in turn over lengths that pass whole blocks:
    every replay leaves what the eager step leaves, bit for bit."""
    graphs = []
    for seed, kw, win in ((3, {}, (0, 0)), (4, dict(B=2, H=16, Hk=8, D=128, S=40, positions=640), (100, 3))):
        st, eager = Stream(seed, **kw), Stream(seed, **kw)
        qkv = st.inputs(st.B)
        row_start, parents = i32(range(st.B + 1)), i32([-1] * st.B)
        ws = qa.alloc_long_attention_workspace(st.cache, st.B, st.H, 1, packed=st.packed, window=win[0], sinks=win[1])
        # some history
        st.packed_len.fill_(64)
        st.cache_len.copy_(i32([5, 31, 29][:st.B]))
        st.packed.k.random_(-127, 128), st.packed.v.random_(-127, 128)
        st.packed.k_scale.uniform_(0.01, 0.02), st.packed.v_scale.uniform_(0.01, 0.02)
        st.k.normal_(), st.v.normal_()
        copy_state(eager, st)
        one_step(eager, qkv, row_start, parents, ws, *win)
        copy_state(eager, st)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = one_step(st, qkv, row_start, parents, ws, *win)
        copy_state(st, eager)
        graphs.append((g, out, st, eager, qkv, row_start, parents, win))
    for turn in range(40):
        for g, _, st, _, qkv, *_ in graphs:
            for x in qkv:
                x.add_(0.1 * (turn % 5 - 2))
        torch.cuda.synchronize()
        for g, *_ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for g, out, st, eager, qkv, row_start, parents, win in graphs:
            want = one_step(eager, qkv, row_start, parents, None, *win)
            torch.cuda.synchronize()
            assert same(out, want), turn
            assert same(state_of(st), state_of(eager)), turn
    assert all((g[2].packed_len >= 96).all() for g in graphs)


def test_streams():
    """Two batches at once, each on a stream of its own with its workspace."""
    sts, want = [], []
    for seed, kw in ((5, dict(S=300, positions=640)), (6, dict(B=2, H=16, Hk=8, D=128, positions=2048))):
        st = Stream(seed, **kw)
        st.packed_len.fill_(512)
        st.cache_len.fill_(20)
        st.packed.k.random_(-127, 128), st.packed.v.random_(-127, 128)
        st.packed.k_scale.fill_(0.01), st.packed.v_scale.fill_(0.02)
        st.k.normal_(), st.v.normal_()
        a = (st.inputs(st.B), i32(range(st.B + 1)), i32([-1] * st.B))
        ws = qa.alloc_long_attention_workspace(st.cache, st.B, st.H, 1, packed=st.packed)
        sts.append((st, a, ws))
        start = Stream(seed, **kw)
        copy_state(start, st)
        ref_state = Stream(seed, **kw)
        copy_state(ref_state, st)
        outs = [[x.clone() for x in one_step(ref_state, *a, ws)] for _ in range(15)]
        want.append((outs, [x.clone() for x in state_of(ref_state)]))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sts]
    got = [[], []]
    for _ in range(15):
        for i, ((st, a, ws), s) in enumerate(zip(sts, streams)):
            with torch.cuda.stream(s):
                got[i].append(one_step(st, *a, ws))
    torch.cuda.synchronize()
    for i in range(2):
        for x, y in zip(got[i], want[i][0]):
            assert same(x, y)
        assert same(state_of(sts[i][0]), want[i][1])
    # ... and given as an argument
    st, a, ws = sts[0]
    before = Stream(5, S=300, positions=640)
    copy_state(before, st)
    torch.cuda.synchronize()
    x = st.layer(*([a[0], a[2], a[1]]), 1, ws=ws, stream=streams[1])
    torch.cuda.synchronize()
    y = before.layer(*([a[0], a[2], a[1]]), 1, ws=ws)
    assert same(x, y)


def test_workspaces():
    """Without a workspace the library's own serves, but not while a graph is
    captured; too small a one is refused."""
    st = Stream(7, B=1, H=16, Hk=8, D=128, positions=4096)
    st.packed_len.fill_(4000), st.cache_len.fill_(20)
    st.k.normal_(), st.v.normal_(), st.packed.k_scale.fill_(0.01)
    x = st.randn(1, 16 * 128)
    args = (x, st.cache, i32([0, 1]), st.cache_len, 1)
    kw = dict(packed=st.packed, packed_len=st.packed_len)
    ws = qa.alloc_long_attention_workspace(st.cache, 1, 16, 1, packed=st.packed)
    assert ws.numel() > 256
    want = qa.long_attention(*args, **kw, workspace=ws)
    assert torch.equal(qa.long_attention(*args, **kw), want)
    with pytest.raises(q.Q3VLError, match="workspace too small"):
        qa.long_attention(*args, **kw, workspace=ws[:256])
    with pytest.raises(ValueError, match="workspace must be"):
        qa.long_attention(*args, **kw, workspace=torch.empty(ws.numel(), dtype=torch.uint8))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(q.Q3VLError, match="needs a workspace of its own"):
            qa.long_attention(*args, **kw)
        out = qa.long_attention(*args, **kw, workspace=ws)
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
