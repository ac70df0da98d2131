"""A step of the operators for rows of tokens together, as a program uses them:
a tree of drafts checked against the tokens that the decode step generates one
by one, the accepted rows moved, and decoding continued from there; the step
captured into a graph and replayed over other lengths; calls on two streams at
once; the same call twice."""
import numpy as np
import pytest

from golden.gen import SMALL, make_kv_cache, make_text_model

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import q3vl_int8 as q  # noqa: E402
from q3vl_int8 import attention as qa  # noqa: E402
from q3vl_int8 import model as qm  # noqa: E402


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Rows:
    """The text model over several rows: its linears, and the operators."""

    def __init__(self, dims, arrays, k, v):
        self.d, self.t = dims, {n: torch.from_numpy(a).cuda() for n, a in arrays.items()}
        t, gs = self.t, dims["gs"]
        self.caches = [qa.KVCache(k[l][None], v[l][None]) for l in range(dims["layers"])]
        self.norms = [qa.QKNorm(t["qnorm_w"][l], t["qnorm_s"][l], t["knorm_w"][l], t["knorm_s"][l], gs, dims["eps"])
                      for l in range(dims["layers"])]
        self.rope = qa.Rope(t["rope_cos"], t["rope_sin"])

    def norm(self, x, name, l=None):
        w, s = self.t[name + "_w"], self.t[name + "_s"]
        w, s = (w, s) if l is None else (w[l], s[l])
        g = w.float() * s.repeat_interleave(self.d["gs"])
        return (x / (x.square().mean(1, keepdim=True) + self.d["eps"]).sqrt() * g).contiguous()

    def step(self, tokens, parents, row_start, cache_len, max_rows):
        d, t, gs = self.d, self.t, self.d["gs"]
        mask, pos, slots = qa.draft_plan(parents, row_start, cache_len, d["max_seq"], max_rows)
        e, s = t["emb_w"][tokens.long()], t["emb_s"][tokens.long()]
        x = e.float() * s.repeat_interleave(gs, 1)
        for l in range(d["layers"]):
            qkv = q.linear_i8_multi(self.norm(x, "anorm", l), [t["w" + n][l] for n in "qkv"], [t["s" + n][l] for n in "qkv"], gs)
            qr = qa.qk_norm_rope(*qkv, self.caches[l], slots, pos, self.norms[l], self.rope)
            a = qa.tree_attention(qr, self.caches[l], row_start, cache_len, max_rows, mask=mask)
            x = x + q.linear_i8(a, t["wo"][l], t["so"][l], gs)
            y = self.norm(x, "mnorm", l)
            x = x + q.mlp_i8(y, t["wg"][l], t["sg"][l], t["wu"][l], t["su"][l], t["wd"][l], t["sd"][l], gs)
        return q.linear_i8(self.norm(x, "fnorm"), t["emb_w"], t["emb_s"], gs)


def test_drafts_checked_against_decode_steps():
    """Row by row the tree's logits are the decode step's: to 1 % of their norm.
    (The two differ where an int16 activation rounds the other way, 2^-7 of a
    group's rms in about one of 10^4, and by the decode step's exponential, a
    few 10^-4 of the attention's output; over 14 products of two layers that is
    a few 10^-3.) Where the first two logits are apart by 5 % of their spread,
    the drafted token that the decode step chose has rank 0."""
    dims, ctx, steps = dict(SMALL), 57, 5
    arrays = make_text_model(17, dims)
    k16, v16 = make_kv_cache(18, dims, ctx)
    dev = lambda a: torch.from_numpy(a.view(np.int16).copy()).cuda()  # noqa: E731
    k, v = dev(k16), dev(v16)
    model = qm.DeviceTextModel(dims, arrays)
    ws = qm.alloc_decode_workspace(model)
    tok, pos, logits = i32([7]), i32([ctx]), torch.zeros(dims["vocab"], device="cuda")
    chosen, want = [7], []
    for _ in range(steps + 1):
        qm.decode_step(model, k, v, tok, pos, logits, ws)
        want.append(logits.clone())
        chosen.append(int(tok.item()))
    # the same tokens as one branch of a tree, with others beside them
    tokens = [7, 99, chosen[1], chosen[2], 1234, 55, chosen[3], chosen[4], 4095]
    parents = [-1, 0, 0, 2, 2, 4, 3, 6, 6]
    path = [0, 2, 3, 6, 7]
    k2, v2 = (dev(a).view(torch.float16) for a in (k16, v16))
    rows = Rows(dims, arrays, k2, v2)
    got = rows.step(i32(tokens), i32(parents), i32([0, 9]), i32([ctx]), 9)
    r = q.token_logprobs(got, i32([chosen[i + 1] if j in path and (i := path.index(j)) is not None else 0 for j in range(9)]), top_k=2)
    for i, j in enumerate(path):
        w = want[i].double()
        assert float((got[j].double() - w).norm() / w.norm()) < 1e-2, (i, j)
        first, second = torch.topk(w, 2).values.tolist()
        if first - second > 0.05 * float(w.std()):
            assert int(r.rank[j]) == 0 and int(r.top_ids[j, 0]) == chosen[i + 1]
        exact = torch.log_softmax(got[j].double(), 0)
        assert abs(float(r.logprob[j]) - float(exact[chosen[i + 1]])) <= 1e-5 * max(1.0, abs(float(exact[chosen[i + 1]])))
    # the accepted rows to their places, and on from there: the decode step
    # gives what it gave on its own path
    for c in (k2, v2):
        c[:, :, ctx:ctx + len(path)] = c[:, :, [ctx + j for j in path]].clone()
    tok.fill_(chosen[len(path)])
    pos.fill_(ctx + len(path))
    qm.decode_step(model, k2.view(torch.int16), v2.view(torch.int16), tok, pos, logits, ws)
    w = want[len(path)].double()
    assert float((logits.double() - w).norm() / w.norm()) < 1e-2


def make_step(seed, B=3, T=9, S=700, H=8, Hk=4, D=128, V=3000):
    """One layer's operators and the scoring over their own tensors."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    N = B * T
    st = {"parents": torch.tensor([max(-1, t - 1 - t % 3) for _ in range(B) for t in range(T)], dtype=torch.int32, device="cuda"),
          "row_start": i32([T * b for b in range(B + 1)]), "cache_len": i32([100 * b + 5 for b in range(B)]),
          "q": randn(N, H * D), "k": randn(N, Hk * D), "v": randn(N, Hk * D), "logits": randn(N, V) * 3,
          "tokens": torch.randint(0, V, (N,), device="cuda", generator=g, dtype=torch.int32),
          "kc": randn(B, Hk, S, D).half(), "vc": randn(B, Hk, S, D).half()}
    w = lambda: torch.randint(50, 127, (D,), device="cuda", generator=g, dtype=torch.int8)  # noqa: E731
    s = lambda: torch.rand(D // 64, device="cuda", generator=g) * 0.01 + 0.005  # noqa: E731
    st["norm"] = qa.QKNorm(w(), s(), w(), s(), 64, 1e-6)
    a = torch.arange(S, device="cuda")[:, None] * 0.01 * torch.rand((1, D // 2), device="cuda", generator=g)
    st["rope"] = qa.Rope(a.cos(), a.sin())
    st["cache"] = qa.KVCache(st["kc"], st["vc"])
    st["ws"] = qa.alloc_tree_attention_workspace(st["cache"], N, H, T, S)
    st["lws"] = q.alloc_token_logprobs_workspace(N, V)
    st["T"], st["S"] = T, S
    return st


def run_step(st, stream=None):
    mask, pos, slots = qa.draft_plan(st["parents"], st["row_start"], st["cache_len"], st["S"], st["T"], stream=stream)
    qr = qa.qk_norm_rope(st["q"], st["k"], st["v"], st["cache"], slots, pos, st["norm"], st["rope"], stream=stream)
    o = qa.tree_attention(qr, st["cache"], st["row_start"], st["cache_len"], st["T"], mask=mask, max_len=st["S"],
                          workspace=st["ws"], stream=stream)
    r = q.token_logprobs(st["logits"], st["tokens"], top_k=7, workspace=st["lws"], stream=stream)
    return [mask, pos, slots, qr, o, *r]


def same(a, b):
    return all(torch.equal(x.view(torch.uint8) if x.numel() else x, y.view(torch.uint8) if y.numel() else y) for x, y in zip(a, b))


def test_the_same_call_twice():
    st = make_step(1)
    a = [x.clone() for x in run_step(st)]
    b = run_step(st)
    torch.cuda.synchronize()
    assert same(a, b)


def test_captured_step_replays_over_other_lengths():
    """Lengths, trees and inputs are read at replay: each replay equals the
    eager call, with eager work and waits between, and two graphs with
    workspaces of their own do not disturb each other."""
    one, two = make_step(2), make_step(3, B=2, T=20)
    graphs = []
    for st in (one, two):
        run_step(st)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run_step(st)
        graphs.append((g, out))
    for turn in range(4):
        for st in (one, two):
            st["cache_len"].add_(31 * turn)
            st["q"].mul_(1.1)
            st["logits"].add_(0.25)
            st["tokens"].copy_(st["tokens"].roll(1))
        if turn == 2:
            one["row_start"].copy_(i32([0, 4, 4, 20]))  # fewer rows: the rest hold no token
            one["parents"].fill_(-1)
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        got = [[x.clone() for x in out] for _, out in graphs]
        for (st, out), have in zip(((one, graphs[0][1]), (two, graphs[1][1])), got):
            live = int(st["row_start"][-1])
            eager = run_step(st)
            torch.cuda.synchronize()
            for i, (x, y) in enumerate(zip(have, eager)):
                if i in (3, 4):  # rows without a token are left as they were
                    x, y = x[:live], y[:live]
                assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)), (turn, i)


def test_calls_on_two_streams():
    """Two batches at once, each on a stream of its own with its workspaces."""
    sts = [make_step(5, T=30), make_step(6, B=2, T=3)]
    want = []
    for st in sts:
        want.append([x.clone() for x in run_step(st)])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sts]
    got = [[], []]
    for _ in range(20):
        for i, (st, s) in enumerate(zip(sts, streams)):
            got[i].append(run_step(st, stream=s))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            assert same(g, want[i])
    # ... and on the current stream where that is another one
    with torch.cuda.stream(streams[0]):
        g = run_step(sts[0])
    torch.cuda.synchronize()
    assert same(g, want[0])


def test_workspace_of_the_library():
    """Without a workspace the library's own buffer serves: the same bits."""
    st = make_step(8)
    want = [x.clone() for x in run_step(st)]
    st["ws"] = st["lws"] = None
    assert same(run_step(st), want)
    torch.cuda.synchronize()


def test_too_small_a_workspace_is_refused():
    st = make_step(9, S=6000)
    assert st["ws"].numel() > 256
    st["ws"] = st["ws"][:256]
    with pytest.raises(q.Q3VLError, match="workspace too small"):
        run_step(st)
    torch.cuda.synchronize()


def test_bindings_refuse_what_does_not_fit():
    st = make_step(10)
    with pytest.raises(ValueError, match="row_start must hold"):
        qa.tree_attention(st["q"], st["cache"], st["row_start"][:-1], st["cache_len"], st["T"])
    with pytest.raises(ValueError, match="line for each row"):
        qa.tree_attention(st["q"], st["cache"], st["row_start"], st["cache_len"], st["T"],
                          mask=torch.zeros((2, 1), dtype=torch.int64, device="cuda"))
    with pytest.raises(TypeError, match="torch.float32 or torch.float16"):
        qa.tree_attention(st["q"].double(), st["cache"], st["row_start"], st["cache_len"], st["T"])
    with pytest.raises(TypeError, match="torch.float32"):
        qa.tree_attention(st["q"], st["cache"], st["row_start"], st["cache_len"], st["T"], out=st["q"].half())
    with pytest.raises(ValueError, match="contiguous rows"):
        q.token_logprobs(st["logits"].t(), st["tokens"])
    with pytest.raises(ValueError, match="16-byte aligned"):
        x = torch.zeros((1, 1, 8, 132), dtype=torch.float16, device="cuda")[..., :128]
        qa.KVCache(x, x)
    with pytest.raises(ValueError, match="shape mismatch"):
        qa.qk_norm_rope(st["q"], st["k"][:, :128], st["v"], st["cache"], st["tokens"].long(), st["tokens"], st["norm"], st["rope"])
    with pytest.raises(q.Q3VLError, match="top_k=65"):
        q.token_logprobs(st["logits"], st["tokens"], top_k=65)


def test_captured_calls_need_their_own_workspace():
    """The library's buffer may be freed to grow it, and a graph would keep its
    address: refused, while the capture goes on; a call that needs none is
    captured."""
    st = make_step(11)
    attn = lambda cache, rows, **kw: qa.tree_attention(st["q"], cache, st["row_start"], st["cache_len"], rows, **kw)  # noqa: E731
    ws = st["ws"]
    assert ws.numel() > 256  # the attention of this step is split
    want = [x.clone() for x in run_step(st)]
    st["ws"] = st["lws"] = None
    run_step(st)  # the library's buffer is large enough
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(q.Q3VLError, match="needs a workspace of its own"):
            attn(st["cache"], st["T"], max_len=st["S"])
        with pytest.raises(q.Q3VLError, match="needs a workspace of its own"):
            q.token_logprobs(st["logits"], st["tokens"], top_k=3)
        unsplit = attn(st["cache"], st["T"], max_len=1)
        split = attn(st["cache"], st["T"], max_len=st["S"], workspace=ws)
    eager = attn(st["cache"], st["T"], max_len=1).clone(), attn(st["cache"], st["T"], max_len=st["S"], workspace=ws).clone()
    for _ in range(3):
        unsplit.zero_(), split.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(unsplit, eager[0]) and torch.equal(split, eager[1])
    assert same(run_step(st), want)


def test_workspaces_that_no_kernel_may_write():
    """A host tensor, or every other byte of one: refused before the launch."""
    st = make_step(12)
    n = st["ws"].numel()
    for ws in (torch.empty(n, dtype=torch.uint8), torch.empty(n, dtype=torch.uint8).pin_memory(),
               torch.empty((n, 2), dtype=torch.uint8, device="cuda")[:, 0], 4096):
        with pytest.raises(ValueError, match="workspace must be"):
            qa.tree_attention(st["q"], st["cache"], st["row_start"], st["cache_len"], st["T"], max_len=st["S"], workspace=ws)
        with pytest.raises(ValueError, match="workspace must be"):
            q.token_logprobs(st["logits"], st["tokens"], workspace=ws)
