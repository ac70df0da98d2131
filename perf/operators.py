"""Timed cases of the operators for rows of tokens over the caches: a draft's
plan, head norms with the rotary position, attention over a cache, and the log
probabilities of given tokens. They are what a step over several rows needs
beside the linears: a prompt, a batch of sequences, or a tree of drafted tokens
that is checked in one pass.

Each operator has its plain form here (elementary torch operations in 32 bits,
or 64 where a long sum asks for it), the framework's call, and its definition
in 64 bits. The head layout 16 / 8 of 128, the vocabulary 151936 and groups of
64 are the text decoder's that perf/cases.py times; `draw` takes others too.

Kinds:
  plan   ancestor masks, positions and cache slots of every sequence's draft
  rope   RMS norm of each query and key head, rotation by one position or by
         three (time, height, width), keys and values stored to the cache
  attn   the rows of a batch over their caches: a chain, or a tree of drafts
  logp   log probability, rank, entropy and best alternatives per row of logits
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

HEADS, KV_HEADS, HEAD_DIM, VOCAB, THETA, EPS, GS = 16, 8, 128, 151936, 5e6, 1e-6, 64
SECTIONS = {64: (12, 10, 10), 128: (24, 20, 20)}  # frequencies by time, height and width


def listed():
    return [
        # a few sequences with small trees, one word of mask a row
        {"name": "plan_b8_t32", "kind": "plan", "B": 8, "T": 32},
        # a full serving batch with wide trees
        {"name": "plan_b96_t500", "kind": "plan", "B": 96, "T": 500},
        # one new token of each of four sequences: latency alone
        {"name": "rope_m4", "kind": "rope", "M": 4, "Bc": 4, "axes": 1, "out": "fp32", "heads": HEADS, "kv_heads": KV_HEADS,
         "hd": HEAD_DIM, "fused": False},
        # the drafts of a batch, queries in half precision
        {"name": "rope_tree_m333", "kind": "rope", "M": 333, "Bc": 9, "axes": 1, "out": "fp16", "heads": HEADS,
         "kv_heads": KV_HEADS, "hd": HEAD_DIM, "fused": False},
        # a prompt with images: positions on three axes
        {"name": "rope_image_m4999", "kind": "rope", "M": 4999, "Bc": 1, "axes": 3, "out": "fp32", "heads": HEADS,
         "kv_heads": KV_HEADS, "hd": HEAD_DIM, "fused": False},
        # one token of one sequence, the smallest attention there is
        {"name": "attn_token_1024", "kind": "attn", "B": 1, "T": 1, "ctx": 1024, "tree": False, "type": "fp32", "heads": HEADS,
         "kv_heads": KV_HEADS, "hd": HEAD_DIM},
        # one token of each sequence of a ragged batch: the caches' reads
        {"name": "attn_batch_b24", "kind": "attn", "B": 24, "T": 1, "ctx": 6000, "tree": False, "type": "fp32", "heads": HEADS,
         "kv_heads": KV_HEADS, "hd": HEAD_DIM},
        # trees of up to 61 drafts over long contexts
        {"name": "attn_tree_b3_16k", "kind": "attn", "B": 3, "T": 61, "ctx": 16000, "tree": True, "type": "fp32",
         "heads": HEADS, "kv_heads": KV_HEADS, "hd": HEAD_DIM},
        # a prompt's chunk behind what is cached already: products
        {"name": "attn_prompt_fp16", "kind": "attn", "B": 1, "T": 2000, "ctx": 1200, "tree": False, "type": "fp16",
         "heads": HEADS, "kv_heads": KV_HEADS, "hd": HEAD_DIM},
        # one generated token with its five best alternatives
        {"name": "logp_m1", "kind": "logp", "M": 1, "V": VOCAB, "k": 5, "type": "fp32", "pad": 0},
        # the rows of a draft tree, twenty alternatives each
        {"name": "logp_m61", "kind": "logp", "M": 61, "V": VOCAB, "k": 20, "type": "fp32", "pad": 0},
        # a prompt's tokens scored, no alternatives, logits in half precision
        {"name": "logp_prompt_m777", "kind": "logp", "M": 777, "V": VOCAB, "k": 0, "type": "fp16", "pad": 64},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "rope", "attn", "attn", "attn", "logp"])
    if kind == "plan":
        return {"kind": kind, "B": _log(rng, 1, 96), "T": _log(rng, 1, 500)}
    if kind == "logp":
        V = rng.choice([VOCAB, VOCAB, 32000, _log(rng, 1000, 150000)])
        return {"kind": kind, "M": _log(rng, 1, 500), "V": V, "k": rng.choice([0, 1, 5, 20, 64]),
                "type": rng.choice(["fp32", "fp32", "fp16"]), "pad": rng.choice([0, 1, 24])}
    heads, kv_heads, hd = rng.choice([(HEADS, KV_HEADS, HEAD_DIM), (HEADS, KV_HEADS, HEAD_DIM), (32, 8, 128), (12, 4, 64), (8, 8, 64),
                                      (28, 4, 128), (5, 1, 64)])
    if kind == "rope":
        M = _log(rng, 1, 4500)
        return {"kind": kind, "M": M, "Bc": rng.randint(1, min(M, 12)), "axes": rng.choice([1, 3]), "out": rng.choice(["fp32", "fp16"]),
                "heads": heads if heads <= 16 else HEADS, "kv_heads": kv_heads, "hd": hd, "fused": rng.random() < 0.5}
    c = {"kind": kind, "B": 1, "T": 1, "ctx": 0, "tree": False, "type": rng.choice(["fp32", "fp32", "fp16"]), "heads": heads,
         "kv_heads": kv_heads, "hd": hd}
    use = rng.choice(["token", "tree", "tree", "prompt"])
    if use == "token":
        c |= {"B": _log(rng, 1, 40), "ctx": _log(rng, 1, 12000)}
    elif use == "tree":
        c |= {"B": _log(rng, 1, 16), "T": _log(rng, 2, 100), "ctx": _log(rng, 1, 16000), "tree": True}
    else:
        c |= {"B": rng.randint(1, 3), "T": _log(rng, 64, 1400), "ctx": _log(rng, 1, 2000)}
    while c["B"] * c["ctx"] * kv_heads * hd > 24 * 6000 * KV_HEADS * HEAD_DIM:
        c["ctx"] //= 2
    while heads * hd * c["B"] * c["T"] * (c["ctx"] + c["T"] / 2) > HEADS * HEAD_DIM * 2000 * 2200:
        c["T"] = c["T"] * 3 // 4
    return c


# ------------------------------------------------------------------- inputs
def _lens(case):
    """Rows and cached positions of each sequence: the first has the case's
    own, the others fewer, now and then none."""
    B, T, ctx = case["B"], case["T"], case.get("ctx", 6000)
    r = random.Random(B * 1009 + T * 17 + ctx)
    rows = [T] + [0 if T > 1 and r.random() < 0.06 else r.randint(max(1, T // 4), T) for _ in range(B - 1)]
    return rows, [ctx] + [r.randint(ctx // 2, ctx) for _ in range(B - 1)]


def _ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device="cuda")


def _starts(rows):
    out = [0]
    for n in rows:
        out.append(out[-1] + n)
    return out


def _trees(g, rows):
    """A parent for each row: -1 (the last cached token) or an earlier row."""
    t = torch.cat([torch.arange(n, device="cuda") for n in rows])
    u = torch.rand(t.numel(), device="cuda", generator=g)
    return (t - 1 - (u * u * (t + 1)).long()).clamp_(min=-1).int()


def _tree_mask(parents, starts, rows, words):
    """Ancestor bits (the row itself among them) as 64-bit words, for the attention cases' inputs."""
    par, out, at = parents.tolist(), [], 0
    for n in rows:
        m = []
        for t in range(n):
            p = par[at + t]
            m.append((m[p] if p >= 0 else 0) | 1 << t)
        at += n
        for v in m:
            w = [v >> 64 * i & (1 << 64) - 1 for i in range(words)]
            out.append([x - (1 << 64) if x >> 63 else x for x in w])
    return _ints(out, torch.int64)


def _norm_weight(g, n):
    """int8 norm weights around one with a scale per group, as the exporter writes them."""
    w = torch.empty(n, device="cuda").uniform_(0.5, 1.5, generator=g).reshape(-1, GS)
    s = w.abs().amax(1) / 127
    return (w / s[:, None]).round().clamp(-127, 127).to(torch.int8).reshape(n), s


def _tables(rows, hd):
    inv = THETA ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)
    a = torch.arange(rows, dtype=torch.float64)[:, None] * inv
    return a.cos().float().cuda(), a.sin().float().cuda()


def _make(case, seed):
    """Everything a user's program has in hand, on the device."""
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    randn = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    st, kind = {"kind": case["kind"]}, case["kind"]
    if kind == "plan":
        rows, lens = _lens(case)
        st["row_start"], st["parents"] = _ints(_starts(rows)), _trees(g, rows)
        st["cache_len"] = _ints(lens) + torch.randint(0, 50, (case["B"],), device="cuda", generator=g, dtype=torch.int32)
        st["delta"] = torch.randint(-400, 1, (case["B"],), device="cuda", generator=g, dtype=torch.int32)
        st["max_seq"], st["max_rows"] = 6000 + 50 + case["T"], case["T"]
    elif kind == "rope":
        M, H, Hk, D = case["M"], case["heads"], case["kv_heads"], case["hd"]
        per = -(-M // case["Bc"])
        S, pads = per + 200, M // 16
        qkv = [3 * randn(M, n * D) for n in (H, Hk, Hk)]
        if case["fused"]:  # views of one projection's output
            qkv = list(torch.cat(qkv, 1).split([n.shape[1] for n in qkv], 1))
        st["q"], st["k"], st["v"] = qkv
        st["kc"], st["vc"] = randn(case["Bc"], Hk, S, D).half(), randn(case["Bc"], Hk, S, D).half()
        i = torch.arange(M, device="cuda")
        first = torch.randint(0, 200, (case["Bc"],), device="cuda", generator=g)
        slots, pos = i % case["Bc"] * S + first[i % case["Bc"]] + i // case["Bc"], first[i % case["Bc"]] + i // case["Bc"]
        if case["axes"] == 3:
            pos = pos[:, None] // 2 + torch.stack([i * 0, i // 28 % 28, i % 28], 1)
        slots[M - pads:], pos[M - pads:] = -1, -1  # rows that hold no token
        st["slots"], st["pos"], st["axes"] = slots.contiguous(), pos.int().contiguous(), case["axes"]
        st["qw"], st["qs"] = _norm_weight(g, D)
        st["kw"], st["ks"] = _norm_weight(g, D)
        st["cos"], st["sin"] = _tables(S + 64, D)
        st["out"] = randn(M, H * D).to(torch.float16 if case["out"] == "fp16" else torch.float32)
        st["sections"] = SECTIONS[D]
    elif kind == "attn":
        rows, lens = _lens(case)
        H, Hk, D, N = case["heads"], case["kv_heads"], case["hd"], sum(rows)
        S = (case["ctx"] + case["T"] + 7) // 8 * 8
        st["row_start"], st["cache_len"] = _ints(_starts(rows)), _ints(lens)
        st["q"] = (2 * randn(N, H * D)).to(torch.float16 if case["type"] == "fp16" else torch.float32)
        st["k"], st["v"] = (torch.empty((case["B"], Hk, S, D), dtype=torch.float16, device="cuda").normal_(generator=g) for _ in range(2))
        st["max_rows"], st["max_len"] = case["T"], case["ctx"] + case["T"]
        st["mask"] = _tree_mask(_trees(g, rows), _starts(rows), rows, -(-case["T"] // 64)) if case["tree"] else None
    else:
        M, V, dt = case["M"], case["V"], torch.float16 if case["type"] == "fp16" else torch.float32
        x = torch.empty((M, V + case["pad"]), dtype=dt, device="cuda").normal_(0, 3, generator=g)[:, :V]
        r = torch.arange(M, device="cuda")
        x[r, torch.randint(0, V, (M,), device="cuda", generator=g)] += (randn(M).abs() * 8).to(dt)  # peaked, as a model's rows are
        if M > 2:
            x[1, V // 7:] = -math.inf  # tokens ruled out
        st["x"], st["k"] = x, case["k"]
        st["tokens"] = torch.randint(0, V, (M,), device="cuda", generator=g, dtype=torch.int32)
        if M > 2:
            st["tokens"][1] = V // 9
    return st


# ------------------------------------------------------------------ the path
def prepare(case, seed):
    st = _make(case, seed)
    if own:
        qa, q = st["lib"] = _framework()
        kind = st["kind"]
        if kind == "rope":
            st["cache"] = qa.KVCache(st["kc"], st["vc"])
            st["norm"] = qa.QKNorm(st["qw"], st["qs"], st["kw"], st["ks"], GS, EPS)
            st["rope"] = qa.Rope(st["cos"], st["sin"], st["sections"] if st["axes"] == 3 else None, interleaved=True)
        elif kind == "attn":
            st["cache"] = qa.KVCache(st["k"], st["v"])
            st["ws"] = qa.alloc_tree_attention_workspace(st["cache"], st["q"].shape[0], case["heads"], st["max_rows"], st["max_len"])
        elif kind == "logp":
            st["ws"] = q.alloc_token_logprobs_workspace(case["M"], case["V"])
    return st


def _framework():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen3-vl-2b-inference_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import q3vl_int8
    from q3vl_int8 import attention
    return attention, q3vl_int8


def run(st):
    if own:
        return _run_own(st)
    return {"plan": _plain_plan, "rope": _plain_rope, "attn": _plain_attention, "logp": _plain_logprobs}[st["kind"]](st)


def _run_own(st):
    qa, q = st["lib"]
    kind = st["kind"]
    if kind == "plan":
        mask, pos, slots = qa.draft_plan(st["parents"], st["row_start"], st["cache_len"], st["max_seq"], st["max_rows"], pos_delta=st["delta"])
        return {"mask": mask, "pos": pos, "slots": slots}
    if kind == "rope":
        out = qa.qk_norm_rope(st["q"], st["k"], st["v"], st["cache"], st["slots"], st["pos"], st["norm"], st["rope"], out=st["out"])
        return {"q": out, "k": st["kc"], "v": st["vc"]}
    if kind == "attn":
        return qa.tree_attention(st["q"], st["cache"], st["row_start"], st["cache_len"], st["max_rows"], mask=st["mask"],
                                 max_len=st["max_len"], workspace=st["ws"])
    r = q.token_logprobs(st["x"], st["tokens"], top_k=st["k"], workspace=st["ws"])
    return {"logprob": r.logprob, "rank": r.rank, "entropy": r.entropy, "top_ids": r.top_ids, "top_logprobs": r.top_logprobs}


# ----------------------------------------------------------- the plain forms
def _local(row_start):
    """Each row's sequence and its place there."""
    n = (row_start[1:] - row_start[:-1]).long()
    seq = torch.repeat_interleave(torch.arange(n.numel(), device="cuda"), n)
    return seq, torch.arange(seq.numel(), device="cuda") - row_start.long()[seq]


def _plain_plan(st):
    T = st["max_rows"]
    words = -(-T // 64)
    seq, t = _local(st["row_start"])
    up = st["parents"].long()
    anc = t[:, None] == torch.arange(words * 64, device="cuda")  # [rows, bits]: the row itself
    at = torch.where(up < 0, torch.arange(t.numel(), device="cuda"), st["row_start"].long()[seq] + up)
    for _ in range(max(1, (T - 1).bit_length())):  # the ancestors of twice as many generations a turn
        anc, at = anc | anc[at], at[at]
    depth = anc.sum(1) - 1
    bits = torch.ones((), dtype=torch.int64, device="cuda") << torch.arange(64, device="cuda")
    mask = (anc.reshape(-1, words, 64) * bits).sum(2)
    pos = st["cache_len"].long()[seq] + st["delta"].long()[seq] + depth
    return {"mask": mask, "pos": pos.int(), "slots": seq * st["max_seq"] + st["cache_len"].long()[seq] + t}


def _axis(hd, sections):
    """The position axis of each frequency: the three axes in turn while they last, the rest time."""
    i = torch.arange(hd // 2, device="cuda")
    return torch.where((i % 3 == 1) & (i < 3 * sections[1]), 1, torch.where((i % 3 == 2) & (i < 3 * sections[2]), 2, 0))


def _plain_rope(st):
    D = st["kc"].shape[3]
    S, pos = st["kc"].shape[2], st["pos"].long().reshape(-1, st["axes"])
    held = pos[:, 0] >= 0
    axis = _axis(D, st["sections"]) if st["axes"] == 3 else torch.zeros(D // 2, dtype=torch.int64, device="cuda")
    at = pos.clamp(min=0)[:, axis]  # [M, D/2]
    f = torch.arange(D // 2, device="cuda")
    cos, sin = st["cos"][at, f][:, None], st["sin"][at, f][:, None]

    def turned(x, w, s):
        x = x.reshape(x.shape[0], -1, D)
        y = x / (x.square().mean(2, keepdim=True) + EPS).sqrt() * (w.float().reshape(-1, GS) * s[:, None]).reshape(-1)
        a, b = y[..., : D // 2], y[..., D // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], 2)

    qn = turned(st["q"], st["qw"], st["qs"]).reshape(st["out"].shape).to(st["out"].dtype)
    torch.where(held[:, None], qn, st["out"], out=st["out"])
    # a row without a slot writes again what is in the first row's place
    slot = torch.where(held, st["slots"], st["slots"][0])
    for c, x in ((st["kc"], turned(st["k"], st["kw"], st["ks"])), (st["vc"], st["v"].reshape(-1, st["kc"].shape[1], D))):
        c[slot // S, :, slot % S] = torch.where(held[:, None, None], x, x[:1]).half()
    return {"q": st["out"], "k": st["kc"], "v": st["vc"]}


def _plain_attention(st):
    k, v, S = st["k"].float(), st["v"].float(), st["k"].shape[2]
    B, Hk, _, D = k.shape
    T, N = st["max_rows"], st["q"].shape[0]
    t, j = torch.arange(T, device="cuda"), torch.arange(S, device="cuda")
    rows = (st["row_start"][1:] - st["row_start"][:-1]).long()
    at = (st["row_start"][:-1, None] + t).clamp(max=N - 1).long()  # [B, T], padded
    q = st["q"].float()[at].reshape(B, T, Hk, -1, D).transpose(1, 2).reshape(B, Hk, -1, D)
    d = j - st["cache_len"].long()[:, None]  # [B, S]: place among the drafts
    if st["mask"] is None:
        seen = d[:, None] <= t[:, None]
    else:
        m = st["mask"][at]
        word = (d // 64).clamp(0, m.shape[2] - 1)[:, None].expand(B, T, S)
        seen = (d < 0)[:, None] | (m.gather(2, word) >> (d % 64)[:, None] & 1).bool()
    seen = seen & (d < rows[:, None])[:, None]  # [B, T, S]
    s = torch.matmul(q, k.transpose(2, 3)).reshape(B, Hk, T, -1, S) / math.sqrt(D)
    s = s.masked_fill(~seen[:, None, :, None], -math.inf)
    top = s.amax(4, keepdim=True)
    p = torch.exp(s - top.masked_fill(top == -math.inf, 0))
    p = p / p.sum(4, keepdim=True).clamp(min=1e-30)
    o = torch.matmul(p.reshape(B, Hk, -1, S), v).reshape(B, Hk, T, -1, D).transpose(1, 2).reshape(B, T, -1)
    return o[t < rows[:, None]].to(st["q"].dtype)


def _plain_logprobs(st):
    x, V = st["x"].float(), st["x"].shape[1]
    top = x.amax(1, keepdim=True)
    d = x - top
    e = torch.exp(d)
    s = e.sum(1, dtype=torch.float64)
    logs = s.log()
    mean = torch.where(e > 0, e * d, 0).sum(1, dtype=torch.float64) / s
    at = torch.arange(V, device="cuda")
    xt = x.gather(1, st["tokens"].long()[:, None])
    ahead = (x > xt) | (x == xt) & (at < st["tokens"][:, None])
    out = {"logprob": ((xt - top)[:, 0].double() - logs).float(), "rank": ahead.sum(1).int(), "entropy": (logs - mean).float()}
    # values in order, equal ones by their place: the bits of a float, made to
    # order like whole numbers, over the place
    b = torch.where(x == 0, 0.0, x).view(torch.int32).long()
    key = torch.where(b < 0, b ^ 0x7FFFFFFF, b) << 32 | (V - 1 - at)
    ids = V - 1 - (key.topk(st["k"], 1).values & 0xFFFFFFFF)
    return out | {"top_ids": ids.int(), "top_logprobs": ((x.gather(1, ids) - top).double() - logs[:, None]).float()}


def work(case):
    kind = case["kind"]
    if kind == "plan":
        n, words = sum(_lens(case)[0]), -(-case["T"] // 64)
        return {"bytes": n * (4 + 8 * words + 4 + 8) + 12 * case["B"], "flops": n * words}
    if kind == "rope":
        M, D, H, Hk = case["M"] - case["M"] // 16, case["hd"], case["heads"], case["kv_heads"]
        io = 4 * D * (H + 2 * Hk) + D * H * (2 if case["out"] == "fp16" else 4) + 4 * D * Hk
        tables = 4 * D * min(M, -(-case["M"] // case["Bc"]) + 200)
        return {"bytes": M * (io + 4 * case["axes"] + 8) + tables, "flops": M * (H + Hk) * D * 7}
    if kind == "attn":
        rows, lens = _lens(case)
        D, H, Hk, e = case["hd"], case["heads"], case["kv_heads"], 2 if case["type"] == "fp16" else 4
        cached = sum(n + c for n, c in zip(rows, lens) if n)
        # a chain's row sees half the rows on average; so many of a tree's count as well
        pairs = sum(n * c + n * (n + 1) // 2 for n, c in zip(rows, lens))
        return {"bytes": 4 * D * Hk * cached + 2 * e * H * D * sum(rows), "flops": 4 * D * H * pairs}
    M, V = case["M"], case["V"]
    return {"bytes": M * V * (2 if case["type"] == "fp16" else 4) + M * (16 + 8 * case["k"]), "flops": 5 * M * V}


# ----------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    if case["kind"] == "plan":
        return None  # whole numbers
    st = _make(case, seed)
    return {"rope": _exact_rope, "attn": _exact_attention, "logp": _exact_logprobs}[st["kind"]](st)


def _exact_rope(st):
    Bc, Hk, S, D = st["kc"].shape
    half, axes = D // 2, st["axes"]
    pos = st["pos"].cpu().reshape(-1, axes)
    axis = [0] * half
    if axes == 3:
        for a in (1, 2):
            for n in range(st["sections"][a]):
                axis[3 * n + a] = a
    live = [i for i in range(pos.shape[0]) if int(pos[i, 0]) >= 0]
    row = torch.tensor(live, device="cuda")
    cs = torch.stack([st["cos"].double()[pos[live][:, a].long().cuda(), i] for i, a in enumerate(axis)], 1)
    sn = torch.stack([st["sin"].double()[pos[live][:, a].long().cuda(), i] for i, a in enumerate(axis)], 1)

    def head(x, w, s):
        x = x.double()[row].reshape(len(live), -1, D)
        z = torch.complex(x[..., :half], x[..., half:])
        g = w.double() * s.double().repeat_interleave(GS)
        z = torch.complex(z.real * g[:half], z.imag * g[half:])
        r = torch.linalg.vector_norm(x, dim=2, keepdim=True) / math.sqrt(D)
        z = z / torch.hypot(r, torch.tensor(math.sqrt(EPS), dtype=torch.float64, device="cuda"))
        z = z * torch.complex(cs, sn)[:, None]
        return torch.cat([z.real, z.imag], 2)

    q, k, v = st["out"].double(), st["kc"].double(), st["vc"].double()
    q[row] = head(st["q"], st["qw"], st["qs"]).reshape(len(live), -1)
    b, at = st["slots"][row] // S, st["slots"][row] % S
    k[b, :, at] = head(st["k"], st["kw"], st["ks"])
    v[b, :, at] = st["v"].double()[row].reshape(len(live), Hk, D)
    return {"q": q, "k": k, "v": v}


def _exact_attention(st):
    H, D = st["q"].shape[1] // st["k"].shape[3], st["k"].shape[3]
    Hk, out = st["k"].shape[1], []
    start, lens = st["row_start"].tolist(), st["cache_len"].tolist()
    for b, c in enumerate(lens):
        n = start[b + 1] - start[b]
        if n == 0:
            continue
        q = st["q"][start[b]:start[b + 1]].double().reshape(n, H, D)
        if st["mask"] is None:
            tail = torch.ones((n, n), dtype=torch.bool, device="cuda").tril()
        else:
            w = st["mask"][start[b]:start[b + 1]]
            tail = torch.stack([(w[:, i // 64] >> i % 64) & 1 for i in range(n)], 1) == 1
        seen = torch.cat([torch.ones((n, c), dtype=torch.bool, device="cuda"), tail], 1)
        o = torch.empty((n, H, D), dtype=torch.float64, device="cuda")
        for h in range(H):
            k, v = (st[x][b, h // (H // Hk), : c + n].double() for x in ("k", "v"))
            s = (q[:, h] @ k.t().contiguous()) / math.sqrt(D)
            o[:, h] = torch.softmax(s.masked_fill(~seen, -math.inf), 1) @ v
        out.append(o.reshape(n, H * D))
    return torch.cat(out)


def _exact_logprobs(st):
    out = {"logprob": [], "rank": None, "entropy": [], "top_ids": None, "top_logprobs": []}
    for x, t in zip(st["x"], st["tokens"].tolist()):
        lp = torch.log_softmax(x.double(), 0)
        out["logprob"].append(lp[t])
        out["entropy"].append(-torch.special.xlogy(lp.exp(), lp.exp()).sum())
        out["top_logprobs"].append(lp.sort(descending=True).values[: st["k"]])
    return {n: torch.stack(v) if v is not None else None for n, v in out.items()}
