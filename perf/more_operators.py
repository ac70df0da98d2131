"""Timed cases of the operators for long contexts and for checking drafts: a
cache whose whole blocks of 32 positions are held in 8 bits (written, read back,
attended to), attention through a window with a few first positions that stay
visible, and drafted tokens judged against the target's probabilities.

Each operator has its plain form here (elementary torch operations in 32 bits,
64 where a comparison or a long sum asks for it), the framework's call, and its
definition in 64 bits. The head layout 16 / 8 of 128 and the vocabulary 151936
are the text decoder's that perf/cases.py times; `draw` takes others too.

Kinds:
  store   whole blocks of the newest rows go to 8 bits, the rest moves to the
          front; what was stored is read back
  load    a cache's 8-bit blocks back to fp16
  attn    the rows of a batch (a token each, trees of drafts, a prompt's chunk)
          over 8-bit blocks and the fp16 rows behind them, or over fp16 rows
          alone; everything before a row, or a window and the first positions
  verify  rejection sampling along chains or trees of drafts

A block holds 32 positions of one kv head in the order in which the matrix
instructions take them: see `_to_blocks`.
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

HEADS, KV_HEADS, HEAD_DIM, VOCAB, BLOCK = 16, 8, 128, 151936, 32
MODEL = {"heads": HEADS, "kv_heads": KV_HEADS, "hd": HEAD_DIM}


def listed():
    return [
        # a serving batch's step: one sequence in two has filled a block
        {"name": "store_step_b24", "kind": "store", "B": 24, "rows": 63, "kv_heads": KV_HEADS, "hd": HEAD_DIM},
        # a prompt that has just been read
        {"name": "store_prompt_4099", "kind": "store", "B": 1, "rows": 4099, "kv_heads": KV_HEADS, "hd": HEAD_DIM},
        # a short sequence handed to the one-token decode step
        {"name": "load_1000", "kind": "load", "B": 1, "ctx": 1000, "kv_heads": KV_HEADS, "hd": HEAD_DIM},
        # four long ones
        {"name": "load_b4_16k", "kind": "load", "B": 4, "ctx": 16000, "kv_heads": KV_HEADS, "hd": HEAD_DIM},
        # one token of one sequence: latency alone
        {"name": "packed_token_1024", "kind": "attn", "B": 1, "T": 1, "ctx": 1024, "packed": True, "window": 0, "sinks": 0, "tree": False,
         "type": "fp32", **MODEL},
        # one token of each sequence of a ragged batch: the cache's reads
        {"name": "packed_batch_b24_12k", "kind": "attn", "B": 24, "T": 1, "ctx": 12000, "packed": True, "window": 0, "sinks": 0, "tree": False,
         "type": "fp32", **MODEL},
        # trees of up to 61 drafts over long contexts
        {"name": "packed_tree_b3_16k", "kind": "attn", "B": 3, "T": 61, "ctx": 16000, "packed": True, "window": 0, "sinks": 0, "tree": True,
         "type": "fp32", **MODEL},
        # a prompt's chunk behind what is packed already: products
        {"name": "packed_prompt_fp16", "kind": "attn", "B": 1, "T": 1000, "ctx": 8000, "packed": True, "window": 0, "sinks": 0, "tree": False,
         "type": "fp16", **MODEL},
        # a batch far into its streams, each token looking back 4096 positions
        {"name": "window_batch_b16_30k", "kind": "attn", "B": 16, "T": 1, "ctx": 30000, "packed": False, "window": 4096, "sinks": 4,
         "tree": False, "type": "fp32", **MODEL},
        # a long prompt read through a window
        {"name": "window_prompt_fp16", "kind": "attn", "B": 1, "T": 4000, "ctx": 0, "packed": False, "window": 1024, "sinks": 4, "tree": False,
         "type": "fp16", **MODEL},
        # seven drafted tokens a sequence, drawn from a draft model
        {"name": "verify_chain_b16", "kind": "verify", "B": 16, "T": 8, "V": VOCAB, "probs": True, "tree": False, "type": "fp32", "pad": 0},
        # trees of drafts whose source is certain of each
        {"name": "verify_tree_b3", "kind": "verify", "B": 3, "T": 61, "V": VOCAB, "probs": False, "tree": True, "type": "fp32", "pad": 0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["store", "load", "attn", "attn", "attn", "attn", "verify", "verify"])
    heads, kv_heads, hd = rng.choice([(HEADS, KV_HEADS, HEAD_DIM), (HEADS, KV_HEADS, HEAD_DIM), (32, 8, 128), (12, 4, 64), (8, 8, 64),
                                      (28, 4, 128), (5, 1, 64)])
    if kind == "store":
        B = _log(rng, 1, 48)
        return {"kind": kind, "B": B, "rows": _log(rng, 33, max(80, 8000 // B)), "kv_heads": kv_heads, "hd": hd}
    if kind == "load":
        B = _log(rng, 1, 16)
        return {"kind": kind, "B": B, "ctx": _log(rng, 32, 64000 // B), "kv_heads": kv_heads, "hd": hd}
    if kind == "verify":
        tree = rng.random() < 0.5
        V = rng.choice([VOCAB, VOCAB, 32000, _log(rng, 1000, 150000)])
        c = {"kind": kind, "B": _log(rng, 1, 24), "T": _log(rng, 2, 61) if tree else rng.randint(2, 9), "V": V, "probs": rng.random() < 0.5,
             "tree": tree, "type": rng.choice(["fp32", "fp32", "fp16"]), "pad": rng.choice([0, 1, 24])}
        while c["B"] * c["T"] > 128:
            c["B"] = c["B"] * 3 // 4
        return c
    c = {"kind": kind, "B": 1, "T": 1, "ctx": 0, "packed": rng.random() < 0.6, "window": 0, "sinks": 0, "tree": False,
         "type": rng.choice(["fp32", "fp32", "fp16"]), "heads": heads, "kv_heads": kv_heads, "hd": hd}
    use = rng.choice(["token", "tree", "tree", "prompt"])
    if use == "token":
        c |= {"B": _log(rng, 1, 40), "ctx": _log(rng, 1, 20000)}
    elif use == "tree":
        c |= {"B": _log(rng, 1, 16), "T": _log(rng, 2, 100), "ctx": _log(rng, 1, 20000), "tree": True}
    else:
        c |= {"B": rng.randint(1, 3), "T": _log(rng, 64, 2500), "ctx": _log(rng, 1, 8000)}
    if not c["packed"] or rng.random() < 0.4:  # over fp16 rows alone there is an operator without a window
        c |= {"window": _log(rng, max(100, c["T"]) if c["tree"] else 16, 6000), "sinks": rng.choice([0, 1, 4, 64])}
    while c["B"] * c["ctx"] * kv_heads * hd > 24 * 12000 * KV_HEADS * HEAD_DIM:
        c["ctx"] //= 2
    while heads * hd * c["B"] * c["T"] * (c["ctx"] + c["T"] / 2) > HEADS * HEAD_DIM * 8e6:
        c["T"] = c["T"] * 3 // 4
    return c


# ------------------------------------------------------------------- inputs
def _lens(case):
    """Of each sequence: its rows, packed positions (whole blocks) and fp16 rows
    before its own. The first has the case's own length, the others less."""
    B, T, ctx = case["B"], case.get("T", 1), case["ctx"]
    r = random.Random(B * 1009 + T * 17 + ctx)
    rows = [T] + [0 if T > 1 and r.random() < 0.06 else r.randint(max(1, T // 4), T) for _ in range(B - 1)]
    lens = [ctx] + [r.randint(ctx // 2, ctx) for _ in range(B - 1)]
    if not case.get("packed", True):
        return rows, [0] * B, lens
    held = [max(0, n - r.randint(0, BLOCK)) // BLOCK * BLOCK for n in lens]
    return rows, held, [n - h for n, h in zip(lens, held)]


def _newest(case):
    """A store's lengths: packed positions before it, fp16 rows."""
    r = random.Random(case["B"] * 31 + case["rows"])
    rows = [case["rows"]] + [r.randint(case["rows"] // 4, case["rows"]) for _ in range(case["B"] - 1)]
    return [BLOCK * r.randint(0, 20) for _ in rows], rows


def _ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device="cuda")


def _starts(rows):
    out = [0]
    for n in rows:
        out.append(out[-1] + n)
    return out


def _trees(g, rows, wide):
    """A parent for each row: -1 or an earlier row. `wide`: every other row below the first."""
    t = torch.cat([torch.arange(n, device="cuda") for n in rows])
    u = torch.rand(t.numel(), device="cuda", generator=g)
    p = t - 1 - (u * u * (t + 1)).long()
    return torch.where(t == 0, -1, p.clamp(min=0)).int() if wide else p.clamp_(min=-1).int()


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


def _to_blocks(k, v):
    """Blocks [..., 32, D] in their order in memory [..., 32 * D]. A lane takes 16
    bytes at once. Keys: position 16 a + i and values 64 c + 32 s + 8 g + e lie at
    [a][c][g][i][s][e]; values: position 16 a + 4 g + e and value 32 c + 16 s + i at
    [c][g][i][s][a][e]."""
    D, lead = k.shape[-1], k.shape[:-2]
    n = len(lead)
    k = k.reshape(*lead, 2, 16, D // 64, 2, 4, 8).permute(*range(n), n, n + 2, n + 4, n + 1, n + 3, n + 5)
    v = v.reshape(*lead, 2, 4, 4, D // 32, 2, 16).permute(*range(n), n + 3, n + 1, n + 5, n + 4, n, n + 2)
    return k.reshape(*lead, BLOCK * D), v.reshape(*lead, BLOCK * D)


def _from_blocks(k, v):
    """The reverse of _to_blocks."""
    D, lead = k.shape[-1] // BLOCK, k.shape[:-1]
    n = len(lead)
    k = k.reshape(*lead, 2, D // 64, 4, 16, 2, 8).permute(*range(n), n, n + 3, n + 1, n + 4, n + 2, n + 5)
    v = v.reshape(*lead, D // 32, 4, 16, 2, 2, 4).permute(*range(n), n + 4, n + 1, n + 5, n, n + 3, n + 2)
    return k.reshape(*lead, BLOCK, D), v.reshape(*lead, BLOCK, D)


def _quantised(x):
    """Blocks [..., 32, D] as whole numbers of at most 127 and a scale each."""
    s = x.abs().amax((-1, -2)) / 127
    return (x / torch.where(s > 0, s, 1)[..., None, None]).round().to(torch.int8), s


def _held(g, B, Hk, blocks, D, outliers):
    """A cache's 8-bit blocks: keys with a few strong channels, as rotated keys have."""
    k = torch.empty((B, Hk, blocks, BLOCK, D), device="cuda").normal_(generator=g)
    if outliers:
        k[..., :: D // 4] *= 3
    (k, ks), (v, vs) = _quantised(k), _quantised(torch.empty_like(k).normal_(generator=g))
    k, v = _to_blocks(k, v)
    return k, v, ks, vs


def _make(case, seed):
    """Everything a user's program has in hand, on the device."""
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    randn = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    half = lambda *s: torch.empty(s, dtype=torch.float16, device="cuda").normal_(generator=g)  # noqa: E731
    kind = case["kind"]
    st = {"kind": kind}
    if kind == "store":
        B, Hk, D, n = case["B"], case["kv_heads"], case["hd"], case["rows"]
        before, rows = _newest(case)
        st["k"], st["v"] = half(B, Hk, n + 8, D), half(B, Hk, n + 8, D)
        blocks = max(before) // BLOCK + n // BLOCK
        st["k8"], st["v8"], st["ks"], st["vs"] = _held(g, B, Hk, blocks, D, False)
        st["k_back"], st["v_back"] = half(B, Hk, max(n, 32), D), half(B, Hk, max(n, 32), D)
        st["cache_len"], st["packed_len"] = _ints(rows), _ints(before)
        st["end"], st["count"] = _ints([b + n // BLOCK * BLOCK for b, n in zip(before, rows)]), n // BLOCK * BLOCK
    elif kind == "load":
        B, Hk, D = case["B"], case["kv_heads"], case["hd"]
        blocks = -(-case["ctx"] // BLOCK)
        st["k8"], st["v8"], st["ks"], st["vs"] = _held(g, B, Hk, blocks, D, True)
        st["packed_len"] = _ints([-(-n // BLOCK) * BLOCK for n in map(sum, zip(*_lens(case)[1:]))])
        st["k"], st["v"] = half(B, Hk, blocks * BLOCK, D), half(B, Hk, blocks * BLOCK, D)
    elif kind == "attn":
        rows, held, lens = _lens(case)
        H, Hk, D, N = case["heads"], case["kv_heads"], case["hd"], sum(rows)
        S = (max(n + c for n, c in zip(rows, lens)) + 7) // 8 * 8
        st["row_start"], st["cache_len"] = _ints(_starts(rows)), _ints(lens)
        st["q"] = (2 * randn(N, H * D)).to(torch.float16 if case["type"] == "fp16" else torch.float32)
        st["k"], st["v"] = half(case["B"], Hk, S, D), half(case["B"], Hk, S, D)
        st["packed_len"] = _ints(held) if case["packed"] else None
        if case["packed"]:
            st["k8"], st["v8"], st["ks"], st["vs"] = _held(g, case["B"], Hk, max(1, max(held) // BLOCK), D, True)
        st["max_rows"], st["max_len"] = case["T"], case["ctx"] + case["T"]
        st["window"], st["sinks"] = case["window"], case["sinks"]
        st["mask"] = _tree_mask(_trees(g, rows, False), _starts(rows), rows, -(-case["T"] // 64)) if case["tree"] else None
    else:
        B, T, V = case["B"], case["T"], case["V"]
        r = random.Random(B * 1009 + T * 17 + V)
        rows = [T] + [r.randint(max(1, T // 4), T) for _ in range(B - 1)]
        N = sum(rows)
        x = torch.empty((N, V + case["pad"]), device="cuda").normal_(0, 3, generator=g)[:, :V]
        x[torch.arange(N, device="cuda"), torch.randint(0, V, (N,), device="cuda", generator=g)] += randn(N).abs() * 8  # peaked, as a model's rows are
        t = torch.cat([torch.arange(n, device="cuda") for n in rows])
        st["row_start"], st["max_rows"] = _ints(_starts(rows)), T
        st["parents"] = _trees(g, rows, True) if case["tree"] else (t - 1).int()
        seq = torch.repeat_interleave(torch.arange(B, device="cuda"), _ints(rows).long())
        up = st["row_start"].long()[seq] + st["parents"].long().clamp(min=0)
        q = torch.softmax(x + 0.7 * torch.empty((N, V), device="cuda").normal_(generator=g), 1)  # the draft's view of the same
        u = torch.rand(N, device="cuda", generator=g, dtype=torch.float64)
        st["tokens"] = torch.searchsorted(q.double().cumsum(1)[up], u[:, None])[:, 0].clamp(max=V - 1).int()
        if case["type"] == "fp16":
            wide = torch.empty((N, V + case["pad"]), dtype=torch.float16, device="cuda")
            wide[:, :V] = x
            x = wide[:, :V]
        st["x"], st["q"] = x, q if case["probs"] else None
        st["accept_u"], st["sample_u"] = (torch.rand(N, device="cuda", generator=g) for _ in range(2))
        st["temperature"] = 0.8
    return st


# ------------------------------------------------------------------ the path
def prepare(case, seed):
    st = _make(case, seed)
    if own:
        qa = st["lib"] = _framework()
        kind = st["kind"]
        if "k8" in st:
            st["packed"] = qa.PackedKV(st["k8"], st["v8"], st["ks"], st["vs"])
        if "k" in st:
            st["cache"] = qa.KVCache(st["k"], st["v"])
        if kind == "store":
            st["back"] = qa.KVCache(st["k_back"], st["v_back"])
        elif kind == "attn":
            st["ws"] = qa.alloc_long_attention_workspace(st["cache"], st["q"].shape[0], case["heads"], st["max_rows"], st["max_len"],
                                                         packed=st.get("packed"), window=st["window"], sinks=st["sinks"])
        elif kind == "verify":
            st["ws"] = qa.alloc_verify_drafts_workspace(*st["x"].shape)
    return st


def _framework():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen3-vl-2b-inference_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    from q3vl_int8 import attention
    return attention


def run(st):
    if own:
        return _run_own(st)
    return {"store": _plain_store, "load": _plain_load, "attn": _plain_attention, "verify": _plain_verify}[st["kind"]](st)


def _run_own(st):
    qa, kind = st["lib"], st["kind"]
    if kind == "store":
        qa.kv_pack(st["cache"], st["packed"], st["cache_len"], st["packed_len"])
        qa.kv_unpack(st["packed"], st["end"], st["back"], first=st["packed_len"], count=st["count"])
        return {n: st[n] for n in ("k", "v", "ks", "vs", "k_back", "v_back")}
    if kind == "load":
        qa.kv_unpack(st["packed"], st["packed_len"], st["cache"])
        return {"k": st["k"], "v": st["v"]}
    if kind == "attn":
        return qa.long_attention(st["q"], st["cache"], st["row_start"], st["cache_len"], st["max_rows"], packed=st.get("packed"),
                                 packed_len=st["packed_len"], window=st["window"], sinks=st["sinks"], mask=st["mask"],
                                 max_len=st["max_len"], workspace=st["ws"])
    r = qa.verify_drafts(st["x"], st["tokens"], st["parents"], st["row_start"], st["accept_u"], st["sample_u"], st["max_rows"],
                         draft_probs=st["q"], temperature=st["temperature"], workspace=st["ws"])
    return {"accepted": r.accepted, "path": r.path, "next": r.next}


# ----------------------------------------------------------- the plain forms
def _plain_store(st):
    B, Hk, S, D = st["k"].shape
    most = st["count"] // BLOCK
    n = st["cache_len"].long() // BLOCK
    j = torch.arange(most, device="cuda")
    b, j = torch.nonzero(j < n[:, None], as_tuple=True)  # the whole blocks
    at = st["packed_len"].long()[b] // BLOCK + j
    k, v = (st[x][:, :, : most * BLOCK].reshape(B, Hk, most, BLOCK, D)[b, :, j].float() for x in ("k", "v"))
    (k, ks), (v, vs) = _quantised(k), _quantised(v)
    st["k8"][b, :, at], st["v8"][b, :, at] = _to_blocks(k, v)
    st["ks"][b, :, at], st["vs"][b, :, at] = ks, vs
    rows = torch.arange(S, device="cuda")
    first = BLOCK * n[:, None]
    move = torch.where((rows < st["cache_len"][:, None] - first) & (first > 0), rows + first, rows)[:, None, :, None].expand(B, Hk, S, D)
    for x, w, s in (("k", k, ks), ("v", v, vs)):
        st[x].copy_(st[x].gather(2, move))
        back = st[x + "_back"][:, :, : most * BLOCK].reshape(B, Hk, most, BLOCK, D).clone()
        back[b, :, j] = (w.float() * s[..., None, None]).half()
        st[x + "_back"][:, :, : most * BLOCK] = back.reshape(B, Hk, -1, D)
    return {x: st[x] for x in ("k", "v", "ks", "vs", "k_back", "v_back")}


def _values(st):
    """The packed positions' keys and values [B, Hk, positions, D]."""
    k, v = _from_blocks(st["k8"], st["v8"])
    B, Hk, n, _, D = k.shape
    return [(x.float() * s[..., None, None]).reshape(B, Hk, n * BLOCK, D) for x, s in ((k, st["ks"]), (v, st["vs"]))]


def _plain_load(st):
    there = torch.arange(st["k"].shape[2], device="cuda") < st["packed_len"][:, None]
    for x, w in zip(("k", "v"), _values(st)):
        st[x].copy_(torch.where(there[:, None, :, None], w.half(), st[x]))
    return {"k": st["k"], "v": st["v"]}


def _plain_attention(st):
    k, v, S = st["k"].float(), st["v"].float(), st["k"].shape[2]
    B, Hk, _, D = k.shape
    T, N = st["max_rows"], st["q"].shape[0]
    t, j = torch.arange(T, device="cuda"), torch.arange(S, device="cuda")
    rows = (st["row_start"][1:] - st["row_start"][:-1]).long()
    at = (st["row_start"][:-1, None] + t).clamp(max=N - 1).long()  # [B, T], padded
    q = st["q"].float()[at].reshape(B, T, Hk, -1, D).transpose(1, 2).reshape(B, Hk, -1, D)
    d = j - st["cache_len"].long()[:, None]  # [B, S]: place among the step's rows
    if st["mask"] is None:
        seen = d[:, None] <= t[:, None]
    else:
        m = st["mask"][at]
        word = (d // 64).clamp(0, m.shape[2] - 1)[:, None].expand(B, T, S)
        seen = (d < 0)[:, None] | (m.gather(2, word) >> (d % 64)[:, None] & 1).bool()
    seen = seen & (d < rows[:, None])[:, None]  # [B, T, S]
    if st["packed_len"] is not None:
        pk, pv = _values(st)
        k, v = torch.cat([pk, k], 2), torch.cat([pv, v], 2)
        held = torch.arange(pk.shape[2], device="cuda") < st["packed_len"][:, None]
        seen = torch.cat([held[:, None].expand(B, T, -1), seen], 2)
    if st["window"]:
        place = seen.cumsum(2)  # of what the row sees, from 1
        seen = seen & ((place <= st["sinks"]) | (place > place[..., -1:] - st["window"]))
    s = torch.matmul(q, k.transpose(2, 3)).reshape(B, Hk, T, -1, k.shape[2]) / math.sqrt(D)
    s = s.masked_fill(~seen[:, None, :, None], -math.inf)
    top = s.amax(4, keepdim=True)
    p = torch.exp(s - top.masked_fill(top == -math.inf, 0))
    p = p / p.sum(4, keepdim=True).clamp(min=1e-30)
    o = torch.matmul(p.reshape(B, Hk, -1, k.shape[2]), v).reshape(B, Hk, T, -1, D).transpose(1, 2).reshape(B, T, -1)
    return o[t < rows[:, None]].to(st["q"].dtype)


def _plain_verify(st):
    N, V = st["x"].shape
    T, start, par = st["max_rows"], st["row_start"].long(), st["parents"].long()
    seq = torch.repeat_interleave(torch.arange(start.numel() - 1, device="cuda"), start[1:] - start[:-1])
    row = torch.arange(N, device="cuda")
    x = st["x"].double()
    e = torch.exp((x - x.amax(1, keepdim=True)) / st["temperature"])
    total = e.sum(1, keepdim=True)
    tok = st["tokens"].long()
    kid = (par >= 0)[:, None] & (start[seq] + par)[:, None].eq(row)  # [row, parent]
    none = torch.full((N,), N, device="cuda")
    if st["q"] is None:
        pick = _first_over(e, st["sample_u"])
        taken = torch.where(kid & (tok[:, None] == pick), row[:, None], N).amin(0)
    else:
        q, taken = st["q"].double(), none
        order = kid.cumsum(0)  # a child's place among its parent's, from 1
        c, w = torch.zeros_like(total), e
        for n in range(int(order.amax()) if T > 1 else 0):
            child = torch.where(kid & (order == n + 1), row[:, None], N).amin(0)  # of each row, N: none
            to_try = (child < N) & (taken == N)
            at = child.clamp(max=N - 1)
            t = tok[at][:, None]
            z = w.sum(1, keepdim=True) / total
            yes = st["accept_u"].double()[at][:, None] * q.gather(1, t) * z < w.gather(1, t) / total
            taken = torch.where(to_try & yes[:, 0], child, taken)
            c = torch.where((to_try & ~yes[:, 0])[:, None], c + z, c)
            w = (e - c * total * q).clamp(min=0)
        w = torch.where(w.sum(1, keepdim=True) > 0, w, e)
        pick = _first_over(w, st["sample_u"])
    at, count = start[:-1].clone(), torch.ones_like(start[:-1])
    path = torch.full((start.numel() - 1, T), -1, device="cuda")
    path[:, 0] = 0
    for n in range(1, T):
        go = taken[at]
        on = go < N
        at = torch.where(on, go, at)
        path[:, n] = torch.where(on, at - start[:-1], -1)
        count = count + on
    return {"accepted": count.int(), "path": path.int(), "next": pick[at].int()}


def _first_over(w, u):
    """The first index whose cumulated weight passes u times the sum."""
    s = w.cumsum(1)
    over = (s > u.double()[:, None] * s[:, -1:]) & (w > 0)
    at = torch.arange(w.shape[1], device="cuda")
    return torch.where(over.any(1), over.int().argmax(1), torch.where(w > 0, at, -1).amax(1))


def work(case):
    kind = case["kind"]
    D = case.get("hd")
    if kind == "store":
        blocks, Hk = sum(n // BLOCK for n in _newest(case)[1]), case["kv_heads"]
        rest = sum(n % BLOCK for n in _newest(case)[1])
        # rows to 8 bits, those back to rows, what is left moved
        return {"bytes": Hk * (blocks * 2 * (BLOCK * D * (2 + 1 + 1 + 2) + 8) + rest * 8 * D), "flops": Hk * blocks * BLOCK * D * 8}
    if kind == "load":
        n = sum(-(-c // BLOCK) for c in map(sum, zip(*_lens(case)[1:])))
        return {"bytes": n * case["kv_heads"] * 2 * (BLOCK * D * 3 + 4), "flops": n * case["kv_heads"] * 2 * BLOCK * D}
    if kind == "attn":
        rows, held, lens = _lens(case)
        H, Hk, e, W = case["heads"], case["kv_heads"], 2 if case["type"] == "fp16" else 4, case["window"]
        pairs = read = 0
        for n, h, c in zip(rows, held, lens):
            if not n:
                continue
            all_, first = h + c + n, 0  # positions read: the first and those that some row's window holds
            if W:
                first = max(min(case["sinks"], h + c + 1), h + c + 1 - W)
                first = max(0, first - min(case["sinks"], h + c + 1))
            h8 = h - min(first, h)
            read += Hk * (h8 * (2 * D + 0.25) + (all_ - first - h8) * 4 * D)
            # a chain's row sees half the rows on average; so many of a tree's count as well
            pairs += sum(min(h + c + i + 1, W + case["sinks"]) if W else h + c + i + 1 for i in range(n))
        return {"bytes": read + 2 * e * H * D * sum(rows), "flops": 4 * D * H * pairs}
    r = random.Random(case["B"] * 1009 + case["T"] * 17 + case["V"])
    N = case["T"] + sum(r.randint(max(1, case["T"] // 4), case["T"]) for _ in range(case["B"] - 1))
    return {"bytes": N * case["V"] * ((2 if case["type"] == "fp16" else 4) + 4 * case["probs"]) + 20 * N, "flops": 6 * N * case["V"]}


# ----------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    if case["kind"] == "verify":
        return None  # whole numbers
    st = _make(case, seed)
    return {"store": _exact_store, "load": _exact_load, "attn": _exact_attention}[st["kind"]](st)


def _exact_blocks(st, b):
    """One sequence's packed keys and values in 64 bits, position by position."""
    Hk, n, D = st["k8"].shape[1], st["k8"].shape[2], st["k8"].shape[3] // BLOCK
    p, d = torch.arange(BLOCK, device="cuda")[:, None], torch.arange(D, device="cuda")
    ka = (((p // 16 * (D // 64) + d // 64) * 4 + d % 32 // 8) * 16 + p % 16) * 16 + d % 64 // 32 * 8 + d % 8
    va = ((d // 32 * 4 + p % 16 // 4) * 16 + d % 16) * 16 + d % 32 // 16 * 8 + p // 16 * 4 + p % 4
    return [(st[x + "8"][b][:, :, a].double() * st[x + "s"][b].double()[..., None, None]).reshape(Hk, n * BLOCK, D)
            for x, a in (("k", ka), ("v", va))]


def _exact_store(st):
    out = {n: st[n].double() for n in ("k", "v", "ks", "vs", "k_back", "v_back")}
    for b, (n, at) in enumerate(zip(st["cache_len"].tolist(), st["packed_len"].tolist())):
        whole = n // BLOCK * BLOCK
        for x in "kv":
            rows = st[x][b].double()
            for i in range(0, whole, BLOCK):
                y = rows[:, i:i + BLOCK]
                s = y.abs().flatten(1).max(1).values / 127
                out[x + "s"][b, :, (at + i) // BLOCK] = s
                out[x + "_back"][b, :, i:i + BLOCK] = torch.round(y / s[:, None, None]) * s[:, None, None]
            if whole:
                out[x][b, :, : n - whole] = rows[:, whole:n]
    return out


def _exact_load(st):
    out = {"k": st["k"].double(), "v": st["v"].double()}
    for b, n in enumerate(st["packed_len"].tolist()):
        for x, w in zip("kv", _exact_blocks(st, b)):
            out[x][b, :, :n] = w[:, :n]
    return out


def _exact_attention(st):
    H, D = st["q"].shape[1] // st["k"].shape[3], st["k"].shape[3]
    Hk, out = st["k"].shape[1], []
    start, lens = st["row_start"].tolist(), st["cache_len"].tolist()
    packed = st["packed_len"].tolist() if st["packed_len"] is not None else [0] * len(lens)
    for b, (c, h) in enumerate(zip(lens, packed)):
        n = start[b + 1] - start[b]
        if n == 0:
            continue
        q = st["q"][start[b]:start[b + 1]].double().reshape(n, H, D)
        if st["mask"] is None:
            tail = torch.ones((n, n), dtype=torch.bool, device="cuda").tril()
        else:
            w = st["mask"][start[b]:start[b + 1]]
            tail = torch.stack([(w[:, i // 64] >> i % 64) & 1 for i in range(n)], 1) == 1
        seen = torch.cat([torch.ones((n, h + c), dtype=torch.bool, device="cuda"), tail], 1)
        if st["window"]:
            ahead, behind = seen.cumsum(1) - 1, seen.flip(1).cumsum(1).flip(1) - 1
            seen = seen & ((ahead < st["sinks"]) | (behind < st["window"]))
        kv = [st[x][b, :, : c + n].double() for x in "kv"]
        if h:
            kv = [torch.cat([x[:, :h], y], 1) for x, y in zip(_exact_blocks(st, b), kv)]
        o = torch.empty((n, H, D), dtype=torch.float64, device="cuda")
        for i in range(H):
            k, v = (x[i // (H // Hk)] for x in kv)
            s = (q[:, i] @ k.t().contiguous()) / math.sqrt(D)
            o[:, i] = torch.softmax(s.masked_fill(~seen, -math.inf), 1) @ v
        out.append(o.reshape(n, H * D))
    return torch.cat(out)
