"""Refusals and sizes of the operators for long contexts and judged drafts
(q3vl_kv_pack, q3vl_kv_advance, q3vl_kv_unpack, q3vl_long_attention,
q3vl_verify_drafts): every bad argument is turned away before any device work,
so this needs no GPU. Pointers are fake, aligned and never read."""
import ctypes
import math

import numpy as np
import pytest

import long_ref as ref
import q3vl_int8 as q
from q3vl_int8 import attention as qa
from test_rows_capi import cache, refused

P = 1 << 20
BAD, UNS = q.ERR_INVALID_ARGUMENT, q.ERR_UNSUPPORTED


def blocks(**over):
    f = dict(k=P, v=P, k_scale=P, v_scale=P, batch=2, kv_heads=2, blocks=8, head_dim=128)
    f.update(over)
    return qa._BlocksC(*f.values())


def pack(cache_over={}, blocks_over={}, fn="q3vl_kv_pack", **over):
    f = dict(cache=ctypes.byref(cache(**cache_over)), blocks=ctypes.byref(blocks(**blocks_over)), cache_len=P, packed_len=2 * P, stream=None)
    f.update(over)
    return getattr(qa._L(), fn)(*f.values())


SHARED = [
    (dict(cache=None), BAD, "null cache"),
    (dict(blocks=None), BAD, "null blocks"),
    (dict(cache_over=dict(head_dim=96, row_stride=96)), UNS, "head_dim=96"),
    (dict(cache_over=dict(k=P + 8)), BAD, "aligned"),
    (dict(blocks_over=dict(v=None)), BAD, "null blocks"),
    (dict(blocks_over=dict(k_scale=None)), BAD, "null blocks"),
    (dict(blocks_over=dict(head_dim=64)), BAD, "heads of 64"),
    (dict(blocks_over=dict(kv_heads=1)), BAD, "x 1 heads"),
    (dict(blocks_over=dict(batch=3)), BAD, "blocks of 3"),
    (dict(blocks_over=dict(blocks=0)), BAD, "blocks=0"),
    (dict(blocks_over=dict(blocks=(1 << 25) + 1)), BAD, "blocks="),
    (dict(blocks_over=dict(k=P + 4)), BAD, "16-byte"),
    (dict(blocks_over=dict(v_scale=P + 2)), BAD, "misaligned scales"),
]


@pytest.mark.parametrize("fn", ["q3vl_kv_pack", "q3vl_kv_advance"])
@pytest.mark.parametrize("over,code,text", SHARED + [(dict(cache_len=None), BAD, "null"), (dict(packed_len=None), BAD, "null")])
def test_pack_refusals(fn, over, code, text):
    refused(pack(fn=fn, **over), code, text)


def test_caches_that_share_rows_are_not_written():
    for over in (dict(seq_stride=0), dict(head_stride=0)):
        refused(pack(cache_over=over), BAD, "share their rows")
        refused(unpack(cache_over=over), BAD, "share their rows")
    assert pack(cache_over=dict(seq_stride=0, batch=1), blocks_over=dict(batch=1), cache_len=None) == BAD
    assert "null" in q.last_error()


def test_pack_sizes_and_one_array():
    refused(pack(cache_over=dict(batch=1 << 20, max_seq=1 << 20), blocks_over=dict(batch=1 << 20)), UNS, "too large")
    refused(pack(fn="q3vl_kv_advance", packed_len=P), BAD, "one array")


def unpack(cache_over={}, blocks_over={}, **over):
    f = dict(blocks=ctypes.byref(blocks(**blocks_over)), packed_len=P, first=None, cache=ctypes.byref(cache(**cache_over)), count=64,
             stream=None)
    f.update(over)
    return qa._L().q3vl_kv_unpack(*f.values())


@pytest.mark.parametrize("over,code,text", SHARED + [
    (dict(packed_len=None), BAD, "null"),
    (dict(count=-1), BAD, "count=-1"),
    (dict(count=65), BAD, "max_seq=64"),
])
def test_unpack_refusals(over, code, text):
    refused(unpack(**over), code, text)


def test_unpack_of_nothing():
    assert unpack(count=0, packed_len=None) == q.OK


def attn(cache_over={}, blocks_over={}, **over):
    f = dict(q=P, ldq=512, out=2 * P, ldo=512, dtype=q.FP32, rows=3, heads=4, cache=ctypes.byref(cache(**cache_over)), row_start=P,
             cache_len=P, blocks=ctypes.byref(blocks(**blocks_over)), packed_len=P, mask=P, words=1, max_rows=3, max_len=0, window=0,
             sinks=0, scale=0.1, ws=None, wsb=0, stream=None)
    f.update(over)
    return qa._L().q3vl_long_attention(*f.values())


@pytest.mark.parametrize("over,code,text", SHARED[:1] + SHARED[2:] + [
    (dict(blocks=None), BAD, "come together"),
    (dict(packed_len=None), BAD, "come together"),
    (dict(heads=3), BAD, "multiple of kv_heads"),
    (dict(dtype=q.INT8), UNS, "dtype"),
    (dict(ldq=500), BAD, "row stride"),
    (dict(words=0), BAD, "mask_words"),
    (dict(max_rows=-1), BAD, "max_rows"),
    (dict(max_len=-1), BAD, "max_len"),
    (dict(window=-1), BAD, "window=-1"),
    (dict(window=9, sinks=-1), BAD, "sinks=-1"),
    (dict(sinks=4), BAD, "without a window"),
    (dict(window=2), UNS, "window=2 over masks of up to 3"),
    (dict(scale=math.nan), BAD, "scale"),
    (dict(scale=3e38), BAD, "scale"),
    (dict(out=P, ldo=600), BAD, "over q"),
    (dict(q=None), BAD, "null"),
    (dict(row_start=None), BAD, "null"),
    (dict(rows=1 << 30), UNS, "too large"),
    (dict(cache_over=dict(max_seq=2 ** 31 - 1000), blocks_over=dict(blocks=1 << 24)), UNS, "too many positions"),
])
def test_long_attention_refusals(over, code, text):
    refused(attn(**over), code, text)


def test_long_attention_empty_calls():
    assert attn(rows=0, q=None) == q.OK
    assert attn(max_rows=0, q=None) == q.OK
    L, c, p = qa._L(), cache(), blocks()
    assert L.q3vl_long_attention_workspace_bytes(1, 3, 1, 0, 0, 0, ctypes.byref(c), ctypes.byref(p)) == 0
    assert "multiple" in q.last_error()
    assert L.q3vl_long_attention_workspace_bytes(1, 4, 1, 0, 0, 2, ctypes.byref(c), None) == 0
    assert "window" in q.last_error()


def verify(**over):
    f = dict(x=P, ld=1000, dtype=q.FP32, draft=None, ldp=0, tokens=P, parents=P, row_start=P, accept_u=P, sample_u=P, batch=2, rows=8,
             V=1000, max_rows=8, temperature=1.0, accepted=P, path=P, next=P, ws=None, wsb=0, stream=None)
    f.update(over)
    return qa._L().q3vl_verify_drafts(*f.values())


@pytest.mark.parametrize("over,code,text", [
    (dict(dtype=q.INT8), UNS, "dtype"),
    (dict(V=0), BAD, "V=0"),
    (dict(ld=999), BAD, "ld=999"),
    (dict(draft=P, ldp=999), BAD, "ldp=999"),
    (dict(batch=-1), BAD, "batch"),
    (dict(max_rows=-1), BAD, "max_rows"),
    (dict(max_rows=1025), UNS, "at most 1024"),
    (dict(temperature=0.0), BAD, "temperature=0"),
    (dict(temperature=-1.0), BAD, "temperature"),
    (dict(temperature=math.nan), BAD, "temperature"),
    (dict(temperature=math.inf), BAD, "temperature"),
    (dict(temperature=1e-310), BAD, "temperature"),
    (dict(rows=(1 << 22) + 1), UNS, "too large"),
    (dict(V=(1 << 30) + 1, ld=1 << 31), UNS, "too large"),
    (dict(batch=(1 << 22) + 1), UNS, "too large"),
    (dict(x=None), BAD, "null"),
    (dict(row_start=None), BAD, "null"),
    (dict(sample_u=None), BAD, "null"),
    (dict(path=None), BAD, "null"),
    (dict(next=None), BAD, "null"),
    (dict(x=P + 2), BAD, "misaligned logits"),
    (dict(draft=P + 2, ldp=1000), BAD, "misaligned draft"),
    (dict(ws=P, wsb=16), BAD, "workspace too small"),
    (dict(ws=P + 16, wsb=1 << 30), BAD, "256-byte"),
])
def test_verify_refusals(over, code, text):
    refused(verify(**over), code, text)


def test_verify_empty_and_workspace():
    assert verify(batch=0, x=None) == q.OK
    size = qa._L().q3vl_verify_drafts_workspace_bytes
    assert size(0, 10) == 0 and size(10, 0) == 0
    for V in (1, 1000, 151936, 1 << 30):
        sizes = [size(M, V) for M in sorted({*range(1, 600), *(1 << i for i in range(23))})]
        assert all(0 < a <= b for a, b in zip(sizes, sizes[1:]))
        assert all(size(M, max(1, V - 1)) <= size(M, V) for M in (1, 61, 500))


@pytest.mark.parametrize("D", [64, 128])
def test_block_orders(D):
    """Each order names every (position, value) once."""
    for order in (ref.key_order, ref.value_order):
        p, d = order(D)
        assert sorted(zip(p.tolist(), d.tolist())) == [(i, j) for i in range(32) for j in range(D)]
        n = np.arange(32 * D).reshape(32, D) % 251 - 125
        assert (ref.from_bytes(ref.to_bytes(n, order), order) == n).all()


def test_verify_reference_keeps_the_targets_distribution():
    """The definition itself: over many draws a chain's and a tree's next tokens
    come as the target's probabilities say (five sigma)."""
    rng = np.random.default_rng(1)
    V, n = 5, 6000
    x = rng.standard_normal((3, V)) * 1.5
    p = np.exp(x) / np.exp(x).sum(1, keepdims=True)
    dr = np.exp(rng.standard_normal((3, V)))
    dr = (dr / dr.sum(1, keepdims=True)).astype(np.float32)
    first = np.zeros(V)
    for _ in range(n):
        tok = [0] + [int(rng.choice(V, p=dr[0].astype(float) / dr[0].astype(float).sum())) for _ in range(2)]
        a, path, nx = ref.verify(x, tok, [-1, 0, 0], [0, 3], rng.random(3), rng.random(3), 3, draft=dr)
        first[tok[path[0, 1]] if a[0] > 1 else nx[0]] += 1
    assert (np.abs(first / n - p[0]) < 5 * np.sqrt(p[0] / n)).all()
