"""Refusals and sizes of the operators for rows of tokens over the caches
(q3vl_draft_plan, q3vl_qk_norm_rope, q3vl_tree_attention,
q3vl_token_logprobs): every bad argument is turned away before any device
work, so this needs no GPU. Pointers are fake, aligned and never read."""
import ctypes
import math

import pytest

import q3vl_int8 as q
from q3vl_int8 import attention as qa

P = 1 << 20


def cache(**over):
    f = dict(k=P, v=P, batch=2, kv_heads=2, max_seq=64, head_dim=128, seq_stride=2 * 64 * 128, head_stride=64 * 128, row_stride=128)
    f.update(over)
    return qa._CacheC(*f.values())


def refused(rc, code, text):
    assert rc == code, q.last_error()
    assert text in q.last_error()


def plan(**over):
    f = dict(parents=P, row_start=P, cache_len=P, pos_delta=None, batch=2, rows=8, max_rows=8, max_seq=64, mask=P, words=1,
             pos=P, slots=P, stream=None)
    f.update(over)
    return qa._L().q3vl_draft_plan(*f.values())


@pytest.mark.parametrize("over,code,text", [
    (dict(batch=-1), q.ERR_INVALID_ARGUMENT, "batch"),
    (dict(max_rows=-1), q.ERR_INVALID_ARGUMENT, "max_rows"),
    (dict(max_rows=1025, words=17), q.ERR_UNSUPPORTED, "at most 1024"),
    (dict(max_rows=65), q.ERR_INVALID_ARGUMENT, "do not hold 65 rows"),
    (dict(max_seq=0), q.ERR_INVALID_ARGUMENT, "max_seq"),
    (dict(rows=1 << 31), q.ERR_UNSUPPORTED, "too large"),
    (dict(parents=None), q.ERR_INVALID_ARGUMENT, "null"),
    (dict(mask=None), q.ERR_INVALID_ARGUMENT, "null"),
    (dict(slots=None), q.ERR_INVALID_ARGUMENT, "null"),
])
def test_draft_plan_refusals(over, code, text):
    refused(plan(**over), code, text)


def rope_call(cache_over={}, norm_over={}, rope_over={}, **over):
    n = dict(q_w=P, q_s=P, k_w=P, k_s=P, group_size=64, eps=1e-6)
    n.update(norm_over)
    r = dict(cos=P, sin=P, rows=100, axes=1, sections=(0, 0, 0), interleaved=0)
    r.update(rope_over)
    r["sections"] = (ctypes.c_int * 3)(*r["sections"])
    f = dict(q=P, ldq=512, k=P, ldk=256, v=P, ldv=256, out=2 * P, ldo=512, dtype=q.FP32, rows=3, heads=4,
             cache=ctypes.byref(cache(**cache_over)), slots=P, pos=P, norm=ctypes.byref(qa._NormC(*n.values())),
             rope=ctypes.byref(qa._RopeC(*r.values())), stream=None)
    f.update(over)
    return qa._L().q3vl_qk_norm_rope(*f.values())


BAD, UNS = q.ERR_INVALID_ARGUMENT, q.ERR_UNSUPPORTED


@pytest.mark.parametrize("over,code,text", [
    (dict(cache_over=dict(head_dim=96, row_stride=96)), UNS, "head_dim=96"),
    (dict(cache_over=dict(k=None)), BAD, "null cache"),
    (dict(cache_over=dict(k=P + 8)), BAD, "aligned"),
    (dict(cache_over=dict(head_stride=100)), BAD, "aligned"),
    (dict(cache_over=dict(row_stride=64)), BAD, "strides"),
    (dict(cache_over=dict(row_stride=1 << 24)), BAD, "strides"),
    (dict(cache_over=dict(max_seq=0)), BAD, "bad cache"),
    (dict(cache_over=dict(max_seq=2 ** 31 - 1)), UNS, "too large"),
    (dict(cache=None), BAD, "null cache"),
    (dict(norm=None), BAD, "null norm"),
    (dict(dtype=q.INT8), UNS, "q_dtype"),
    (dict(heads=0), BAD, "heads"),
    (dict(ldq=500), BAD, "row stride"),
    (dict(ldv=255), BAD, "row stride"),
    (dict(out=P, dtype=q.FP16), BAD, "over q"),
    (dict(out=P, ldo=600), BAD, "over q"),
    (dict(norm_over=dict(group_size=48)), BAD, "group_size"),
    (dict(norm_over=dict(group_size=0)), BAD, "group_size"),
    (dict(norm_over=dict(k_s=None)), BAD, "null"),
    (dict(rope_over=dict(rows=0)), BAD, "tables"),
    (dict(rope_over=dict(axes=2)), UNS, "axes"),
    (dict(rope_over=dict(axes=3, sections=(24, 20, 19))), BAD, "not 64"),
    (dict(rope_over=dict(axes=3, sections=(84, -20, 0))), BAD, "section"),
    (dict(rope_over=dict(axes=3, sections=(20, 22, 22), interleaved=1)), BAD, "a third"),
    (dict(rope_over=dict(sin=None)), BAD, "null"),
    (dict(slots=None), BAD, "null"),
    (dict(rows=1 << 33), UNS, "too large"),
])
def test_qk_norm_rope_refusals(over, code, text):
    refused(rope_call(**over), code, text)


def attn(cache_over={}, **over):
    f = dict(q=P, ldq=512, out=P, ldo=512, dtype=q.FP32, rows=3, heads=4, cache=ctypes.byref(cache(**cache_over)), row_start=P,
             cache_len=P, mask=P, words=1, max_rows=3, max_len=0, scale=0.1, ws=None, wsb=0, stream=None)
    f.update(over)
    return qa._L().q3vl_tree_attention(*f.values())


@pytest.mark.parametrize("over,code,text", [
    (dict(cache_over=dict(head_dim=256, row_stride=256)), UNS, "head_dim=256"),
    (dict(cache_over=dict(batch=0)), BAD, "bad cache"),
    (dict(cache_over=dict(v=P + 2)), BAD, "aligned"),
    (dict(heads=3), BAD, "multiple of kv_heads"),
    (dict(heads=0), BAD, "multiple of kv_heads"),
    (dict(dtype=q.INT32), UNS, "dtype"),
    (dict(ldo=511), BAD, "row stride"),
    (dict(words=0), BAD, "mask_words"),
    (dict(mask=None, words=-1), BAD, "mask_words"),
    (dict(max_rows=-1), BAD, "max_rows"),
    (dict(max_len=-1), BAD, "max_len"),
    (dict(scale=math.inf), BAD, "scale"),
    (dict(scale=math.nan), BAD, "scale"),
    (dict(scale=3e38), BAD, "scale"),  # times log2 e it is none in fp32
    (dict(scale=-3e38), BAD, "scale"),
    (dict(q=None), BAD, "null"),
    (dict(cache_len=None), BAD, "null"),
    (dict(rows=1 << 30), UNS, "too large"),
    (dict(cache_over=dict(batch=1 << 24), rows=1 << 20, max_rows=64), UNS, "too large"),
])
def test_tree_attention_refusals(over, code, text):
    refused(attn(**over), code, text)


def logp(**over):
    f = dict(x=P, ld=1000, dtype=q.FP32, tokens=P, M=2, V=1000, k=5, lp=P, rank=None, ent=None, ids=P, top=P, ws=None, wsb=0, stream=None)
    f.update(over)
    return q.lib().q3vl_token_logprobs(*f.values())


@pytest.mark.parametrize("over,code,text", [
    (dict(dtype=q.INT8), UNS, "dtype"),
    (dict(V=0), BAD, "V=0"),
    (dict(ld=999), BAD, "ld=999"),
    (dict(k=-1), BAD, "top_k=-1"),
    (dict(k=65), BAD, "top_k=65"),
    (dict(V=3, k=4), BAD, "top_k=4"),
    (dict(M=(1 << 22) + 1), UNS, "too large"),
    (dict(V=(1 << 30) + 1, ld=1 << 31), UNS, "too large"),
    (dict(x=P + 2), BAD, "misaligned"),
    (dict(x=None), BAD, "null"),
    (dict(lp=None), BAD, "null"),
    (dict(ids=None), BAD, "null"),
    (dict(ws=P, wsb=16), BAD, "workspace too small"),
    (dict(ws=P + 16, wsb=1 << 30), BAD, "256-byte"),
])
def test_token_logprobs_refusals(over, code, text):
    refused(logp(**over), code, text)


def test_empty_calls_are_fine():
    """No rows: nothing to do, whatever the pointers."""
    assert plan(rows=0, parents=None) == q.OK
    assert rope_call(rows=0, q=None) == q.OK
    assert attn(rows=0, q=None) == q.OK
    assert attn(max_rows=0, q=None) == q.OK
    assert logp(M=0, x=None) == q.OK


def test_workspace_sizes():
    L = qa._L()
    c = cache(batch=1, max_seq=40000, kv_heads=8, head_stride=40000 * 128)
    one = L.q3vl_tree_attention_workspace_bytes(1, 16, 1, 40000, ctypes.byref(c))
    many = L.q3vl_tree_attention_workspace_bytes(8192, 16, 8192, 40000, ctypes.byref(c))
    assert one % 256 == 0 and many % 256 == 0 and one < 16 << 20
    assert L.q3vl_tree_attention_workspace_bytes(1, 15, 1, 40000, ctypes.byref(c)) == 0  # refused: its reason is told
    assert "multiple" in q.last_error()
    a, b = (q.lib().q3vl_token_logprobs_workspace_bytes(M, 151936) for M in (1, 512))
    assert 0 < a < b < 8 << 20
    assert q.lib().q3vl_token_logprobs_workspace_bytes(0, 10) == 0


def test_bindings_refuse_host_tensors():
    torch = pytest.importorskip("torch")
    x = torch.zeros((2, 128))
    i = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="device tensor"):
        q.token_logprobs(x, i)
    with pytest.raises(TypeError, match="torch.Tensor"):
        q.token_logprobs([1.0], i)
    with pytest.raises(ValueError, match="device tensor"):
        qa.KVCache(x.half().reshape(1, 1, 2, 128), x.half().reshape(1, 1, 2, 128))
    with pytest.raises(ValueError, match="device tensor"):
        qa.draft_plan(i, i, i, 10, 3)


@pytest.mark.parametrize("V", [1, 1000, 4096, 32000, 151936, 1 << 20, 1 << 30])
def test_logprobs_workspace_serves_fewer_rows(V):
    """A workspace for M rows holds what fewer rows, and shorter ones, need: the
    size asked for never falls with M or V."""
    size = q.lib().q3vl_token_logprobs_workspace_bytes
    rows = sorted({*range(1, 1200), *(1 << i for i in range(23)), *((1 << i) - 1 for i in range(11, 23))})
    sizes = [size(M, V) for M in rows]
    assert all(0 < a <= b for a, b in zip(sizes, sizes[1:]))
    assert all(size(M, max(1, V - 1)) <= size(M, V) and size(M, V // 2 + 1) <= size(M, V) for M in rows)


@pytest.mark.parametrize("over", [dict(out=P, ldo=600), dict(out=P, ldq=640)], ids=str)
def test_tree_attention_in_place_needs_one_stride(over):
    """out over q with another stride: its rows would lie over other rows'
    queries."""
    refused(attn(**over), BAD, "over q")
