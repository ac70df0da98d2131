"""Workspaces of the attention over long contexts: the bytes for as many rows
serve any call of no more. Sizes alone need no GPU; a server's calls of fewer
and fewer rows with one workspace do."""
import ctypes

import numpy as np
import pytest

import q3vl_int8 as q
from q3vl_int8 import attention as qa
from test_long_capi import blocks
from test_rows_capi import cache

torch = pytest.importorskip("torch")

ROWS = sorted({*range(1, 150), *(1 << i for i in range(18)), *(5 << i for i in range(15)), 511, 513, 1000, 1001, 4097, 100000})


@pytest.mark.parametrize("packed", [True, False], ids=["packed", "fp16 rows"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (4096, 4)], ids=str)
@pytest.mark.parametrize("D,heads,kv_heads", [(128, 16, 8), (64, 12, 4), (128, 32, 4), (64, 5, 5)], ids=str)
def test_bytes_never_fall_with_more_rows(packed, window, sinks, D, heads, kv_heads):
    size = qa._L().q3vl_long_attention_workspace_bytes
    some = 0
    for batch in (1, 3, 16, 64):
        for n in (64, 700):  # blocks
            for max_rows in (1, 9, 32, 100, 3000):
                c = cache(batch=batch, kv_heads=kv_heads, head_dim=D, row_stride=D, max_seq=2048 if packed else 32 * n)
                p = ctypes.byref(blocks(batch=batch, kv_heads=kv_heads, head_dim=D, blocks=n)) if packed else None
                got = [size(r, heads, max_rows, 0, window, sinks, ctypes.byref(c), p) for r in ROWS]
                assert all(a <= b for a, b in zip(got, got[1:])), (batch, n, max_rows)
                some += sum(x > 0 for x in got)
                if max_rows * heads // kv_heads > 64:  # not without measure: no more than the most splits of all its rows
                    assert all(x <= r * heads * 32 * (4 * D + 8) + 512 for x, r in zip(got, ROWS))
    assert some > 1000


@pytest.mark.gpu
@pytest.mark.parametrize("packed", [True, False], ids=["packed", "fp16 rows"])
def test_one_workspace_for_steps_of_fewer_rows(packed):
    """The same max_rows, workspace and batch; step by step other rows take part,
    and each row's result is what a workspace of the step's own gives."""
    rng = np.random.default_rng(3)
    i32 = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")  # noqa: E731
    for B, max_rows, held in ((1, 9, 1984), (16, 32, 1984), (3, 100, 4064), (1, 300, 960)):
        H, Hk, D, S = 16, 8, 128, max_rows + 64
        g = torch.Generator(device="cuda").manual_seed(max_rows)
        k, v = (torch.randn((B, Hk, held + S if not packed else S, D), device="cuda", generator=g).half() for _ in range(2))
        c, kw = qa.KVCache(k, v), {}
        lens = i32([50 if packed else held] * B)
        if packed:
            p = qa.alloc_packed_kv(B, Hk, held, D)
            p.k.random_(-127, 128), p.v.random_(-127, 128), p.k_scale.uniform_(0.005, 0.02), p.v_scale.uniform_(0.005, 0.02)
            kw = dict(packed=p, packed_len=i32([held] * B))
        N = B * max_rows
        ws = qa.alloc_long_attention_workspace(c, N, H, max_rows, packed=kw.get("packed"))
        for rows in sorted({1, 2, 3, 5, 8, 9, 16, 17, 33, 64, 65, N // 2, N - 1, N}, reverse=True):
            if rows > N or rows < 1:
                continue
            cut = np.sort(rng.integers(0, rows + 1, B - 1))
            start = np.concatenate([[0], np.minimum(cut, np.arange(1, B) * max_rows), [rows]])
            if np.diff(start).max() > max_rows or np.diff(start).min() < 0:
                start = np.minimum(np.arange(B + 1) * max_rows, rows)
            x = torch.randn((rows, H * D), device="cuda", generator=g)
            mine = qa.long_attention(x, c, i32(start), lens, max_rows, workspace=ws, **kw)
            own = qa.alloc_long_attention_workspace(c, rows, H, max_rows, packed=kw.get("packed"))
            assert own.numel() <= ws.numel()
            assert torch.equal(mine, qa.long_attention(x, c, i32(start), lens, max_rows, workspace=own, **kw))
