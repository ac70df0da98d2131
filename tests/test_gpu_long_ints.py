"""GPU tests of numbers that a C int does not hold: the bindings of the operators
for long contexts and judged drafts refuse them, where their low bits would make
another call."""
import pytest

from test_gpu_long import Long, i32
from test_gpu_verify import Drafts

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import q3vl_int8 as q  # noqa: E402
from q3vl_int8 import attention as qa  # noqa: E402

WIDE = pytest.mark.parametrize("n", [1 << 31, (1 << 32) + 5, 1 << 63, (1 << 63) - 1], ids=["2^31", "2^32+5", "2^63", "2^63-1"])


@WIDE
def test_attention(n):
    B = Long(1, [2], [20], [64], 4, 2, 64, False, False, window=5)
    for over in (dict(window=n), dict(sinks=n), dict(max_rows=n), dict(max_len=n)):
        with pytest.raises(ValueError, match="below 2\\^31"):
            B.run(**over)
        a = dict(window=5, sinks=0, max_rows=2, max_len=0) | over
        with pytest.raises(ValueError, match="below 2\\^31"):
            qa.alloc_long_attention_workspace(qa.KVCache(*[torch.zeros((1, 2, 32, 64), dtype=torch.float16, device="cuda")] * 2), 2, 4, **a)
    B.window = (1 << 31) - 1  # the most there is
    B.check(B.run())


@WIDE
def test_unpack(n):
    kv = [torch.zeros((1, 2, 64, 64), dtype=torch.float16, device="cuda") for _ in range(2)]
    with pytest.raises(ValueError, match="below 2\\^31"):
        qa.kv_unpack(qa.alloc_packed_kv(1, 2, 64, 64), i32([64]), qa.KVCache(*kv), count=n)


@WIDE
def test_verify(n):
    with pytest.raises(ValueError, match="below 2\\^31"):
        Drafts(1, [1], 5, False, False).run(max_rows=n)


def test_negative_ones_are_still_refused():
    B = Long(1, [2], [20], [64], 4, 2, 64, False, False)
    with pytest.raises(q.Q3VLError, match="window=-1"):
        B.run(window=-1)
    with pytest.raises(q.Q3VLError, match="max_rows=-3"):
        B.run(max_rows=-3)
