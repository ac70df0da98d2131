"""GPU tests of queries so small that the score's factor (log2 e over the
queries' power of two) has no finite inverse: rows of one wave that begin to see
positions at different ones, in both attentions over rows of tokens. Scores are
0 to within 2^-80 then, so a row is the mean of the values that it sees."""
import numpy as np
import pytest

from test_gpu_long import Long

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from q3vl_int8 import attention as qa  # noqa: E402

SIZES = pytest.mark.parametrize("qscale", [1e-34, 1e-37, 1e-40])


@SIZES
@pytest.mark.parametrize("T", [2, 7, 20, 80])
@pytest.mark.parametrize("held", [False, True], ids=["fp16 rows", "packed"])
def test_windows(T, held, qscale):
    for window in (50, 100, 131):
        B = Long(T + window, [T, 2], [300, 150], [160, 320] if held else None, 4, 2, 64, False, False, window=window, qscale=qscale)
        B.check(B.run())


@SIZES
@pytest.mark.parametrize("T", [16, 100, 190])
@pytest.mark.parametrize("H,Hk", [(2, 2), (4, 2)], ids=str)
def test_masks(T, H, Hk, qscale):
    """Nothing cached: every other row sees no draft before the 33rd (or T / 2)."""
    B = Long(T, [T, 40], [0, 0], None, H, Hk, 128, False, True, qscale=qscale)
    for r in range(B.mask.shape[0]):
        t = r if r < T else r - T
        n = (T, 40)[r >= T]
        first = 0 if t % 2 == 0 else min(32, n // 2)
        bits = sum(1 << i for i in range(first, n))
        for w in range(B.mask.shape[1]):
            B.mask[r, w] = bits >> 64 * w & (1 << 64) - 1
    B.check(B.run())
    a = {n: v for n, v in B.tensors().items() if n not in ("window", "sinks")}
    got = qa.tree_attention(**a)
    torch.cuda.synchronize()
    B.check(got.cpu().numpy())
