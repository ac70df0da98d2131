"""GPU test of packing through a view of a cache's first rows, as a program does
that knows how many can have filled: what the whole cache would give, for
sequences whose rows are all in the view; the others are left alone."""
import numpy as np
import pytest

from test_gpu_long import Store, i32

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from q3vl_int8 import attention as qa  # noqa: E402


@pytest.mark.parametrize("by_row", [False, True])
@pytest.mark.parametrize("view", [64, 71])
def test_pack_through_a_view(view, by_row):
    cached, at = [33, 64, 17, 100, 63, 0], [0, 32, 64, 96, 128, 160]
    whole, part = (Store(7, len(cached), 2, 128, 500, 11, by_row).device() for _ in range(2))
    fits = [n if n <= view else 0 for n in cached]
    lens = [i32(fits), i32(at)], [i32(cached), i32(at)]
    few = qa.KVCache(*[x[:, :, :view] for x in part[0]])
    qa.kv_pack(whole[2], whole[3], *lens[0])
    qa.kv_pack(few, part[3], *lens[1])
    qa.kv_advance(whole[2], whole[3], *lens[0])
    qa.kv_advance(few, part[3], *lens[1])
    for x, y in zip(whole[0] + whole[1], part[0] + part[1]):
        assert torch.equal(x, y)
    assert lens[0][1].tolist() == lens[1][1].tolist()
    assert lens[1][0].tolist() == [a if n <= view else n for a, n in zip(lens[0][0].tolist(), cached)]
    assert np.array(lens[1][0].tolist()).max() == 100
