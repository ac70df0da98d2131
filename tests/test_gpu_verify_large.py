"""GPU tests of judged drafts where rows are cut into large chunks (more than
4095 chunks of 2048 values in a call): both types, with and without draft
probabilities, odd strides, and rows that reject more children than the rounds
that all workgroups share."""
import numpy as np
import pytest

from test_gpu_verify import Drafts, dev

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("V,rows", [(151936, [40, 1, 0, 19]), (60001, [90, 60])], ids=str)
@pytest.mark.parametrize("probs", [False, True], ids=["certain", "probs"])
@pytest.mark.parametrize("half", [False, True], ids=["fp32", "fp16"])
def test_large_chunks(half, probs, V, rows):
    d = Drafts(V + half, rows, V, True, probs, half, spread=1.5, near=1.5)
    assert d.x.shape[0] * -(-V // 2048) >= 4096
    for s, n in zip(d.start, rows):  # eight children, drawn from their parent's draft anew
        for t in range(1, min(n, 9)):
            d.parents[s + t] = 0
            if probs:
                c = np.cumsum(d.draft[s].astype(np.float64))
                d.tokens[s + t] = min(V - 1, int(np.searchsorted(c / c[-1], d.rng.random())))
    if probs:  # the first four are tokens that the draft gives more than the target: with these numbers all rejected
        p = np.exp((d.x[0].astype(np.float64) - d.x[0].max()) / 0.9)
        d.tokens[1:5] = np.argsort(p / p.sum() - d.draft[0])[:4]
        d.ua[1:5] = 1 - 2.0 ** -24
    d.us[::3] = 1 - 2.0 ** -20  # tokens from the rows' ends
    want = d.check(temperature=0.9)
    if probs:
        assert want[0][0] == 1 or want[1][0, 1] > 4
    # the same rows as views of wider, oddly placed ones
    wide = torch.full((len(d.x), V + 21), float("nan"), device="cuda").to(torch.float16 if half else torch.float32)
    wide[:, 13:13 + V] = dev(d.x)
    over = dict(logits=wide[:, 13:13 + V], temperature=0.9)
    if probs:
        pw = torch.full((len(d.x), V + 3), float("nan"), device="cuda")
        pw[:, 1:1 + V] = dev(d.draft)
        over["draft_probs"] = pw[:, 1:1 + V]
    for g, w in zip(d.run(**over), want):
        np.testing.assert_array_equal(g, w)
