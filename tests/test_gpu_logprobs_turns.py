"""GPU tests of the log probabilities over so many rows that a wave of the scan
has several turns: the turn's values are loaded a turn ahead, the running
maximum moves and rescales the sums, and finite turns take a shorter path. A
sample of the rows is checked against the plain 64-bit form (rows_ref.py)."""
import math

import numpy as np
import pytest

import rows_ref as ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import q3vl_int8 as q  # noqa: E402

LOWEST = float(np.finfo(np.float32).min)


def turns_of(V, off=0):
    return -(-(V + off) // 1024)


def several_turns(M, V):
    """Waves get a second turn from 4 x 4096 turns over all rows on, in rows of
    more turns than a block has waves."""
    assert turns_of(V) > 4 and turns_of(V) * M >= 16384, "every wave has one turn: the case shows nothing"


def logits(M, V, half, seed, off=0, pad=0):
    """[M, V] on the device, as a view that starts `off` into wider rows."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    wide = torch.empty((M, V + off + pad), dtype=torch.float16 if half else torch.float32, device="cuda")
    return wide.normal_(0, 3, generator=g)[:, off:off + V]


def check(x, tokens, k, rows):
    """One call over all of x; `rows` of it against 64 bits.

    The sum r of the weights e^(x - m): the exponent (x - m) log2 e is rounded
    three times (2^-24 each, of at most 21 for weights that count) and its power
    of two is good to 2^-23: 21 2^-23 with room. Additions of a lane in order
    and the joins: half a step each, fewer than 4 V^0.5 at every size here.
    Entropy: the sum of w (x - m) has the same errors of each term, and log1p(r)
    and t / s add up."""
    M, V = x.shape
    several_turns(M, V)
    r = q.token_logprobs(x, torch.tensor(tokens, dtype=torch.int32, device="cuda"), top_k=k)
    lp, rank, ent, ids, top = (a.cpu().numpy() for a in r)
    e = 21 * 2.0 ** -23 + V ** 0.5 * 2.0 ** -22
    for m in rows:
        row = x[m].cpu().numpy()
        elp, erank, eent, eids, etop = ref.logprobs(row, int(tokens[m]), k)
        np.testing.assert_array_equal(ids[m], eids, err_msg=f"row {m}")
        assert rank[m] == erank, (m, rank[m], erank)
        logs = eent if np.isfinite(eent) else 1.0  # (log s is at most the entropy)
        for got, want in [(lp[m], elp)] + list(zip(top[m], etop)):
            with np.errstate(over="ignore"):
                single = np.float32(want)  # (-inf past fp32's range)
            if not np.isfinite(single):
                want = single
                assert (np.isnan(want) and np.isnan(got)) or got == want, (m, got, want)
            else:
                assert abs(got - want) <= e * min(math.expm1(min(logs, 50.0)), 1.0) + (abs(want) + logs) * 2.0 ** -22, (m, got, want)
        if np.isfinite(eent):
            assert abs(ent[m] - eent) <= 4 * e * eent + 1e-30, (m, ent[m], eent)
        else:
            assert np.isnan(ent[m]), (m, ent[m])


@pytest.mark.parametrize("M,V", [(120, 151936), (600, 32000)], ids=str)
def test_lowest_values_in_later_turns(M, V):
    """The type's lowest value as a mask, and other values near its end, beside
    ordinary ones and beside the largest there are: the entropy is that of the
    rest. Whatever part of a row a wave has, some of its later turns hold them."""
    x = logits(M, V, False, 1)
    x[0, V // 9:] = LOWEST
    x[1, ::2] = LOWEST
    x[2, 1::1024] = LOWEST
    x[3, V // 2:] = -3e38
    x[4, 700::1000] = -2.4e38
    x[5, V - 1] = LOWEST
    x[6] = LOWEST
    x[6, V - 5] = 2.0
    x[7, 1::2] = LOWEST
    x[7, V - 300] = 3e38   # x - m itself is -inf
    x[8, :] = -2e38
    x[8, V // 2:] = 2e38   # the same among many
    x[9, ::2] = 1e30       # just where x - m stays finite
    x[9, 1::2] = LOWEST
    x[10, :] = LOWEST      # all equal
    x[11, 5::7] = -math.inf
    x[11, 6::7] = LOWEST
    tokens = [(m * 977 + V - 1) % V for m in range(M)]
    check(x, tokens, 5, list(range(12)) + [M - 1])


@pytest.mark.parametrize("k", [0, 20, 64])
@pytest.mark.parametrize("half", [False, True], ids=["fp32", "fp16"])
@pytest.mark.parametrize("M,V,off,pad", [(120, 151936, 0, 0), (600, 151936, 3, 1), (1200, 32000, 0, 64), (3001, 8191, 1, 0)], ids=str)
def test_later_turns(M, V, off, pad, half, k):
    """The maximum in the first, a middle or the last turn, or moving in every
    one; what is no number, or rules a value out, only from a late turn on;
    tokens at both ends and in the middle; rows that start anywhere."""
    x = logits(M, V, half, M + V, off, pad)
    rise = torch.linspace(-9, 9, V, device="cuda")
    x[0], x[1] = rise, -rise
    x[2, 3], x[3, V // 2 + 1], x[4, V - 2] = 25.0, 25.0, 25.0
    x[5, V - 7] = math.nan
    x[6, V // 3] = math.inf
    x[7, V * 3 // 4:] = -math.inf
    x[8, :V - 40] = -math.inf
    x[9] = torch.randint(-2, 3, (V,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(k)).to(x.dtype)
    x[10, V // 2] = math.nan
    x[10, V // 2 + 1] = -math.inf
    x[11] = -math.inf
    x[12, V // 5:V // 4] = float(torch.finfo(x.dtype).min)
    ends = [0, V - 1, V // 2, 1, V - 2, V // 2 + 1, 1023 % V, 1024 % V]
    tokens = [ends[m % 8] for m in range(M)]
    tokens[3], tokens[4], tokens[7], tokens[8], tokens[9], tokens[12] = V // 2 + 1, V - 2, V - 1, V - 3, V - 4, V // 5 + 3
    tokens[13], tokens[14] = -1, V
    check(x, tokens, k, list(range(16)) + [M // 2, M - 2, M - 1])


def test_row_counts_agree():
    """The same row gives the same ids and rank however many others there are,
    with one turn a wave and with several."""
    V, k = 151936, 20
    x = logits(600, V, False, 7)
    tokens = torch.arange(0, 600 * 250, 250, dtype=torch.int32, device="cuda")
    want = q.token_logprobs(x, tokens, top_k=k)
    for M in (1, 109, 110, 223, 599):
        r = q.token_logprobs(x[:M], tokens[:M], top_k=k)
        assert torch.equal(r.rank, want.rank[:M]) and torch.equal(r.top_ids, want.top_ids[:M])
        # both are off by at most the bound that `check` derives
        e = 21 * 2.0 ** -23 + V ** 0.5 * 2.0 ** -22
        assert ((r.logprob - want.logprob[:M]).abs().double() <= 2 * (e + 30 * 2.0 ** -22)).all()
        assert ((r.entropy - want.entropy[:M]).abs().double() <= 2 * 4 * e * want.entropy[:M].double()).all()


@pytest.mark.parametrize("most,V", [(333, 151936), (777, 151936), (512, 32000)], ids=str)
def test_one_workspace_for_fewer_rows(most, V):
    """A workspace for the largest batch serves the smaller ones, those that
    are split into more parts among them."""
    x = logits(most, V, True, 11)
    tokens = torch.arange(most, dtype=torch.int32, device="cuda")
    ws = q.alloc_token_logprobs_workspace(most, V)
    for M in sorted({1, 109, 110, 322, 329, 426, 511, 768, 769, most}):
        if M <= most:
            r = q.token_logprobs(x[:M], tokens[:M], top_k=3, workspace=ws)
            own = q.token_logprobs(x[:M], tokens[:M], top_k=3, workspace=q.alloc_token_logprobs_workspace(M, V))
            assert all(torch.equal(a, b) for a, b in zip(r, own)), M
