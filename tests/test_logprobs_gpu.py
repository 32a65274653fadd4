"""Log probabilities of given tokens, entropy, rank and alternatives against 64 bits.

Tolerances count roundings, u = 2^-24: an exponent of the fp32 sums is off by u of itself and ex2 by 2 ulp (4 u), the sums by chains of at most 16 logits and of V / 4096 groups, so
log S is off by at most (80 + the mean exponent) u; a token's distance from the maximum is exact but for the constant log2 e (half an ulp of it); the result is
rounded once.  The mean of x - m is at most the entropy in size and is off by 80 u of itself.  Ranks and alternatives are exact."""
import numpy as np
import pytest
import torch

from seq2seqsharp_b200 import _native as N
from seq2seqsharp_b200.ops import Ops

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = 2.0 ** -24


def check(x, tokens, top, got=None):
    rows, V = x.shape
    lp, ent, rank, ids, best = got or Ops.TokenLogProbs(x, tokens, top)
    z = x.double().cpu().numpy()
    m = z.max(1, keepdims=True)
    e = np.exp(z - m)
    log_s = np.log(e.sum(1, keepdims=True))
    want = z - m - log_s
    p = np.exp(want)
    h = -(p * np.where(p > 0, want, 0)).sum(1)
    t = tokens.cpu().numpy()
    far = np.abs(z[np.arange(rows), t] - m[:, 0])
    long = V / 4096
    w = want[np.arange(rows), t]
    # log(sum) of a row whose probabilities are all tiny: the mean exponent is at most the entropy
    room = U * (80 + long + h + np.where(np.isfinite(far), 2 * far, 0) + np.where(np.isfinite(w), np.abs(w), 0))
    assert np.array_equal(np.isneginf(w), np.isneginf(lp.cpu().numpy()))
    fine = np.isfinite(w)
    assert (np.abs(lp.double().cpu().numpy() - w)[fine] <= room[fine]).all()
    assert (np.abs(ent.double().cpu().numpy() - h) <= U * (80 + long) * (1 + 2 * h)).all()
    at = z[np.arange(rows), t][:, None]
    j = np.arange(V)[None]
    assert np.array_equal(rank.cpu().numpy(), ((z > at) | ((z == at) & (j < t[:, None]))).sum(1))
    order = np.argsort(-z, axis=1, kind="stable")[:, :top]
    assert ids.shape == best.shape == (rows, top) and np.array_equal(ids.cpu().numpy(), order)
    b = np.take_along_axis(want, order, 1)
    fb = np.isfinite(b)
    assert np.array_equal(fb, np.isfinite(best.cpu().numpy()))
    if fb.any():
        assert (np.abs(best.double().cpu().numpy() - b)[fb] <= (U * (80 + long + h[:, None] + 3 * np.abs(b)))[fb]).all()


def rows_of(seed, rows, V, t, scale=2.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(rows, V, generator=g, device="cuda") * scale).to(t)
    return x, torch.randint(0, V, (rows,), generator=g, device="cuda").int()


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("rows,V,top", [(1, 1, 1), (1, 1, 0), (3, 5, 5), (2, 40, 32), (1, 2047, 1), (1, 2048, 32), (1, 32000, 5), (2, 50257, 20), (20, 50257, 32), (64, 4099, 7), (300, 2048, 1), (400, 999, 0),
                                        (500, 33, 32), (3, 131072, 32), (160, 9001, 20), (1, 1000003, 10)])
def test_log_probs(cuda, t, rows, V, top):
    check(*rows_of(rows + V, rows, V, t), top)


@pytest.mark.parametrize("t", [F32, F16, BF16])
def test_rows_that_start_anywhere(cuda, t):
    for rows, V, off, width in ((4, 1001, 1, 1003), (3, 50257, 5, 50300), (310, 700, 3, 711), (1, 9000, 7, 9007)):
        x, tok = rows_of(V, rows, width, t)
        check(x[:, off: off + V], tok.clamp(max=V - 1), 9)
    x, tok = rows_of(1, 1, 6000, t)
    check(x.expand(5, 6000), tok.expand(5).contiguous(), 3)


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("rows,V", [(1, 50257), (200, 3001), (2, 900)])
def test_equal_logits(cuda, t, rows, V):
    """Ties, of a few values and of all: more words reach the bound than a CTA orders at once."""
    x, tok = rows_of(3, rows, V, t)
    for y in (x.round(), x.sign(), torch.zeros_like(x), torch.full_like(x, -3.0), x.abs() * 0 - 0.0):
        check(y, tok, 32)
        check(y, tok, 1)


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("rows,V", [(1, 32000), (300, 1500), (3, 5000)])
@pytest.mark.parametrize("low", ["inf", "lowest"])
def test_masked_words(cuda, t, rows, V, low):
    """Words that cannot come: runs of them, all but a few, all but one; by -infinity and by the type's lowest value."""
    x, tok = rows_of(4, rows, V, t)
    mask = -float("inf") if low == "inf" else torch.finfo(t).min
    for keep in (slice(0, 700), slice(V - 300, V), slice(100, 111), slice(V // 2, V // 2 + 1)):
        y = torch.full_like(x, mask)
        y[:, keep] = x[:, keep]
        check(y, tok, 20)
        check(y, torch.full_like(tok, keep.start), 1)


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("rows,V", [(1, 50257), (40, 9000), (300, 1500)])
def test_fewer_words_than_alternatives(cuda, t, rows, V):
    """Alternatives that cannot come follow by index, those at the row's ends and behind its last piece too; a NaN comes after them."""
    x, tok = rows_of(11, rows, V + 1, t)
    for off in (0, 1):
        z = x[:, off: off + V]
        for keep in ([], [3, V // 2], list(range(0, 10)), [V - 1, V - 2], list(range(31)), list(range(0, V, V // 33))[:33]):
            y = torch.full_like(z, -float("inf"))
            y[:, keep] = z[:, keep]
            if keep:
                check(y, torch.full_like(tok, keep[0]), 32)
            order = torch.sort(y.float(), dim=1, descending=True, stable=True).indices[:, :32].int()
            wide = torch.empty(rows, V + 1, dtype=t, device="cuda")
            wide[:, off: off + V] = y
            got = Ops.TokenLogProbs(wide[:, off: off + V], tok, 32)
            assert torch.equal(got[3], order)
    y = torch.full((rows, V), float("nan"), dtype=t, device="cuda")
    y[:, V - 3] = 1
    y[:, 5] = -float("inf")
    ids = Ops.TokenLogProbs(y, tok, 4)[3]
    assert (ids == torch.tensor([V - 3, 5, 0, 1], dtype=torch.int32, device="cuda")).all()


@pytest.mark.parametrize("t", [F32, F16, BF16])
def test_rows_of_the_lowest_value_are_uniform(cuda, t):
    for rows, V in ((1, 32000), (200, 1000)):
        x = torch.full((rows, V), torch.finfo(t).min, dtype=t, device="cuda")
        check(x, torch.full((rows,), 17, dtype=torch.int32, device="cuda"), 3)


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("V", [3, 3000, 50257])
def test_rows_without_a_distribution(cuda, t, V):
    x, tok = rows_of(5, 5, V, t)
    x[1] = -float("inf")
    x[2, V // 2] = float("nan")
    x[3, V - 1] = float("inf")
    lp, ent, rank, ids, best = Ops.TokenLogProbs(x, tok, 3)
    for r in (1, 2, 3):
        assert lp[r].isnan() and ent[r].isnan() and best[r].isnan().all()
    assert ids[1].tolist() == [0, 1, 2] and ids[3, 0] == V - 1
    z = x[2].double().cpu().numpy()
    assert ids[2].tolist() == np.argsort(-np.where(np.isnan(z), -np.inf, z), kind="stable")[:3].tolist()   # a NaN comes last
    keep = [0, 4]
    check(x[keep], tok[keep], 3, tuple(v[keep] for v in (lp, ent, rank, ids, best)))


def test_rows_without_a_token(cuda):
    x, _ = rows_of(6, 4, 500, F32)
    tok = torch.tensor([-1, 499, 500, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    lp, ent, rank, ids, _ = Ops.TokenLogProbs(x, tok, 2)
    assert lp[0] == 0 and rank[0] == -1 and lp[2:].isnan().all() and (rank[2:] == -1).all() and ent.isfinite().all()
    check(x[1:2], tok[1:2], 2, tuple(v[1:2] for v in Ops.TokenLogProbs(x, tok, 2)))
    assert torch.equal(ids, x.topk(2, 1).indices.int())


def test_certain_tokens_keep_their_digits(cuda):
    """A word whose probability is 1 - 1e-6: its log probability is the sum of the others', but for those that one thread adds to the 1 in fp32 (at
    most 12 of 3000, 20 of 40000: 1 part in 250; a sum in fp32 would have 1 part in 17)."""
    for V in (40000, 3000):
        x = torch.zeros(2, V, device="cuda")
        x[:, 7] = float(np.log(V * 1e6))
        lp, ent, rank, ids, _ = Ops.TokenLogProbs(x, torch.tensor([7, 7], dtype=torch.int32, device="cuda"), 1)
        want = -np.log1p((V - 1) * np.exp(-float(x[0, 7])))
        assert abs(lp[0].item() / want - 1) < 5e-3 and lp[0] == lp[1] and rank.tolist() == [0, 0] and ids.tolist() == [[7], [7]]
        assert ent[0] >= 0


def test_the_same_from_call_to_call_and_in_a_graph(cuda):
    x, tok = rows_of(8, 70, 20011, BF16)
    want = Ops.TokenLogProbs(x, tok, 32)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = Ops.TokenLogProbs(x, tok, 32)
    for _ in range(3):
        g.replay()
        again = Ops.TokenLogProbs(x, tok, 32)
        for a, b, c in zip(want, out, again):
            assert torch.equal(a, b) and torch.equal(a, c)
    y, other = rows_of(9, 70, 20011, BF16)
    x.copy_(y)
    tok.copy_(other)
    g.replay()
    check(x, tok, 32, out)


def test_refusals(cuda):
    x, tok = rows_of(1, 2, 20, F32)
    for call, words in ((lambda: Ops.TokenLogProbs(x, tok, 21), "alternatives"), (lambda: Ops.TokenLogProbs(x, tok, 33), "alternatives"), (lambda: Ops.TokenLogProbs(x, tok.long()), "tokens"),
                        (lambda: Ops.TokenLogProbs(x, tok[:1]), "tokens"), (lambda: Ops.TokenLogProbs(x.int(), tok), "unsupported"), (lambda: Ops.TokenLogProbs(x.t(), tok), "logits"),
                        (lambda: Ops.TokenLogProbs(x[0], tok), "unsupported")):
        with pytest.raises(N.TSB200Error, match=words):
            call()
    assert Ops.TokenLogProbs(x[:0], tok[:0], 3)[3].shape == (0, 3)
