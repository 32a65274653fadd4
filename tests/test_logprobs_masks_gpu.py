"""Log probabilities of rows with large finite logits: words masked by constants, maxima far from zero, logits around the size from which exponents are taken as differences.

Tolerances: those of test_logprobs_gpu.check.  From that size on an exponent is a difference (exact between numbers within a factor of two, else half a step, u = 2^-24), times log2 e
(0.3 u off), rounded: 2.3 u of itself where products are 1.3 u off.  The mean exponent is at most the entropy, here at most 12, so that log S is off by 12 u more at most, of which the 80 u of check()
have room (ex2 4 u, chains of sums 32 u)."""
import pytest
import torch

from seq2seqsharp_b200.ops import Ops
from tests.test_logprobs_gpu import BF16, F16, F32, check, rows_of

pytestmark = pytest.mark.gpu
SHAPES = [(1, 32000), (300, 1500), (3, 5000), (64, 50257)]


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("rows,V", SHAPES)
@pytest.mark.parametrize("mask", [-1e4, -1e6, -1e9, -1e10, -1e20, -1e30, -1e37, -1.5e38, -3e38])
def test_words_masked_by_a_constant(cuda, t, rows, V, mask):
    x, tok = rows_of(14, rows, V, t)
    for keep in (slice(0, 700), slice(V - 300, V), slice(100, 111), slice(V // 2, V // 2 + 1), slice(0, V, 97)):
        y = torch.full_like(x, mask)
        y[:, keep] = x[:, keep]
        check(y, tok, 20)
        check(y, torch.full_like(tok, keep.start), 1)
        check(y, tok, 0)


@pytest.mark.parametrize("rows,V", SHAPES[:3])
@pytest.mark.parametrize("mask", [-1e4, -3e4, -6e4])
def test_words_masked_by_a_constant_of_fp16(cuda, rows, V, mask):
    x, tok = rows_of(15, rows, V, F16)
    for keep in (slice(100, 111), slice(V // 2, V // 2 + 1), slice(0, V, 97)):
        y = torch.full_like(x, mask)
        y[:, keep] = x[:, keep]
        check(y, tok, 20)


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("rows,V", SHAPES[:3])
@pytest.mark.parametrize("to", [-3e38, -1e30, -1e10, -1e7, 1e7, 1e10, 1e20, 1e37, 3e38])
def test_rows_of_one_far_value(cuda, t, rows, V, to):
    """Uniform rows, and rows with one maximum far above the rest."""
    x, tok = rows_of(16, rows, V, t)
    check(torch.full_like(x, to), tok, 5)
    y = x.clone()
    y[:, V // 3] = abs(to)
    check(y, tok, 5)
    check(y, torch.full_like(tok, V // 3), 1)


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("rows,V", SHAPES[:3])
def test_masks_of_several_values(cuda, t, rows, V):
    """Constants of different sizes in one row, with -infinity and the type's lowest value among them: a mask added to logits that were masked already."""
    x, tok = rows_of(17, rows, V, t)
    some = torch.tensor([-1e4, -1e6, -2e9, -1e10, -1e20, -1e30, -1e37, -3e38, torch.finfo(t).min, -float("inf")], device="cuda").to(t)
    at = torch.randint(0, len(some), (rows, V), device="cuda", generator=torch.Generator(device="cuda").manual_seed(5))
    for keep in (slice(100, 111), slice(0, V, 97), slice(V, V)):
        y = some[at]
        y[:, keep] = x[:, keep]
        check(y, tok, 20)


@pytest.mark.parametrize("rows,V", SHAPES)
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("base", [1e4, 1e5, 2.0 ** 20, 2.0 ** 20 + 6, 2.0 ** 22, 1e7, 2.0 ** 24, 1e8])
def test_logits_far_from_zero(cuda, rows, V, sign, base):
    """Distributions in fp32 around a value of every size that leaves them more than one step: maxima of threads fall on both sides of the border."""
    x, tok = rows_of(18, rows, V, F32)
    check(sign * base + x, tok, 20)
    check(sign * base + 4 * x, tok, 1)


def test_far_masks_in_a_graph_and_from_call_to_call(cuda):
    x, tok = rows_of(19, 40, 20011, F32)
    y = torch.full_like(x, -1e10)
    y[:, 5:900] = x[:, 5:900]
    want = Ops.TokenLogProbs(y, tok, 20)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = Ops.TokenLogProbs(y, tok, 20)
    g.replay()
    for a, b in zip(want, out):
        assert torch.equal(a, b)
    y[:, 5:900] = -1e30
    y[:, 7000:7003] = x[:, 7000:7003]
    g.replay()
    check(y, tok, 20, out)
