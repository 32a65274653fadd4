"""Attention over pages for every way in which a CTA looks for its run: 32 sequences and fewer (a warp by itself), as many as the CTA has threads (one scan; 128, 160,
256 and 384 threads, by kernel), and more (a scan per so many), one to both sides of each border."""
import numpy as np
import pytest
import torch

from seq2seqsharp_b200.ops import Ops
from tests.test_paged_gpu import check, problem

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.mark.parametrize("B", [31, 32, 33, 64, 127, 128, 129, 160, 161, 255, 256, 257, 384, 385])
@pytest.mark.parametrize("t,H,Hkv,hd,n", [(F16, 8, 2, 64, 1), (BF16, 4, 1, 128, 5), (F16, 4, 1, 128, 40), (BF16, 6, 2, 64, 30), (F32, 2, 2, 64, 1), (F32, 4, 1, 64, 24), (BF16, 4, 2, 80, 3)])
def test_every_number_of_sequences(cuda, t, H, Hkv, hd, n, B):
    rng = np.random.default_rng(B + n)
    new = [n] + [int(x) for x in np.where(rng.random(B - 1) < 0.1, 0, rng.integers(1, n + 1, B - 1))]
    lens = [m + int(x) for m, x in zip(new, rng.integers(0, 400, B))]
    lens[B - 1] += 3000                                       # the last of them is the longest: ends of runs lie behind all the others
    a = problem(t, H, Hkv, hd, 16, lens, new, seed=B)
    got = Ops.PagedAttention(None, *a[:4], a[4], a[5], n)
    assert check(got, *a, hd ** -0.5).all()
    for _ in range(20):                                       # whichever warp comes first
        assert torch.equal(got, Ops.PagedAttention(None, *a[:4], a[4], a[5], n))


@pytest.mark.parametrize("t,n", [(F16, 1), (F16, 12), (F32, 1), (F32, 20)])
def test_a_batch_of_equal_sequences(cuda, t, n):
    # 64 of the same length: every run ends inside a sequence, most of them beyond the first 32
    a = problem(t, 8, 2, 64, 16, [700] * 64, [n] * 64, seed=3)
    got = Ops.PagedAttention(None, *a[:4], a[4], a[5], n)
    assert check(got, *a, 0.125).all()
    for _ in range(50):
        assert torch.equal(got, Ops.PagedAttention(None, *a[:4], a[4], a[5], n))
