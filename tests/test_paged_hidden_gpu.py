"""What no row of a call may see reaches none of them, whatever the cache holds there: here the keys and values in front of every window, whose last ones lie in the
same tiles as visible ones (a weight of 0 times infinity or NaN would be NaN).  Behind a sequence's end and in missing pages: tests/test_paged_gpu.py."""
import pytest
import torch

from seq2seqsharp_b200.ops import Ops
from tests.test_paged_gpu import check, problem

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.mark.parametrize("stale", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("window", [1, 50, 200, 256])
@pytest.mark.parametrize("t,H,Hkv,hd,n", [(F16, 4, 1, 64, 1), (BF16, 8, 2, 128, 1), (F16, 8, 2, 128, 7), (BF16, 4, 2, 64, 16), (F16, 8, 2, 64, 30), (BF16, 8, 2, 128, 300), (F16, 3, 1, 128, 50),
                                          (F32, 2, 2, 64, 1), (F32, 4, 2, 128, 3), (F32, 4, 2, 64, 40), (F32, 2, 1, 128, 100), (BF16, 4, 2, 80, 2), (F16, 2, 1, 256, 9), (F32, 2, 1, 256, 20)])
def test_what_lies_in_front_of_every_window(cuda, t, H, Hkv, hd, n, window, stale):
    lens, new = [n + 700, n + 333, n + 20], [n, n, max(1, n // 2)]
    q, K, V, table, starts, lens_ = a = problem(t, H, Hkv, hd, 16, lens, new, seed=window, layout="tokens")
    for b in range(3):
        first = lens[b] - new[b] - window + 1                 # of the first row's window
        for i in range(first):
            K[table[b, i // 16], :, i % 16] = stale
            V[table[b, i // 16], :, i % 16] = stale
    got = Ops.PagedAttention(None, q, K, V, table, starts, lens_, n, window=window)
    finite = [x.nan_to_num(0.0, 0.0, 0.0) for x in (K, V)]
    assert check(got, q, *finite, table, starts, lens_, hd ** -0.5, window).all()
