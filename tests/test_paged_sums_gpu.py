"""The paged cache's numbers where a systematic error would hide behind random ones: weights that all round the same way."""
import math

import pytest
import torch

from seq2seqsharp_b200.ops import Ops
from tests import paged_reference as R

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ---------------------------------------------------------------------------------------------------------------------------- weights
@pytest.mark.parametrize("up", [0.9, -0.9, 0.6])
@pytest.mark.parametrize("t,n,hd,T", [(BF16, 20, 64, 500), (BF16, 20, 128, 500), (F16, 20, 64, 500), (F16, 300, 128, 500), (BF16, 200, 128, 5000), (F16, 1, 128, 500), (BF16, 1, 64, 900),
                                      (BF16, 7, 128, 2000), (F16, 1, 80, 300), (F32, 1, 64, 700), (F32, 40, 64, 700)])
def test_the_mean_of_equal_values_is_the_value(cuda, t, n, hd, T, up):
    """Weights of one key 1, of all others w = 1/2 + up * half a step of the type: rounded to 16 bits each of them is off by nearly half a step, all to the same side.
    Every value is 1, so the output is 1 whatever the weights are, if numerator and denominator are sums of the same numbers: both are fp32 sums of at most T
    of them, off by T 2^-24 each at most, which is less than half a step of the 16-bit types (2^-9, 2^-12 below 1) and what fp32 is allowed."""
    H, Hkv, page = 4, 1, 16
    step = 2.0 ** (-8 if t is BF16 else -11)                  # of numbers between 1/2 and 1
    d = -math.log(0.5 + up * step / 2)
    K = torch.zeros(R.pages(T, page), Hkv, page, hd, dtype=t, device="cuda")
    hi = torch.tensor(-d, device="cuda").to(t)
    lo = torch.tensor(-d - float(hi), device="cuda").to(t)
    K[..., 0], K[..., 1] = hi, lo                             # a score of -d to twice the type's digits
    K[0, :, 0] = 0.0
    V = torch.ones_like(K)
    q = torch.zeros(n, H, hd, dtype=t, device="cuda")
    q[..., :2] = 1.0
    table = torch.arange(K.shape[0], dtype=torch.int32, device="cuda")[None]
    out = Ops.PagedAttention(None, q, K, V, table, ints([0, n]), ints([T]), n, scale=1.0)
    off = (out.double() - 1).abs().max().item()
    assert off <= (2 * (T + 16) * 2.0 ** -24 if t is F32 else 0.0), off
