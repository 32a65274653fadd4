"""The paged cache's numbers where a systematic error would hide behind random ones: weights that all round the same way, angles near whole half turns."""
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


# ---------------------------------------------------------------------------------------------------------------------------- angles
@pytest.mark.parametrize("style,rot", [(1, 64), (2, 64), (1, 18), (2, 16)])
def test_angles_of_fp32_rows(cuda, style, rot):
    """(1, 0) turned by an angle is its cosine and sine, each off by two units in the last place at most, also next to whole half turns where one of
    them is nearly 0 (an angle rounded to fp32 before its sine is taken is off by up to pi 2^-25, whatever the sine's size).  2^-36: the 64-bit angle
    itself, 4095 times a rate off by a few 2^-53."""
    rows, hd = 4096, 64
    q = torch.zeros(rows, 2, hd, device="cuda")
    i = torch.arange(rot // 2, device="cuda")
    lo, hi = (2 * i, 2 * i + 1) if style == 1 else (i, i + rot // 2)
    q[..., lo] = 1.0
    kv = torch.zeros(rows, 1, hd, device="cuda")
    K, V = (torch.zeros(rows // 16, 1, 16, hd, device="cuda") for _ in range(2))
    pos = torch.arange(rows, dtype=torch.int32, device="cuda")
    got = Ops.QKNormRopePaged(None, q, kv, kv, None, None, 0.0, pos, pos, K, V, ropeStyle=style, ropeDims=rot, base=10000.0)
    angle = pos.double()[:, None, None] * torch.exp(-2.0 * i.double() / rot * math.log(10000.0))
    for want, x in ((angle.cos(), got[..., lo]), (angle.sin(), got[..., hi])):
        assert ((x.double() - want).abs() <= 2 * 2.0 ** -23 * want.abs() + 2.0 ** -36).all()
