"""The norm in bytes for rows whose squares, or whose products with the gain, leave fp32 downwards: with an eps of 0 or next to it the result is of ordinary size.

Tolerances as in test_int8_gpu.py: a byte within 0.5 + 381 u of the exact quotient, a scale within 28 u + d / 2048 u; a scale below 2^-126 has steps of 2^-149 and is rounded once, to half of one.
With an eps of 2^-100 or more the product v of a row's element and its gain is one of fp32, with steps of 2^-149 below 2^-126: v and max|v| are off by 2^-150 more each.  127 v / max|v| is then off by
127 2^-150 / max|v| for v and as much again for max|v| (|v| <= max|v|), the scale max|v| root / 127 by 2^-150 root / 127, where root = 1 / sqrt(mean + eps) is at most 2^50.  A max|v| of less than
2^-150 may be 0 there, with bytes of 0: off by at most 127, which is below 127 2^-150 / max|v|."""
import numpy as np
import pytest
import torch

from seq2seqsharp_b200.ops import Ops
from tests.test_int8_gpu import BF16, F16, F32, U, gen, norm_exact, randn

pytestmark = pytest.mark.gpu
SIZES = [1.0, 0.0, 1e-10, 2.0 ** -49, 2.0 ** -50, 2.0 ** -51, 1e-18, 1e-20, 1e-21, 1e-22, 1e-23, 1e-25, 1e-30, 1e-36, 1e-38, 1e-40, 1e-43]


def check(t, rows, d, residual, gain, eps, seed=1):
    g = gen(seed)
    size = torch.tensor([SIZES[i % len(SIZES)] for i in range(rows)], device="cuda")[:, None]
    if t is F16:
        size = size.clamp(min=3e-8) * (size > 0)
    x, r = (randn(g, rows, d) * size).to(t), (randn(g, rows, d) * size).to(t) if residual else None
    gamma = ((1 + 0.3 * torch.randn(d, generator=g, device="cuda")) * gain).to(t)
    eps = float(np.float32(eps))
    h, v, root = norm_exact(x, r, gamma, eps)
    q, scale, got = Ops.RMSNormInt8(None, x, r, gamma, eps)
    assert torch.equal(got, h)
    top = v.abs().amax(1)
    some = top > 0
    quotient = v / torch.where(some, top, torch.ones_like(top))[:, None] * 127
    step = 2.0 ** -150 if eps >= 2.0 ** -100 else 0.0
    lost = torch.where(some, 2 * 127 * step / top.clamp(min=1e-300), torch.zeros_like(top))
    assert ((q.double() - quotient).abs() <= 0.5 + 381 * U + lost[:, None]).all()
    root = torch.where(some, root, torch.zeros_like(root))   # (of a row of zeros without an eps there is none)
    want = top * root / 127
    assert ((scale.double() - want).abs() <= (28 + d / 2048) * U * want + 2.0 ** -150 + step * root / 127).all()
    again = Ops.RMSNormInt8(None, x, r, gamma, eps)
    assert torch.equal(again[0], q) and torch.equal(again[1], scale)
    return q, scale


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("rows,d", [(17, 1), (34, 7), (34, 64), (34, 66), (34, 1001), (34, 4096), (17, 12000), (17, 20000), (17, 40001), (700, 1024), (700, 4096), (650, 8192), (600, 16384)])
@pytest.mark.parametrize("residual", [True, False])
def test_small_rows(cuda, t, rows, d, residual):
    for eps in (0.0, 1e-44, 1e-38, 1e-30, 1e-6):
        check(t, rows, d, residual, 1.0, eps)


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("d", [60, 999, 4096])
@pytest.mark.parametrize("gain", [1e10, 1e-10, 1e-24])
def test_small_rows_with_a_gain(cuda, t, d, gain):
    """Squares that vanish under products that do not, and products near the end of fp32 under squares that are none."""
    for eps in (0.0, 1e-40):
        check(t, 34, d, False, gain, eps)


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("d", [64, 4096])
def test_one_element(cuda, t, d):
    """The smallest numbers of the type, alone in their rows: the root makes sqrt(d) of each."""
    x = torch.zeros(8, d, device="cuda", dtype=t)
    for i, e in enumerate((-149, -140, -133, -127, -126, -100, -75, -60)):
        x[i, 5 * i] = 2.0 ** max(e, -133 if t is BF16 else -149)
    q, scale, _ = Ops.RMSNormInt8(None, x, None, torch.ones(d, device="cuda", dtype=t), 0.0)
    want = float(np.sqrt(d) / 127)
    assert ((scale.double() - want).abs() <= 28 * U * want).all() and torch.equal(q, (x != 0).to(torch.int8) * 127)


def test_bytes_do_not_depend_on_the_kernel(cuda):
    """The same rows alone, a few of them, and many."""
    g, d = gen(3), 4096
    size = 2.0 ** torch.linspace(-140, 0, 700, device="cuda")[:, None]
    x, gamma = (randn(g, 700, d) * size).to(BF16), (1 + 0.3 * torch.randn(d, generator=g, device="cuda")).to(BF16)
    for eps in (0.0, 1e-38):
        q = Ops.RMSNormInt8(None, x, None, gamma, eps)[0]
        for i in (0, 3, 60, 150, 199, 200, 201, 202, 350, 699):
            assert torch.equal(Ops.RMSNormInt8(None, x[i: i + 1], None, gamma, eps)[0], q[i: i + 1])
        assert torch.equal(Ops.RMSNormInt8(None, x[190: 260], None, gamma, eps)[0], q[190: 260])


@pytest.mark.parametrize("rows,d", [(5, 96), (9, 4096), (3, 40000), (700, 4096), (700, 8192)])
@pytest.mark.parametrize("place", ["src", "residual"])
def test_in_place_in_a_graph_and_between_other_rows(cuda, rows, d, place):
    """The sum over an operand, rows of the caller's that lie apart, captured; small rows between ordinary ones."""
    g = gen(rows + d)
    size = torch.ones(rows, 1, device="cuda")
    size[1::2] = 1e-24
    x0, r0 = (randn(g, rows, d) * size).to(BF16), (randn(g, rows, d) * size).to(BF16)
    gamma = (1 + 0.3 * torch.randn(d, generator=g, device="cuda")).to(BF16)
    want = Ops.RMSNormInt8(None, x0, r0, gamma, 0.0)
    x, r = x0.clone(), r0.clone()
    wide = torch.full((rows, d + 32), 99, dtype=torch.int8, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, scale, h = Ops.RMSNormInt8(wide[:, 16: 16 + d], x, r, gamma, 0.0, sum=x if place == "src" else r)
    for _ in range(2):
        x.copy_(x0)
        r.copy_(r0)
        graph.replay()
        assert torch.equal(q, want[0]) and torch.equal(scale, want[1]) and torch.equal(h, want[2])
        assert (wide[:, :16] == 99).all() and (wide[:, 16 + d:] == 99).all()
    assert (scale > 1e-3).all() and (q.abs().amax(1) == 127).all()
