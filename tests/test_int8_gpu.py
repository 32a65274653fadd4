"""Linears in 8-bit integers against plain restatements in 64 bits: the norm and the activations that give bytes, the product, and a run of them together.

Tolerances count roundings, u = 2^-24 for one of fp32.  A byte is rint(x) of x = 127 v / max|v|; v, max|v| and 127 / max|v| are rounded once each, so x is off by at most 3 u 127 and
the byte within 0.5 + 381 u of the exact x.  Of silu and sigmoid the exponential is off by (2 + 1.18 |x|) 2^-23 and the quotient by 2 2^-23, for inputs up to 12 below 20 2^-23 of
the value, in v and in max|v|: 127 * 40 * 2^-23 < 1e-3; erf in gelu adds at most 2^-22 of the input, which is at most 4 max|v| here: 127 * 2^-20 < 1e-3.  The scale of a
norm has at most 40 roundings of the sum of squares (chains of 32 and a tree of 10; d / 1024 more in rows beyond 32768), halved by the root, and eight others.
An output of the product is round_t(acc s + b): the sum, s = sq sw and the result are rounded to fp32 once each: 3 u (|acc s| + |b|), and half a step of t."""
import numpy as np
import pytest
import torch

from seq2seqsharp_b200 import _native as N
from seq2seqsharp_b200.ops import Ops

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = 2.0 ** -24


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, t=F32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(t)


def check_bytes(q, scale, v, factor, slack, scale_roundings):
    """q, scale of the exact rows v (64 bits): scale = max|v| factor / 127."""
    top = v.abs().amax(1)
    x = v / torch.where(top > 0, top, torch.ones_like(top))[:, None] * 127
    assert q.dtype == torch.int8 and q.shape == v.shape
    assert (q.double() - x).abs().max().item() <= 0.5 + 381 * U + slack
    want = top * factor / 127
    assert ((scale.double() - want).abs() <= scale_roundings * U * want).all()


# ---------------------------------------------------------------------------------------------------------------------------- norm
def norm_exact(x, residual, gamma, eps):
    h = x if residual is None else (x.double() + residual.double()).to(x.dtype)   # (the 64-bit sum of two 16-bit numbers is exact, of two fp32 ones rounded twice)
    if residual is not None and x.dtype is F32:
        h = x + residual
    d = h.double()
    return h, d * gamma.double(), 1 / torch.sqrt((d ** 2).mean(1) + eps)


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("rows,d", [(1, 1), (1, 4096), (3, 7), (9, 64), (5, 66), (300, 256), (40, 1001), (17, 2048), (33, 4098), (2, 8200), (7, 12288), (2, 16385), (3, 20000), (1, 32768), (2, 32769),
                                    (1, 70001)])
@pytest.mark.parametrize("residual", [True, False])
def test_norm(cuda, t, rows, d, residual):
    g = gen(rows * d)
    x, r = randn(g, rows, d, t=t), randn(g, rows, d, t=t, scale=3.0) if residual else None
    gamma = (1 + 0.3 * torch.randn(d, generator=g, device="cuda")).to(t)
    q, scale, h = Ops.RMSNormInt8(None, x, r, gamma, 1e-5)
    want, v, root = norm_exact(x, r, gamma, 1e-5)
    assert torch.equal(h, want) and (residual or h is x)
    assert rows == 1 or q.stride(0) % 16 == 0
    check_bytes(q, scale, v, root, 0.0, 28 + d / 2048)


@pytest.mark.parametrize("t", [F16, BF16])
@pytest.mark.parametrize("d", [1024, 2040, 2048, 3016, 4096, 4104, 8192, 8200, 12288, 12296, 16384])
@pytest.mark.parametrize("two", [True, False])
def test_many_rows(cuda, t, d, two):
    """Enough rows for CTAs that walk over several; the sum in place, one row of zeros and one that is not finite among them."""
    g, rows = gen(d), 1203
    x, r = randn(g, rows, d, t=t), randn(g, rows, d, t=t, scale=3.0) if two else None
    x[700] = 0
    x[1202, d - 1] = float("nan")
    if two:
        r[700] = 0
    gamma = (1 + 0.3 * torch.randn(d, generator=g, device="cuda")).to(t)
    fine = torch.arange(rows, device="cuda") != 1202
    want, v, root = norm_exact(x, r, gamma, 1e-5)
    a = x.clone()
    q, scale, h = Ops.RMSNormInt8(None, a, r, gamma, 1e-5, sum=a if two else None)
    assert torch.equal(h[fine], want[fine]) and h is a and scale[700] == 0 and scale[1202].isnan() and (q[[700, 1202]] == 0).all()
    check_bytes(q[fine], scale[fine], v[fine], root[fine], 0.0, 28 + d / 2048)
    q, scale = Ops.RowsInt8(None, x, r, N.ACT_LEAKYRELU)
    v = ACTS[N.ACT_LEAKYRELU](x.double()) * (r.double() if two else 1)
    check_bytes(q[fine], scale[fine], v[fine], 1.0, 127 * U, 5)
    assert scale[700] == 0 and scale[1202].isnan() and (q[[700, 1202]] == 0).all()
    N.call("TSB200_Synchronize", 0, 1)   # no wait has run out


@pytest.mark.parametrize("t", [F32, F16, BF16])
def test_norm_strides_and_places(cuda, t):
    """Rows cut out of wider ones, at odd places; the sum written over either operand; bytes in rows of the caller's."""
    g = gen(5)
    for rows, d, off, width in ((6, 96, 0, 160), (6, 96, 1, 161), (5, 50, 2, 64), (1, 33, 3, 40), (70, 4096, 8, 4200)):
        wide = randn(g, rows, width, t=t)
        x, gamma = wide[:, off: off + d], randn(g, d + 1, t=t)[1:].clone()
        r = randn(g, rows, d, t=t)
        out = torch.full((rows, d + 5), 99, dtype=torch.int8, device="cuda")
        for where in ("new", "residual", "src"):
            xs, rs = (wide.clone()[:, off: off + d], r.clone())
            s = {"new": None, "residual": rs, "src": xs}[where]
            want, v, root = norm_exact(x, r, gamma, 1e-6)
            q, scale, h = Ops.RMSNormInt8(out[:, 2: 2 + d], xs, rs, gamma, 1e-6, sum=s)
            assert torch.equal(h, want) and (s is None or h is s)
            assert torch.equal(rs, want if where == "residual" else r)
            check_bytes(q, scale, v, root, 0.0, 28)
            assert (out[:, :2] == 99).all() and (out[:, 2 + d:] == 99).all()
    same = randn(g, 1, 64, t=t).expand(4, 64)   # one row read four times
    q, scale, _ = Ops.RMSNormInt8(None, same, None, torch.ones(64, dtype=t, device="cuda"))
    assert (q == q[0]).all() and (scale == scale[0]).all()


def test_bytes_do_not_depend_on_the_other_rows(cuda):
    g = gen(6)
    x, r, gamma = randn(g, 700, 1536, t=BF16), randn(g, 700, 1536, t=BF16), randn(g, 1536, t=BF16)
    q, scale, h = Ops.RMSNormInt8(None, x, r, gamma)
    for i in (0, 311, 699):
        q1, s1, h1 = Ops.RMSNormInt8(None, x[i: i + 1], r[i: i + 1], gamma)
        assert torch.equal(q1, q[i: i + 1]) and torch.equal(s1, scale[i: i + 1]) and torch.equal(h1, h[i: i + 1])


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("d", [24, 1000, 5000, 40000])
def test_rows_of_zeros_and_rows_that_are_not_finite(cuda, t, d):
    g = gen(7)
    x = randn(g, 6, d, t=t)
    x[1] = 0
    x[2, d // 2] = float("inf")
    x[3, d - 1] = float("nan")
    x[4, 0] = -float("inf")
    gamma = torch.ones(d, dtype=t, device="cuda")
    for q, scale in (Ops.RMSNormInt8(None, x, None, gamma)[:2], Ops.RowsInt8(None, x)):
        assert scale[1] == 0 and scale[[2, 3, 4]].isnan().all() and (q[1:5] == 0).all()
        assert scale[[0, 5]].isfinite().all() and (q[[0, 5]].abs().amax(1) == 127).all()
    # a masked row whose gate is zero: infinity times zero is no number either
    q, scale = Ops.RowsInt8(None, x[2:3], torch.zeros_like(x[2:3]))
    assert scale.isnan().all() and (q == 0).all()


@pytest.mark.parametrize("t,k", [(F32, 40), (F32, 120), (F32, 140), (BF16, 120), (F16, 20)])
def test_nearly_zero_rows(cuda, t, k):
    """Rows scaled by a power of two have the same bytes as long as the type holds them exactly."""
    x = (torch.arange(1, 65, device="cuda").float() - 20).repeat(2, 1)
    small = x * 2.0 ** -k
    if t is F16:
        x = small = (x.round() * 2.0 ** -k)
    q, scale = Ops.RowsInt8(None, small.to(t))
    want = (x.double() / x.double().abs().amax(1, keepdim=True) * 127).round()
    assert torch.equal(q.double(), want)
    exact = small.to(t).double().abs().amax(1) / 127
    assert ((scale.double() - exact).abs() <= exact * U + 2.0 ** -150).all()


# ---------------------------------------------------------------------------------------------------------------------------- activations
ACTS = {N.ACT_NONE: lambda a: a, N.ACT_RELU: lambda a: a.clamp(min=0), N.ACT_SILU: lambda a: a * torch.sigmoid(a), N.ACT_SWIGLU: lambda a: a * torch.sigmoid(a),
        N.ACT_LEAKYRELU: lambda a: torch.where(a < 0, 0.01 * a, a), N.ACT_GELU: lambda a: a * torch.special.ndtr(a), N.ACT_GLU_NOACT: lambda a: a, N.ACT_SIGMOID: torch.sigmoid}


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("act", sorted(ACTS))
@pytest.mark.parametrize("rows,d,gate", [(1, 1, True), (1, 11008, True), (50, 999, True), (9, 130, False), (300, 512, True), (2, 40001, True), (3, 17000, False)])
def test_rows(cuda, t, act, rows, d, gate):
    g = gen(rows + d)
    wide = randn(g, rows, 2 * d, t=t, scale=1.5).clamp_(-12, 12)
    wide[:, 0] = 2.0    # so that a row's largest value is not small beside its inputs
    wide[:, d] = 3.0
    a, b = wide[:, :d], wide[:, d:] if gate else None
    q, scale = Ops.RowsInt8(None, a, b, act)
    v = ACTS[act](a.double())
    if gate:
        v = v * b.double()
    soft = act in (N.ACT_SILU, N.ACT_SWIGLU, N.ACT_SIGMOID, N.ACT_GELU)
    check_bytes(q, scale, v, 1.0, 1e-3 if soft else 127 * U, 100 if soft else 5)


def test_rows_that_are_all_negative(cuda):
    q, scale = Ops.RowsInt8(None, -torch.rand(3, 100, device="cuda"), None, N.ACT_RELU)
    assert (q == 0).all() and (scale == 0).all()


# ---------------------------------------------------------------------------------------------------------------------------- product
def bytes_of(g, rows, cols, pad=True):
    wide = torch.randint(-128, 128, (rows, -(-cols // 16) * 16 if pad else cols), generator=g, device="cuda", dtype=torch.int8)
    return wide[:, :cols]


def check_linear(y, q, sq, w, sw, bias, t):
    prod = (q.double() @ w.double().t()) * (sq.double()[:, None] * sw.double())
    want = prod if bias is None else prod + bias.double()
    room = 3.01 * U * (prod.abs() + (0 if bias is None else bias.double().abs())) + torch.finfo(t).eps / 2 * want.abs() * 1.001 + (2.0 ** -25 if t is F16 else 0)
    assert y.dtype is t and ((y.double() - want).abs() <= room).all()


def scales(g, n, k=1.0):
    return (0.5 + torch.rand(n, generator=g, device="cuda")) * k


SIZES = [(1, 1, 1), (1, 64, 128), (1, 4096, 22016), (2, 129, 130), (5, 1000, 257), (16, 300, 4096), (17, 2048, 2050), (32, 128, 100), (33, 127, 1000), (64, 11008, 520), (65, 640, 384), (100, 5000, 1030),
         (128, 96, 4100), (129, 256, 128), (203, 1000, 2047), (256, 130, 256), (257, 2048, 1000), (700, 513, 3000), (1025, 64, 50257), (2048, 4096, 1536), (300, 33, 3)]


@pytest.mark.parametrize("M,K,n", SIZES)
@pytest.mark.parametrize("t", [F32, F16, BF16])
def test_linear(cuda, M, K, n, t):
    g = gen(M + K + n)
    q, w = bytes_of(g, M, K), bytes_of(g, n, K)
    sq, sw = scales(g, M, 0.02), scales(g, n, 0.5 / (74 * K ** 0.5))
    for bias in (None, randn(g, n, t=t)):
        check_linear(Ops.LinearInt8(None, q, sq, w, sw, bias, dtype=t), q, sq, w, sw, bias, t)
    N.call("TSB200_Synchronize", 0, 1)   # no wait has run out


@pytest.mark.parametrize("M,K,n", [(1, 100, 200), (3, 65, 64), (70, 130, 129), (200, 1000, 333)])
@pytest.mark.parametrize("t", [F32, BF16])
def test_linear_of_rows_that_start_anywhere(cuda, M, K, n, t):
    g = gen(M * K)
    sq, sw = scales(g, M, 0.02), scales(g, n, 0.5 / (74 * K ** 0.5))
    wide_q, wide_w = bytes_of(g, M, K + 30, pad=False), bytes_of(g, n, K + 47, pad=False)
    for q, w in ((wide_q[:, 3: 3 + K], wide_w[:, :K]), (bytes_of(g, M, K), wide_w[:, 5: 5 + K]), (bytes_of(g, M, K, pad=False), bytes_of(g, n, K, pad=False)),
                 (bytes_of(g, 1, K).expand(M, K), bytes_of(g, n, K))):
        check_linear(Ops.LinearInt8(None, q, sq, w, sw, dtype=t), q, sq, w, sw, None, t)


@pytest.mark.parametrize("M", [3, 40, 100, 300])
@pytest.mark.parametrize("t", [F32, F16])
def test_linear_writes_its_rows_only(cuda, M, t):
    """Outputs at odd places in wider rows; what lies around them stays."""
    g = gen(M)
    for n, off, width in ((260, 1, 270), (256, 4, 264), (127, 0, 127), (130, 2, 200)):
        K = 320
        q, w, sq, sw = bytes_of(g, M, K), bytes_of(g, n, K), scales(g, M, 0.02), scales(g, n + 1, 0.01)[1:].clone()
        wide = torch.full((M + 2, width), 7.0, dtype=t, device="cuda")
        y = wide[1: M + 1, off: off + n]
        assert Ops.LinearInt8(y, q, sq, w, sw) is y
        check_linear(y, q, sq, w, sw, None, t)
        y.fill_(7.0)
        assert (wide == 7.0).all()


@pytest.mark.parametrize("M", [1, 20, 50, 128, 400])
def test_linear_sums_are_exact(cuda, M):
    """The longest rows, of the largest bytes, on every kernel: sums near 2^31."""
    K, n = 2 ** 17 - 1, 136
    q, w = (torch.full((r, 2 ** 17), -128, dtype=torch.int8, device="cuda")[:, :K] for r in (M, n))
    w[1::2] = 127
    one = torch.ones
    y = Ops.LinearInt8(None, q, one(M, device="cuda"), w, one(n, device="cuda"), dtype=F32)
    assert (y[:, ::2] == float(np.float32(128 * 128 * K))).all() and (y[:, 1::2] == float(np.float32(-128 * 127 * K))).all()


@pytest.mark.parametrize("M", [2, 30, 60, 100, 300])
def test_a_row_without_a_scale_stays_without_one(cuda, M):
    g = gen(M)
    q, w, sq, sw = bytes_of(g, M, 256), bytes_of(g, 384, 256), scales(g, M), scales(g, 384)
    sq[1] = float("nan")
    sw[5] = 0
    y = Ops.LinearInt8(None, q, sq, w, sw, dtype=F32)
    assert y[1].isnan().all() and y[0].isfinite().all() and (y[0, 5] == 0) and y[2:].isfinite().all()


def test_linear_refuses_what_does_not_fit(cuda):
    g = gen(1)
    q, w, s4, s8 = bytes_of(g, 4, 64), bytes_of(g, 8, 64), scales(g, 4), scales(g, 8)
    for call, words in ((lambda: Ops.LinearInt8(None, q, s4, bytes_of(g, 8, 65), s8), "weight"), (lambda: Ops.LinearInt8(None, q, s8, w, s8), "srcScale"),
                        (lambda: Ops.LinearInt8(None, q, s4, w, s4), "weightScale"), (lambda: Ops.LinearInt8(None, q.float(), s4, w, s8), "src"),
                        (lambda: Ops.LinearInt8(None, q, s4, w, s8, torch.zeros(8, device="cuda")), "bias"), (lambda: Ops.LinearInt8(None, q, s4, w, s8, dtype=torch.float64), "unsupported"),
                        (lambda: Ops.LinearInt8(torch.zeros(1, 8, device="cuda").expand(4, 8), q, s4, w, s8), "overlap"),
                        (lambda: Ops.LinearInt8(None, q, s4, w.t().contiguous().t(), s8), "weight"), (lambda: Ops.RowsInt8(torch.zeros(4, 64, dtype=torch.uint8, device="cuda"), q.float()), "result"),
                        (lambda: Ops.RowsInt8(None, q), "unsupported"), (lambda: Ops.RowsInt8(None, q.float(), q.half()), "gate"),
                        (lambda: Ops.RMSNormInt8(None, q.float(), None, s8), "gamma"), (lambda: Ops.RMSNormInt8(None, q.float(), None, torch.ones(64, device="cuda"), sum=q.float()), "without a residual"),
                        (lambda: Ops.RMSNormInt8(None, q.float(), q.float()[:3], torch.ones(64, device="cuda")), "residual")):
        with pytest.raises(N.TSB200Error, match=words):
            call()


@pytest.mark.parametrize("rows", [0, 1, 5])
def test_empty_and_short_calls(cuda, rows):
    q, s, h = Ops.RMSNormInt8(None, torch.ones(rows, 48, device="cuda", dtype=F16), torch.ones(rows, 48, device="cuda", dtype=F16), torch.ones(48, device="cuda", dtype=F16))
    assert q.shape == (rows, 48) and s.shape == (rows,) and h.shape == (rows, 48) and (q == 127).all() and (h == 2).all()
    y = Ops.LinearInt8(None, q, s, torch.ones(7, 48, dtype=torch.int8, device="cuda"), torch.ones(7, device="cuda"))
    assert y.shape == (rows, 7) and (y == 48).all()


@pytest.mark.parametrize("M,K,n", [(1, 65536, 8192), (48, 65536, 8192), (120, 65536, 8192), (600, 65536, 8192)])
def test_linears_end_in_order_when_a_wait_runs_out(cuda, M, K, n):
    """One poll per wait (an environment variable, hence a process of its own): every warp gives up in its own place, copies and products in flight end before a CTA leaves its shared
    memory and TMEM, the synchronisation fails once, and the device stays usable."""
    import os
    import subprocess
    import sys
    code = """
import torch
from seq2seqsharp_b200 import _native as N
from seq2seqsharp_b200.ops import Ops
M, K, n = %d, %d, %d
q, w = (torch.randint(-127, 128, (r, K), device="cuda", dtype=torch.int8) for r in (M, n))
sq, sw = torch.ones(M, device="cuda"), torch.ones(n, device="cuda")
for i in range(8):
    y = Ops.LinearInt8(None, q, sq, w, sw)
try:
    N.call("TSB200_Synchronize", 0, 1)
    print("silent")
except N.TSB200Error as e:
    print(e)
N.call("TSB200_Synchronize", 0, 1)
print("usable", torch.equal(w.flip(1).flip(1), w), float(torch.ones(4, device="cuda").sum()))
""" % (M, K, n)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                       env=dict(os.environ, TSB200_WAIT_LIMIT="1"))
    assert r.returncode == 0, r.stderr
    assert "gave up waiting" in r.stdout and "usable True 4.0" in r.stdout, r.stdout


def test_rows_end_in_order_when_a_wait_runs_out(cuda):
    """The same for rows that come through a ring of copies.  A copy is short enough for the one poll to see it at times: then nothing is reported, and the outputs are right."""
    import os
    import subprocess
    import sys
    code = """
import torch
from seq2seqsharp_b200 import _native as N
from seq2seqsharp_b200.ops import Ops
x, r = (torch.randn(6000, 16384, device="cuda", dtype=torch.float16) for _ in range(2))
gain = torch.ones(16384, device="cuda", dtype=torch.float16)
got = [Ops.RMSNormInt8(None, x, r, gain) for i in range(4)]
try:
    N.call("TSB200_Synchronize", 0, 1)
    print("right", all(torch.equal(h, x + r) for _, _, h in got))
except N.TSB200Error as e:
    print(e)
N.call("TSB200_Synchronize", 0, 1)
print("usable", torch.equal(x.flip(1).flip(1), x), float(torch.ones(4, device="cuda").sum()))
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                       env=dict(os.environ, TSB200_WAIT_LIMIT="1"))
    assert r.returncode == 0, r.stderr
    assert ("gave up waiting" in r.stdout or "right True" in r.stdout) and "usable True 4.0" in r.stdout, r.stdout


# ---------------------------------------------------------------------------------------------------------------------------- together
class Block:
    """The feed-forward block of a model and its LM head in bytes: norm, gate | up, gated product, down, norm, logits, log probabilities."""

    def __init__(self, d, F, V, t, seed=3):
        g = gen(seed)
        self.d, self.F, self.t = d, F, t
        full = dict(gate_up=randn(g, 2 * F, d, scale=d ** -0.5, t=t), down=randn(g, d, F, scale=F ** -0.5, t=t), head=randn(g, V, d, scale=2 * d ** -0.5, t=t))
        self.full, self.w = full, {k: Ops.RowsInt8(None, v) for k, v in full.items()}
        self.g1, self.g2 = ((1 + 0.1 * torch.randn(d, generator=g, device="cuda")).to(t) for _ in range(2))

    def __call__(self, x, stream, tokens, top):
        F, t = self.F, self.t
        q, s, stream = Ops.RMSNormInt8(None, x, stream, self.g1)
        wide = Ops.LinearInt8(None, q, s, *self.w["gate_up"], dtype=t)
        q, s = Ops.RowsInt8(None, wide[:, :F], wide[:, F:], N.ACT_SILU)
        x = Ops.LinearInt8(None, q, s, *self.w["down"], dtype=t)
        q, s, stream = Ops.RMSNormInt8(None, x, stream, self.g2)
        logits = Ops.LinearInt8(None, q, s, *self.w["head"], dtype=F32)
        return (stream, logits, *Ops.TokenLogProbs(logits, tokens, top))

    def exact(self, x, stream, tokens):
        """With the weights and rows as they are, in 64 bits."""
        w = {k: v.double() for k, v in self.full.items()}
        norm = lambda h, g: h / torch.sqrt((h ** 2).mean(1, keepdim=True) + 1e-6) * g.double()  # noqa: E731
        h = x.double() + stream.double()
        wide = norm(h, self.g1) @ w["gate_up"].t()
        a, b = wide[:, : self.F], wide[:, self.F:]
        h = h + (a * torch.sigmoid(a) * b) @ w["down"].t()
        logits = norm(h, self.g2) @ w["head"].t()
        return logits, torch.log_softmax(logits, 1).gather(1, tokens.long()[:, None])[:, 0]


@pytest.mark.parametrize("t", [F16, BF16, F32])
@pytest.mark.parametrize("rows", [1, 24, 90, 300])
def test_a_block_in_bytes(cuda, t, rows):
    """A byte is off by half a step of max / 127; with d independent such errors the logits (about 2) are off by about 1 % of their size: held to 4 %."""
    d, F, V = 512, 1376, 2003
    block, g = Block(d, F, V, t), gen(rows)
    x, stream = randn(g, rows, d, t=t), randn(g, rows, d, t=t)
    tokens = torch.randint(0, V, (rows,), generator=g, device="cuda").int()
    got = block(x, stream, tokens, 5)
    logits, lp = block.exact(x, stream, tokens)
    assert ((got[1].double() - logits).square().mean().sqrt() <= 0.04 * logits.square().mean().sqrt()).item()
    assert ((got[2].double() - lp).square().mean().sqrt() <= 0.04 * 2 * 3).item()   # a logit's and the row's, sigma 2, with room of 3
    assert torch.equal(got[5], got[1].topk(5, 1).indices.int())


@pytest.mark.parametrize("rows", [2, 200])
def test_captured_block_with_other_inputs(cuda, rows):
    """Captured once, replayed with other inputs; beside it an eager call on a stream of its own."""
    d, F, V, t = 512, 1408, 1000, BF16
    block, g = Block(d, F, V, t), gen(rows)
    x, stream, tokens = randn(g, rows, d, t=t), randn(g, rows, d, t=t), torch.randint(0, V, (rows,), generator=g, device="cuda").int()
    want = [block(x, stream, tokens, 3)]
    other = randn(g, rows, d, t=t), randn(g, rows, d, t=t), torch.randint(0, V, (rows,), generator=g, device="cuda").int()
    want.append(block(*other, 3))
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        out = block(x, stream, tokens, 3)
    for k in (0, 1, 0):
        if k:
            keep = [v.clone() for v in (x, stream, tokens)]
            for dst, src in zip((x, stream, tokens), other):
                dst.copy_(src)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            beside = block(*other, 3)
        graph.replay()
        torch.cuda.synchronize()
        for a, b, c in zip(out, want[k], beside):
            assert torch.equal(a, b)
        for c, b in zip(beside, want[1]):
            assert torch.equal(c, b)
        if k:
            for dst, src in zip((x, stream, tokens), keep):
                dst.copy_(src)


def test_first_calls_of_a_process_may_be_captured(cuda):
    """What the library asks the driver for once (entry points, attributes of kernels) can be asked for while a stream is captured."""
    import os
    import subprocess
    import sys
    code = """
import torch
from seq2seqsharp_b200 import _native as N
from seq2seqsharp_b200.ops import Ops
g, out = torch.cuda.CUDAGraph(), {}
x = torch.randn(700, 4096, device="cuda", dtype=torch.float16)
gain, w, sw = torch.ones(4096, device="cuda", dtype=torch.float16), torch.randint(-9, 9, (512, 4096), device="cuda", dtype=torch.int8), torch.ones(512, device="cuda")
tokens = torch.zeros(700, device="cuda", dtype=torch.int32)
def run(rows):
    q, s, h = Ops.RMSNormInt8(None, x[:rows], x[:rows], gain)
    y = Ops.LinearInt8(None, q, s, w, sw, dtype=torch.float32)
    return (q, s, h, y, *Ops.TokenLogProbs(y, tokens[:rows], 3))
torch.cuda.synchronize()
with torch.cuda.graph(g):
    for rows in (1, 20, 50, 700):
        out[rows] = run(rows)
g.replay()
torch.cuda.synchronize()
print(all(torch.equal(a, b) for rows in out for a, b in zip(out[rows], run(rows))))
N.call("TSB200_Synchronize", 0, 1)
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert r.returncode == 0 and r.stdout.strip() == "True", r.stdout + r.stderr


@pytest.mark.parametrize("M", [1, 40, 300])
def test_two_linears_at_once(cuda, M):
    """Two streams, no order between them: the calls share nothing."""
    g = gen(M)
    sets = [(bytes_of(g, M, 2048), scales(g, M), bytes_of(g, 4096, 2048), scales(g, 4096)) for _ in range(2)]
    want = [Ops.LinearInt8(None, *s, dtype=F32) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(Ops.LinearInt8(None, *sets[k], dtype=F32))
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(v, want[k]) for v in got[k])
    N.call("TSB200_Synchronize", 0, 1)


@pytest.mark.parametrize("t", [F32, F16])
def test_norm_without_eps(cuda, t):
    x = torch.zeros(3, 40, device="cuda", dtype=t)
    x[1] = 2
    q, scale, _ = Ops.RMSNormInt8(None, x, None, torch.ones(40, device="cuda", dtype=t), 0.0)
    assert scale.tolist() == [0.0, float(np.float32(1) / np.float32(127)), 0.0] and (q[1] == 127).all() and (q[[0, 2]] == 0).all()
