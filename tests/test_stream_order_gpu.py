"""Calls made one after the other on torch's default stream run in that order, whichever of the two streams behind it they go to: the ops of the reference's list
wait for the device and go to the library's own stream, the calls on the paged cache to cudaStreamLegacy.  Nothing is waited for in between."""
import pytest
import torch

from seq2seqsharp_b200 import _native as N
from seq2seqsharp_b200.ops import Ops

pytestmark = pytest.mark.gpu
F16 = torch.float16


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def test_softmax_before_the_check_of_drafts(cuda):
    B, K, V = 64, 7, 50257
    g = torch.Generator(device="cuda").manual_seed(1)
    draft = torch.randint(0, V, (B, K), generator=g, device="cuda", dtype=torch.int32)
    u = torch.rand(B, K + 1, generator=g, device="cuda")
    for i in range(20):
        logits = torch.randn(B * (K + 1), V, generator=g, device="cuda") * 3
        p = torch.full_like(logits, 0.5)                      # what a call that comes too early would read
        got = Ops.VerifyDraft(Ops.Softmax(p, logits), None, draft, u)
        torch.cuda.synchronize()
        want = Ops.VerifyDraft(p, None, draft, u)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_uniform_numbers_before_the_check_of_drafts(cuda):
    B, K, V = 1024, 3, 64
    p = torch.softmax(torch.randn(B * (K + 1), V, device="cuda"), -1)
    draft = torch.randint(0, V, (B, K), device="cuda", dtype=torch.int32)
    big = torch.randn(4096, 4096, device="cuda")
    for i in range(20):
        Ops.Mul(big, big, 1.0)                                # in front of it on the same stream
        u = Ops.PhiloxUniform(B * (K + 1), 7, 100 * i, i).view(B, K + 1)
        got = Ops.VerifyDraft(p, None, draft, u)
        torch.cuda.synchronize()
        want = Ops.VerifyDraft(p, None, draft, u)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def problem(n, T):
    g = torch.Generator(device="cuda").manual_seed(2)
    K, V = (torch.randn(T // 16, 8, 16, 64, generator=g, device="cuda").to(F16) for _ in range(2))
    return torch.randn(n, 16 * 64, generator=g, device="cuda"), K, V, torch.arange(T // 16, dtype=torch.int32, device="cuda")[None], ints([0, n]), ints([T])


def test_ops_before_attention_and_behind_it(cuda):
    n, T = 2048, 4096
    x, K, V, table, starts, lens = problem(n, T)
    gamma = torch.ones(1, 16 * 64, device="cuda")
    for i in range(10):
        y = torch.zeros(n, 16 * 64, dtype=F16, device="cuda")
        h = Ops.Float2Half(y, Ops.RMSNorm(None, x + i, gamma, None))
        out = Ops.PagedAttention(torch.zeros(n, 16, 64, dtype=F16, device="cuda"), h.view(n, 16, 64), K, V, table, starts, lens, n)
        back = Ops.Half2Float(None, out.view(n, -1))
        torch.cuda.synchronize()
        want = Ops.PagedAttention(None, y.view(n, 16, 64), K, V, table, starts, lens, n)
        assert torch.equal(out, want) and torch.equal(back, want.float().view(n, -1))


def test_calls_of_the_library_without_a_stream(cuda):
    """The same through the C entries, where null names the library's own stream: it is in order with the calls on cudaStreamLegacy on both sides."""
    n, T = 2048, 8192
    x, K, V, table, starts, lens = problem(n, T)
    q0 = x.to(F16).view(n, 16, 64)
    want = Ops.PagedAttention(None, q0, K, V, table, starts, lens, n).cpu()
    for _ in range(10):
        q, out = torch.zeros_like(q0), torch.zeros_like(q0)
        host = torch.empty(q0.shape, dtype=F16)
        torch.cuda.synchronize()
        N.call("TSB200_MemcpyD2D", 0, q.data_ptr(), q0.data_ptr(), q0.numel() * 2, None)
        Ops.PagedAttention(out, q, K, V, table, starts, lens, n)
        N.call("TSB200_MemcpyD2H", 0, host.data_ptr(), out.data_ptr(), out.numel() * 2, None)
        assert torch.equal(host, want)
        # and the host's wait for the one has seen the other
        Ops.PagedAttention(out, q, K, V, table, starts, lens, n)
        e = torch.cuda.Event()
        e.record()
        N.call("TSB200_Synchronize", 0, None)
        assert e.query()


def test_a_call_without_a_stream_while_another_stream_is_captured(cuda):
    # both streams are in use; the order between them is no part of a capture that goes on beside
    n, T = 64, 512
    x, K, V, table, starts, lens = problem(n, T)
    q = x.to(F16).view(n, 16, 64)
    want = Ops.PagedAttention(None, q, K, V, table, starts, lens, n)
    a, b, out = torch.randn(1000, device="cuda"), torch.zeros(1000, device="cuda"), torch.zeros_like(q)
    N.call("TSB200_MemcpyD2D", 0, b.data_ptr(), a.data_ptr(), 4000, None)
    torch.cuda.synchronize()
    b.zero_()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            Ops.PagedAttention(out, q, K, V, table, starts, lens, n)
            N.call("TSB200_MemcpyD2D", 0, b.data_ptr(), a.data_ptr(), 4000, None)
        N.call("TSB200_Synchronize", 0, None)
        assert torch.equal(a, b)                              # it ran at once
        g.replay()
        s.synchronize()
    assert torch.equal(out, want)
