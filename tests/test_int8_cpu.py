"""Refusals of the linears in 8-bit integers and of the log probabilities, each before any device is touched."""
import pytest
import torch

from seq2seqsharp_b200 import _native as N
from seq2seqsharp_b200.ops import Ops

P = 4096      # stands for a pointer: no call that is refused looks at it


def refused(name, words, args, bad):
    args.update(bad)
    with pytest.raises(N.TSB200Error, match=words):
        N.call(name, *args.values())


@pytest.mark.parametrize("bad,words", [(dict(dtype=N.I32), "dtype"), (dict(rows=-1), "rows"), (dict(rows=2 ** 31), "rows"), (dict(d=0), "elements"), (dict(d=2 ** 30 + 1), "elements"),
                                       (dict(q=None), "null"), (dict(scale=None), "null"), (dict(x=None), "null"), (dict(gamma=None), "null"), (dict(eps=-1.0), "eps"),
                                       (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"), (dict(residual=None), "go together"), (dict(h=None), "go together"),
                                       (dict(q_row=63), "overlap"), (dict(h_row=10), "overlap"), (dict(x=P + 1), "between"), (dict(residual=P + 1), "between"), (dict(gamma=P + 1), "between"),
                                       (dict(scale=P + 2), "between")])
def test_norm_refuses(native, bad, words):
    refused("TSB200_RMSNormInt8", words, dict(dev=0, dtype=N.F16, q=P, q_row=64, scale=P, h=P, h_row=64, x=P, x_row=64, residual=P, r_row=64, gamma=P, eps=1e-6, rows=3, d=64, s=None), bad)


@pytest.mark.parametrize("bad,words", [(dict(dtype=N.U8), "dtype"), (dict(rows=-3), "rows"), (dict(d=-1), "elements"), (dict(q=None), "null"), (dict(src=None), "null"),
                                       (dict(act=7), "activation"), (dict(act=-2), "activation"), (dict(q_row=1), "overlap"), (dict(gate=P + 1), "between"), (dict(src=P + 1), "between")])
def test_rows_refuse(native, bad, words):
    refused("TSB200_RowsInt8", words, dict(dev=0, dtype=N.BF16, q=P, q_row=64, scale=P, src=P, src_row=64, gate=P, g_row=64, act=N.ACT_SILU, rows=3, d=64, s=None), bad)


@pytest.mark.parametrize("bad,words", [(dict(dtype=N.U8), "dtype"), (dict(rows=-1), "rows"), (dict(rows=2 ** 31 - 5), "rows"), (dict(K=0), "bytes"), (dict(K=2 ** 17), "32 bits"), (dict(N=0), "channels"),
                                       (dict(y=None), "null"), (dict(q=None), "null"), (dict(sq=None), "null"), (dict(w=None), "null"), (dict(sw=None), "null"), (dict(y_row=31), "overlap"),
                                       (dict(q_row=-64), "negative"), (dict(w_row=-64), "negative"), (dict(y=P + 1), "between"), (dict(bias=P + 1), "between"), (dict(sw=P + 1), "between")])
def test_linear_refuses(native, bad, words):
    refused("TSB200_LinearInt8", words, dict(dev=0, dtype=N.F16, y=P, y_row=32, q=P, q_row=64, sq=P, w=P, w_row=64, sw=P, bias=P, rows=3, K=64, N=32, s=None), bad)


@pytest.mark.parametrize("bad,words", [(dict(dtype=N.I32), "dtype"), (dict(rows=-1), "rows"), (dict(V=0), "words"), (dict(top=-1), "alternatives"), (dict(top=33), "alternatives"),
                                       (dict(V=4), "alternatives"), (dict(x=None), "null"), (dict(tokens=None), "null"), (dict(lp=None), "null"), (dict(ranks=None), "null"), (dict(ids=None), "null"),
                                       (dict(x=P + 1), "between"), (dict(tokens=P + 2), "between")])
def test_log_probs_refuse(native, bad, words):
    refused("TSB200_TokenLogProbs", words, dict(dev=0, dtype=N.F16, lp=P, ent=P, ranks=P, ids=P, best=P, top=5, x=P, x_row=100, tokens=P, rows=3, V=100, s=None), bad)


def test_nothing_of_no_rows(native):
    N.call("TSB200_RMSNormInt8", 0, N.F16, None, 0, None, None, 0, None, 0, None, 0, None, 1e-6, 0, 64, None)
    N.call("TSB200_RowsInt8", 0, N.F16, None, 0, None, None, 0, None, 0, N.ACT_NONE, 0, 64, None)
    N.call("TSB200_LinearInt8", 0, N.F16, None, 0, None, 0, None, None, 0, None, None, 0, 64, 32, None)
    N.call("TSB200_TokenLogProbs", 0, N.F16, None, None, None, None, None, 5, None, 0, None, 0, 100, None)


def test_host_tensors_are_refused(native):
    x, g, q, s = torch.zeros(2, 16), torch.ones(16), torch.zeros(2, 16, dtype=torch.int8), torch.ones(2)
    for call in (lambda: Ops.RMSNormInt8(None, x, None, g), lambda: Ops.RowsInt8(None, x), lambda: Ops.LinearInt8(None, q, s, q, s), lambda: Ops.TokenLogProbs(x, s.int())):
        with pytest.raises(N.TSB200Error, match="no CPU fallback"):
            call()
