"""Refusals of the paged cache's calls (each before any device is touched), and the plain plan that the GPU tests compare with."""
import pytest
import torch

from seq2seqsharp_b200 import _native as N
from seq2seqsharp_b200.ops import Ops
from tests import paged_reference as R

P = 4096      # stands for a pointer: no call that is refused looks at it


def refused(name, words, *args):
    with pytest.raises(N.TSB200Error, match=words):
        N.call(name, *args)


def plan_args(**k):
    a = dict(dev=0, cached=P, fresh=P, B=2, page=16, table=P, stride=8, width=8, held=P, free=P, count=P, pages=64, lens=P, starts=P, slots=P, positions=P, rows=4, stream=None)
    a.update(k)
    return list(a.values())


@pytest.mark.parametrize("bad,words", [(dict(cached=None), "null"), (dict(slots=None), "null"), (dict(B=0), "sequences"), (dict(B=8193), "8192"), (dict(page=12), "power of two"),
                                       (dict(page=4), "power of two"), (dict(page=512), "power of two"), (dict(width=0), "table"), (dict(stride=7), "table"),
                                       (dict(width=2 ** 30, stride=2 ** 30), "table"), (dict(pages=-1), "pages"), (dict(pages=2 ** 28), "pages"), (dict(rows=-1), "rows")])
def test_plan_refuses(native, bad, words):
    refused("TSB200_PagedPlan", words, *plan_args(**bad))


def rope_args(**k):
    a = dict(dev=0, dtype=N.F16, out=P, o_row=512, o_head=128, q=P, q_row=512, q_head=128, k=P, k_row=256, k_head=128, v=P, v_row=256, v_head=128, qn=None, kn=None, eps=1e-6,
             positions=P, slots=P, rows=3, H=4, Hkv=2, hd=128, style=1, rot=128, base=1e4, K=P, V=P, c_page=4096, c_head=2048, c_tok=128, pages=8, page=16, stream=None)
    a.update(k)
    return list(a.values())


@pytest.mark.parametrize("bad,words", [(dict(dtype=N.I32), "dtype"), (dict(rows=-1), "rows"), (dict(H=0), "heads"), (dict(Hkv=0), "heads"), (dict(hd=12), "head size"), (dict(hd=264), "head size"),
                                       (dict(hd=0), "head size"), (dict(style=3), "style"), (dict(rot=130), "rotated"), (dict(rot=7), "rotated"), (dict(style=2, rot=24), "rotated"),
                                       (dict(rot=0), "rotated"), (dict(base=0.0), "base"), (dict(base=float("inf")), "base"), (dict(page=15), "power of two"),
                                       (dict(pages=-2), "pages"), (dict(q=None), "null"), (dict(slots=None), "null"), (dict(positions=None), "null"), (dict(V=None), "null")])
def test_norm_rope_refuses(native, bad, words):
    refused("TSB200_QKNormRopePaged", words, *rope_args(**bad))


def attention_args(**k):
    a = dict(dev=0, dtype=N.F16, out=P, o_row=512, o_head=128, q=P, q_row=512, q_head=128, K=P, V=P, c_page=4096, c_head=2048, c_tok=128, pages=8, page=16, table=P, stride=4, width=4,
             starts=P, lens=P, B=2, rows=3, most=2, H=4, Hkv=2, hd=128, scale=0.1, window=0, ws=P, ws_bytes=1 << 40, stream=None)
    a.update(k)
    return list(a.values())


@pytest.mark.parametrize("bad,words", [(dict(dtype=N.U8), "dtype"), (dict(B=-1), "sequences"), (dict(rows=-1), "rows"), (dict(most=0), "new"), (dict(Hkv=3), "heads"), (dict(H=0), "heads"),
                                       (dict(hd=100), "head size"), (dict(hd=512), "head size"), (dict(page=24), "power of two"), (dict(width=0), "per sequence"), (dict(stride=3), "per sequence"),
                                       (dict(width=2 ** 28, stride=2 ** 28), "per sequence"), (dict(pages=-1), "pages"), (dict(window=-1), "window"), (dict(rows=2 ** 29), "rows"),
                                       (dict(out=None), "null"), (dict(lens=None), "null"), (dict(q=P + 8), "16 bytes"), (dict(c_tok=132), "16 bytes"), (dict(o_head=129), "16 bytes")])
def test_attention_refuses(native, bad, words):
    refused("TSB200_PagedAttention", words, *attention_args(**bad))


def test_workspace_sizes(native):
    size = native.TSB200_PagedAttentionWorkspaceBytes
    assert 0 < size(N.F16, 32, 8, 128, 1) <= 64 << 20
    assert 0 < size(N.F32, 32, 8, 128, 4096) <= 64 << 20
    assert size(N.F16, 32, 5, 128, 1) == 0 and size(N.F16, 32, 8, 128, 0) == 0


def verify_args(**k):
    a = dict(dev=0, tokens=P, counts=P, p=P, p_row=100, q=P, q_row=100, draft=P, starts=None, u=P, B=2, K=3, V=100, rows=8, stream=None)
    a.update(k)
    return list(a.values())


@pytest.mark.parametrize("bad,words", [(dict(B=-1), "sequences"), (dict(K=-1), "drafts"), (dict(V=0), "words"), (dict(rows=7), "need more"), (dict(p=None), "null"), (dict(draft=None), "null"),
                                       (dict(u=None), "null"), (dict(tokens=None), "null")])
def test_verify_refuses(native, bad, words):
    refused("TSB200_VerifyDraft", words, *verify_args(**bad))


def test_host_tensors_are_refused():
    i = torch.zeros(2, dtype=torch.int32)
    q, c = torch.zeros(2, 4, 64), torch.zeros(3, 2, 16, 64)
    with pytest.raises(N.TSB200Error, match="no CPU fallback"):
        Ops.PagedPlan(i, i, torch.zeros(2, 4, dtype=torch.int32), i, i, i[:1], 16, 4)
    with pytest.raises(N.TSB200Error, match="no CPU fallback"):
        Ops.QKNormRopePaged(None, q, q[:, :2], q[:, :2], None, None, 1e-6, i, i, c, c)
    with pytest.raises(N.TSB200Error, match="no CPU fallback"):
        Ops.PagedAttention(None, q, c, c, torch.zeros(1, 4, dtype=torch.int32), i, i[:1], 2)
    with pytest.raises(N.TSB200Error, match="no CPU fallback"):
        Ops.VerifyDraft(torch.zeros(8, 10), None, torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, 4))


def test_the_plain_plan():
    table, held, free = [[5, -1, -1], [7, 8, -1]], [1, 2], [1, 2, 3]
    lens, starts, slots, positions = R.plan([4, 9], [5, 8], table, held, free, 8, 15)
    assert table == [[5, 3, -1], [7, 8, 2]] and held == [2, 3] and free == [1]
    assert lens == [9, 17] and starts == [0, 5, 13] and positions == [4, 5, 6, 7, 8, 9, 10, 11, 12, 13, 14, 15, 16, -1, -1]
    assert slots[:5] == [44, 45, 46, 47, 24] and slots[12] == 16 and slots[13:] == [-1, -1]
    assert R.plan([4, 9], [0, 0], table, held, free, 8, 0) == ([4, 9], [0, 0, 0], [], [])
    assert table == [[5, -1, -1], [7, 8, -1]] and held == [1, 2] and free == [1, 2, 3]      # taken and given back: as before
