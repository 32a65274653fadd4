"""Python twin of TensorSharp.Ops (TensorSharp/Ops.cs:15-303) dispatching to the B200 backend.

In the reference every op goes Ops.X -> OpRegistry.Invoke(name, args) -> the backend method registered for the
storage type of the arguments (TensorSharp/OpRegistry.cs:46-64).  Here the tensors are torch CUDA tensors (used
only as device buffers with sizes and strides, exactly the fields of TensorSharp.Tensor) and each function calls
the C-ABI entry point that `B200BasicOps` binds for that op name.  `result=None` allocates the write target the way
TensorResultBuilder.GetWriteTarget does (TensorSharp/Core/TensorResultBuilder.cs:7-37).
"""
import ctypes as C

import torch

from . import _native as N

_DT = {torch.float32: N.F32, torch.float16: N.F16, torch.int32: N.I32, torch.float64: N.F64, torch.uint8: N.U8}


def desc(t):
    """TSB200Tensor descriptor of a torch CUDA tensor (a view: sizes, element strides, data pointer)."""
    if t is None:
        return None
    if not t.is_cuda:
        raise N.TSB200Error("the B200 backend only accepts device tensors (no CPU fallback)")
    if t.dim() < 1 or t.dim() > 4:
        raise N.TSB200Error("tensors must have 1..4 dimensions")
    d = N.Tensor()
    d.data = t.data_ptr()
    d.dtype = _DT[t.dtype]
    d.ndim = t.dim()
    for i in range(t.dim()):
        d.sizes[i] = t.size(i)
        d.strides[i] = t.stride(i)
    return d


def _ref(d):
    return C.byref(d) if d is not None else None


def _stream():
    """The caller's current torch stream.  On torch's legacy default stream (handle 0) the library would fall back to
    its own non-blocking stream, which does not order itself after torch's work, so pending torch work is waited for
    first."""
    h = torch.cuda.current_stream().cuda_stream
    if h == 0:
        torch.cuda.synchronize()
        return None
    return C.c_void_p(h)


def _dev(t):
    return t.device.index or 0


def _target(result, like, sizes=None, dtype=None):
    if result is not None:
        return result
    return torch.empty(tuple(sizes if sizes is not None else like.shape), dtype=dtype or like.dtype, device=like.device)


_MODEL_DT = {torch.float32: N.F32, torch.float16: N.F16, torch.bfloat16: N.BF16}
_I32, _F32 = torch.int32, torch.float32


# The calls on the paged cache take five microseconds and less on the device, so their checks look at each tensor once, and say what is wrong only when something is.
def _queue(device):
    """The stream that torch's work on `device` goes to.  Its default stream has the handle 0, which selects the library's own; named as
    cudaStreamLegacy (1) the call takes its place among torch's work there without a wait of the host.  The library keeps it in order with the calls on its
    own stream, where `_stream` puts the other ops."""
    return torch._C._cuda_getCurrentRawStream(device) or 1


def _device(op, t):
    dev = t.get_device()
    if dev < 0:
        raise N.TSB200Error("%s: the B200 backend only accepts device tensors (no CPU fallback)" % op)
    return dev


def _wrong(op, dev, dtype, **tensors):
    """Raises for the first of `tensors` that is not of `dtype` on device `dev`."""
    for name, t in tensors.items():
        if t is not None and (t.dtype is not dtype or t.get_device() != dev):
            raise N.TSB200Error("%s: %s is %s on %s, %s on cuda:%d is wanted" % (op, name, t.dtype, t.device, dtype, dev))


def _plain(op, dev, dtype, name, t, *shape):
    """Address of a contiguous tensor of this shape."""
    if t.dtype is not dtype or t.get_device() != dev or t.shape != shape or not t.is_contiguous():
        raise N.TSB200Error("%s: %s is %s of %s on %s, contiguous %s of %s on cuda:%d is wanted" % (op, name, t.dtype, tuple(t.shape), t.device, dtype, shape, dev))
    return t.data_ptr()


def _heads(op, dev, dtype, name, t, rows, heads, hd):
    """Address, row and head stride of a [rows, heads, hd] tensor.  The stride of a single entry means nothing and is 0."""
    steps = t.stride()   # as a whole: a stride or size by number takes longer than all of them
    if t.dtype is not dtype or t.get_device() != dev or t.shape != (rows, heads, hd) or steps[2] != 1:
        raise N.TSB200Error("%s: %s is %s of %s with strides %s on %s, %s of %s with elements side by side on cuda:%d is wanted" % (
            op, name, t.dtype, tuple(t.shape), steps, t.device, dtype, (rows, heads, hd), dev))
    return t.data_ptr(), steps[0] if rows > 1 else 0, steps[1] if heads > 1 else 0


def _cache(op, dev, dtype, K, V):
    """Shape of a paged cache, its addresses and its page, head and token strides."""
    if K.dtype is not dtype or V.dtype is not dtype or K.get_device() != dev or V.get_device() != dev:
        _wrong(op, dev, dtype, cacheK=K, cacheV=V)
    shape, steps = K.shape, K.stride()
    if len(shape) != 4 or V.shape != shape or steps[3] != 1 or (V.stride() != steps and any(n > 1 and x != y for n, x, y in zip(shape, steps, V.stride()))):
        raise N.TSB200Error("%s: keys %s with strides %s and values %s with strides %s, the same [pages, heads, page, head size] with elements side by side is wanted"
                            % (op, tuple(shape), steps, tuple(V.shape), V.stride()))
    return shape, (K.data_ptr(), V.data_ptr(), steps[0] if shape[0] > 1 else 0, steps[1] if shape[1] > 1 else 0, steps[2])


def _table(op, dev, t, B):
    """Address, row stride and width of a page table."""
    shape, steps = t.shape, t.stride()
    if t.dtype is not _I32 or t.get_device() != dev or len(shape) != 2 or shape[0] != B or steps[1] != 1:
        raise N.TSB200Error("%s: table is %s of %s with strides %s on %s, int32 of [%d, pages of a sequence] with entries side by side on cuda:%d is wanted" % (
            op, t.dtype, tuple(shape), steps, t.device, B, dev))
    width = shape[1]
    return t.data_ptr(), steps[0] if B > 1 else width, width


class Ops:
    """Static facade with the reference's op names."""

    @staticmethod
    def Copy(result, src):
        N.call("TSB200_Copy", _dev(src), _ref(desc(result)), _ref(desc(src)), _stream())
        return result

    @staticmethod
    def Fill(result, value):
        N.call("TSB200_Fill", _dev(result), _ref(desc(result)), float(value), _stream())
        return result

    @staticmethod
    def AsContiguous(src):
        if src.is_contiguous():
            return src
        r = torch.empty(tuple(src.shape), dtype=src.dtype, device=src.device)
        return Ops.Copy(r, src)

    @staticmethod
    def Addmm(result, beta, src, alpha, m1, m2):
        r = _target(result, src)
        N.call("TSB200_Addmm", _dev(src), _ref(desc(r)), float(beta), _ref(desc(src)), float(alpha), _ref(desc(m1)),
               _ref(desc(m2)), _stream())
        return r

    @staticmethod
    def AddmmBatch(result, beta, src, alpha, m1, m2):
        r = _target(result, src)
        N.call("TSB200_AddmmBatch", _dev(src), _ref(desc(r)), float(beta), _ref(desc(src)), float(alpha),
               _ref(desc(m1)), _ref(desc(m2)), _stream())
        return r

    @staticmethod
    def LayerNorm(result, src, alpha, beta, eps=1e-9):
        r = _target(result, src)
        N.call("TSB200_LayerNorm", _dev(src), _ref(desc(r)), _ref(desc(src)), _ref(desc(alpha)), _ref(desc(beta)),
               float(eps), _stream())
        return r

    @staticmethod
    def RMSNorm(result, src, alpha, beta, eps=1e-9):
        r = _target(result, src)
        N.call("TSB200_RMSNorm", _dev(src), _ref(desc(r)), _ref(desc(src)), _ref(desc(alpha)), _ref(desc(beta)),
               float(eps), _stream())
        return r

    @staticmethod
    def RoPE(result, src, seqLen, rowOffset, base=None):
        r = _target(result, src)
        if base is None:
            N.call("TSB200_RoPE", _dev(src), _ref(desc(r)), _ref(desc(src)), int(seqLen), int(rowOffset), _stream())
        else:
            N.call("TSB200_RoPEEx", _dev(src), _ref(desc(r)), _ref(desc(src)), int(seqLen), int(rowOffset),
                   float(base), _stream())
        return r

    @staticmethod
    def Softmax(result, src):
        r = _target(result, src)
        N.call("TSB200_Softmax", _dev(src), _ref(desc(r)), _ref(desc(src)), _stream())
        return r

    @staticmethod
    def IndexSelect(result, src, indice, isAdd=False):
        r = _target(result, src, sizes=(indice.numel(), src.shape[1]))
        N.call("TSB200_IndexSelect", _dev(src), _ref(desc(r)), _ref(desc(src)), _ref(desc(indice)), int(isAdd),
               _stream())
        return r

    @staticmethod
    def Add(result, lhs, rhs):
        r = _target(result, lhs)
        if isinstance(rhs, (int, float)):
            raise N.TSB200Error("Add with a scalar is not on the GPT decode path")
        N.call("TSB200_Add", _dev(lhs), _ref(desc(r)), _ref(desc(lhs)), _ref(desc(rhs)), _stream())
        return r

    @staticmethod
    def Mul(result, lhs, rhs):
        r = _target(result, lhs)
        if isinstance(rhs, (int, float)):
            N.call("TSB200_MulScalar", _dev(lhs), _ref(desc(r)), _ref(desc(lhs)), float(rhs), _stream())
        else:
            N.call("TSB200_Mul", _dev(lhs), _ref(desc(r)), _ref(desc(lhs)), _ref(desc(rhs)), _stream())
        return r

    @staticmethod
    def Div(result, lhs, rhs):
        r = _target(result, lhs)
        N.call("TSB200_DivScalar", _dev(lhs), _ref(desc(r)), _ref(desc(lhs)), float(rhs), _stream())
        return r

    @staticmethod
    def Relu(result, src):
        r = _target(result, src)
        N.call("TSB200_Relu", _dev(src), _ref(desc(r)), _ref(desc(src)), _stream())
        return r

    @staticmethod
    def SiLU(result, src):
        r = _target(result, src)
        N.call("TSB200_SiLU", _dev(src), _ref(desc(r)), _ref(desc(src)), _stream())
        return r

    @staticmethod
    def LeakyReLU(result, src):
        r = _target(result, src)
        N.call("TSB200_LeakyReLU", _dev(src), _ref(desc(r)), _ref(desc(src)), _stream())
        return r

    @staticmethod
    def Float2Half(result, src):
        r = _target(result, src, dtype=torch.float16)
        N.call("TSB200_Float2Half", _dev(src), _ref(desc(r)), _ref(desc(src)), _stream())
        return r

    @staticmethod
    def Half2Float(result, src):
        r = _target(result, src, dtype=torch.float32)
        N.call("TSB200_Half2Float", _dev(src), _ref(desc(r)), _ref(desc(src)), _stream())
        return r

    @staticmethod
    def Argmax(result, src, dimension):
        if dimension < 0:
            dimension += src.dim()
        sizes = list(src.shape)
        sizes[dimension] = 1
        r = _target(result, src, sizes=sizes)
        N.call("TSB200_Argmax", _dev(src), _ref(desc(r)), _ref(desc(src)), int(dimension), _stream())
        return r

    @staticmethod
    def BuildTriMask(result, value, maskedValue):
        N.call("TSB200_BuildTriMask", _dev(result), _ref(desc(result)), float(value), float(maskedValue), _stream())
        return result

    @staticmethod
    def BuildSelfTriMask(result, originalLengths, paddedSeqLen, value, maskedValue):
        N.call("TSB200_BuildSelfTriMask", _dev(result), _ref(desc(result)), _ref(desc(originalLengths)),
               int(paddedSeqLen), float(value), float(maskedValue), _stream())
        return result

    # ---- device replacement of the host loop ComputeGraphTensor.TopPSample (ComputeGraphTensor.cs:2305-2403)
    @staticmethod
    def TopPSample(probs, topP, repeatPenalty, decodedSequences, u):
        """probs [rows, V] float32; decodedSequences: list of id lists (or None); u: [rows] float32 uniform draws."""
        rows, V = probs.shape
        dev = probs.device
        out = torch.empty(rows, dtype=torch.int32, device=dev)
        ws_bytes = N.lib().TSB200_TopPWorkspaceBytes(rows, V)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
        hist = hist_len = None
        stride = 0
        if decodedSequences is not None:
            stride = max(1, max(len(s) for s in decodedSequences))
            h = torch.zeros((rows, stride), dtype=torch.int32)
            for i, s in enumerate(decodedSequences):
                if len(s):
                    h[i, :len(s)] = torch.tensor(s, dtype=torch.int32)
            hist = h.to(dev)
            hist_len = torch.tensor([len(s) for s in decodedSequences], dtype=torch.int32, device=dev)
        u = u.to(device=dev, dtype=torch.float32).contiguous()
        p = probs.contiguous()
        N.call("TSB200_TopPSample", _dev(probs), out.data_ptr(), p.data_ptr(), rows, V, float(topP),
               float(repeatPenalty), hist.data_ptr() if hist is not None else None,
               hist_len.data_ptr() if hist_len is not None else None, stride, u.data_ptr(), ws.data_ptr(), ws_bytes,
               _stream())
        return out

    @staticmethod
    def PhiloxUniform(n, seed, seq_first, step, device="cuda:0"):
        u = torch.empty(n, dtype=torch.float32, device=device)
        N.call("TSB200_PhiloxUniform", u.device.index or 0, u.data_ptr(), n, seed, seq_first, step, _stream())
        return u

    # ---- paged key / value cache (include/tsb200.h: TSB200_PagedPlan and what follows it)
    @staticmethod
    def PagedPlan(cached, fresh, table, held, freePages, freeCount, pageSize, rows):
        """Pages and places for `fresh` [B] new tokens behind `cached` [B] kept ones.  table [B, max_blocks], held [B], freePages [pages] and freeCount [1]
        (all int32) are updated.  Returns lens [B], starts [B + 1], and slots and positions of `rows` rows (-1 behind the granted ones)."""
        op, dev, B, pages = "PagedPlan", _device("PagedPlan", cached), cached.numel(), freePages.numel()
        if rows < 0:
            raise N.TSB200Error("PagedPlan: %d rows" % rows)
        args = (_plain(op, dev, _I32, "cached", cached, B), _plain(op, dev, _I32, "fresh", fresh, B), B, pageSize, *_table(op, dev, table, B), _plain(op, dev, _I32, "held", held, B),
                _plain(op, dev, _I32, "freePages", freePages, pages), _plain(op, dev, _I32, "freeCount", freeCount, 1), pages)
        out = torch.empty(2 * B + 1 + 2 * rows, dtype=_I32, device=cached.device)
        at = out.data_ptr()
        N.check(N.lib().TSB200_PagedPlan(dev, *args, at, at + 4 * B, at + 8 * B + 4, at + 8 * B + 4 + 4 * rows, rows, _queue(dev)), "TSB200_PagedPlan")
        return out.split_with_sizes((B, B + 1, rows, rows))

    @staticmethod
    def QKNormRopePaged(result, q, k, v, qNorm, kNorm, eps, positions, slots, cacheK, cacheV, ropeStyle=1, ropeDims=None, base=500000.0):
        """q [rows, H, hd] normed per head (qNorm [hd] or None) and rotated into `result` (None: a new tensor; q itself is allowed); k, v [rows, Hkv, hd] (k
        normed and rotated) to their slots of cacheK, cacheV [pages, Hkv, page, hd].  Rows of slot -1 are left out.  ropeStyle 0 none, 1 pairs (2i, 2i + 1), 2 pairs
        (i, i + ropeDims / 2).  Strides are free but for the elements of a head."""
        op, dev, dt = "QKNormRopePaged", _device("QKNormRopePaged", q), q.dtype
        code = _MODEL_DT.get(dt)
        if code is None or q.dim() != 3:
            raise N.TSB200Error("QKNormRopePaged: unsupported q, %s of %s" % (dt, tuple(q.shape)))
        rows, H, hd = q.shape
        (pages, Hkv, page, c_hd), c = _cache(op, dev, dt, cacheK, cacheV)
        q3, k3, v3 = _heads(op, dev, dt, "q", q, rows, H, c_hd), _heads(op, dev, dt, "k", k, rows, Hkv, hd), _heads(op, dev, dt, "v", v, rows, Hkv, hd)
        qn = None if qNorm is None else _plain(op, dev, dt, "qNorm", qNorm, hd)
        kn = None if kNorm is None else _plain(op, dev, dt, "kNorm", kNorm, hd)
        at = _plain(op, dev, _I32, "positions", positions, rows), _plain(op, dev, _I32, "slots", slots, rows)
        if result is None:
            result = torch.empty((rows, H, hd), dtype=dt, device=q.device)
        N.check(N.lib().TSB200_QKNormRopePaged(dev, code, *_heads(op, dev, dt, "result", result, rows, H, hd), *q3, *k3, *v3, qn, kn, eps, *at, rows, H, Hkv, hd, ropeStyle,
                                               hd if ropeDims is None else ropeDims, base, *c, pages, page, _queue(dev)), "TSB200_QKNormRopePaged")
        return result

    @staticmethod
    def PagedAttention(result, q, cacheK, cacheV, table, starts, lens, maxNew, scale=None, window=0):
        """Attention of packed new rows q [rows, H, hd] over cacheK, cacheV [pages, Hkv, page, hd]: rows starts[b] .. starts[b + 1] are the last tokens of the lens[b]
        of sequence b, whose pages are table[b]; each sees the keys up to its own (window > 0: the last `window` of them).  maxNew: the most rows of a
        sequence.  scale None: 1 / sqrt(hd).  Rows of no sequence keep what `result` held.  A bounded wait of the kernels that runs out is reported by TSB200_Synchronize."""
        op, dev, dt = "PagedAttention", _device("PagedAttention", q), q.dtype
        code = _MODEL_DT.get(dt)
        if code is None or q.dim() != 3:
            raise N.TSB200Error("PagedAttention: unsupported q, %s of %s" % (dt, tuple(q.shape)))
        rows, H, hd = q.shape
        (pages, Hkv, page, c_hd), c = _cache(op, dev, dt, cacheK, cacheV)
        q3, B = _heads(op, dev, dt, "q", q, rows, H, c_hd), lens.numel()
        args = (*c, pages, page, *_table(op, dev, table, B), _plain(op, dev, _I32, "starts", starts, B + 1), _plain(op, dev, _I32, "lens", lens, B), B, rows, maxNew, H, Hkv, hd,
                hd ** -0.5 if scale is None else scale, window)
        if result is None:
            result = torch.empty((rows, H, hd), dtype=dt, device=q.device)
        L = N.lib()
        ws_bytes = L.TSB200_PagedAttentionWorkspaceBytes(code, H, Hkv, hd, maxNew)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device)
        N.check(L.TSB200_PagedAttention(dev, code, *_heads(op, dev, dt, "result", result, rows, H, hd), *q3, *args, ws.data_ptr(), ws_bytes, _queue(dev)), "TSB200_PagedAttention")
        return result

    @staticmethod
    def VerifyDraft(targetProbs, draftProbs, draftTokens, u, starts=None):
        """targetProbs [rows, V], draftProbs [B * K, V] (None: the drafts were certain), draftTokens [B, K], u [B, K + 1] uniform numbers; rows starts[b] ..
        starts[b + 1] (None: K + 1 each) of sequence b.  Returns tokens [B, K + 1] (accepted drafts, one drawn token, -1 behind) and counts [B]."""
        op, dev = "VerifyDraft", _device("VerifyDraft", targetProbs)
        if targetProbs.dim() != 2 or draftTokens.dim() != 2:
            raise N.TSB200Error("VerifyDraft: targetProbs [rows, words] and draftTokens [sequences, drafts] are wanted")
        (rows, V), (B, K) = targetProbs.shape, draftTokens.shape
        _wrong(op, dev, _F32, targetProbs=targetProbs, draftProbs=draftProbs)
        probs = []
        for name, t, n in (("targetProbs", targetProbs, rows), ("draftProbs", draftProbs, B * K)):
            if t is None:
                probs += None, 0
                continue
            steps = t.stride()
            if t.shape != (n, V) or (V > 1 and steps[1] != 1):
                raise N.TSB200Error("VerifyDraft: %s is %s, [%d, %d] with words side by side is wanted" % (name, tuple(t.shape), n, V))
            probs += t.data_ptr(), steps[0]
        args = (*probs, _plain(op, dev, _I32, "draftTokens", draftTokens, B, K), None if starts is None else _plain(op, dev, _I32, "starts", starts, B + 1),
                _plain(op, dev, _F32, "u", u, B, K + 1), B, K, V, rows)
        tokens, counts = torch.empty((B, K + 1), dtype=_I32, device=u.device), torch.empty(B, dtype=_I32, device=u.device)
        N.check(N.lib().TSB200_VerifyDraft(dev, tokens.data_ptr(), counts.data_ptr(), *args, _queue(dev)), "TSB200_VerifyDraft")
        return tokens, counts
