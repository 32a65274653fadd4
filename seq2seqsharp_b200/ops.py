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


def _queue(device):
    """The stream that torch's work on `device` goes to.  Its default stream has the handle 0, which selects the library's own; named as
    cudaStreamLegacy (1) the call takes its place among torch's work there without a wait of the host."""
    return torch._C._cuda_getCurrentRawStream(device) or 1


def _placed(op, first, **tensors):
    """Index of the device that all `tensors` (name=(tensor, dtype)) and `first` lie on."""
    if not first.is_cuda:
        raise N.TSB200Error("%s: the B200 backend only accepts device tensors (no CPU fallback)" % op)
    dev = first.device
    for name, (t, dtype) in tensors.items():
        if t is None:
            continue
        if t.dtype != dtype:
            raise N.TSB200Error("%s: %s is %s, %s is wanted" % (op, name, t.dtype, dtype))
        if t.device != dev:
            raise N.TSB200Error("%s: %s is on %s, not on %s" % (op, name, t.device, dev))
    return dev.index


def _plain(op, **tensors):
    """Contiguous tensors of the given shapes (name=(tensor, shape))."""
    for name, (t, shape) in tensors.items():
        if t is not None and (tuple(t.shape) != shape or not t.is_contiguous()):
            raise N.TSB200Error("%s: %s is %s, contiguous %s is wanted" % (op, name, tuple(t.shape), shape))


def _steps(t):
    """Strides of all dimensions but the last; those of a single entry mean nothing and are 0."""
    return [st if n > 1 else 0 for n, st in zip(t.shape[:-1], t.stride())]


def _heads(op, name, t, heads, hd):
    """Row and head stride of a [rows, heads, hd] tensor."""
    if t.dim() != 3 or t.shape[1] != heads or t.shape[2] != hd or t.stride(2) != 1:
        raise N.TSB200Error("%s: %s is %s with strides %s, [rows, %d, %d] with elements side by side is wanted" % (op, name, tuple(t.shape), t.stride(), heads, hd))
    return _steps(t)


def _cache(op, cacheK, cacheV):
    """(pages, KV heads, page, head size) and the strides of a paged cache."""
    if cacheK.dim() != 4 or cacheK.shape != cacheV.shape or _steps(cacheK) != _steps(cacheV) or cacheK.stride(3) != 1 or cacheV.stride(3) != 1:
        raise N.TSB200Error("%s: keys %s with strides %s and values %s with strides %s, the same [pages, heads, page, head size] with elements side by side is wanted"
                            % (op, tuple(cacheK.shape), cacheK.stride(), tuple(cacheV.shape), cacheV.stride()))
    return cacheK.shape, _steps(cacheK)


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
        i32 = torch.int32
        dev = _placed("PagedPlan", cached, cached=(cached, i32), fresh=(fresh, i32), table=(table, i32), held=(held, i32), freePages=(freePages, i32), freeCount=(freeCount, i32))
        B = cached.shape[0] if cached.dim() == 1 else -1
        _plain("PagedPlan", cached=(cached, (B,)), fresh=(fresh, (B,)), held=(held, (B,)), freePages=(freePages, (freePages.numel(),)), freeCount=(freeCount, (1,)))
        if table.dim() != 2 or table.shape[0] != B or table.stride(1) != 1:
            raise N.TSB200Error("PagedPlan: table is %s, [%d, pages of a sequence] with entries side by side is wanted" % (tuple(table.shape), B))
        if rows < 0:
            raise N.TSB200Error("PagedPlan: %d rows" % rows)
        lens, starts, slots, positions = torch.empty(2 * B + 1 + 2 * rows, dtype=i32, device=cached.device).split((B, B + 1, rows, rows))
        N.call("TSB200_PagedPlan", dev, cached.data_ptr(), fresh.data_ptr(), B, pageSize, table.data_ptr(), table.stride(0), table.shape[1], held.data_ptr(),
               freePages.data_ptr(), freeCount.data_ptr(), freePages.numel(), lens.data_ptr(), starts.data_ptr(), slots.data_ptr(), positions.data_ptr(), rows, _queue(dev))
        return lens, starts, slots, positions

    @staticmethod
    def QKNormRopePaged(result, q, k, v, qNorm, kNorm, eps, positions, slots, cacheK, cacheV, ropeStyle=1, ropeDims=None, base=500000.0):
        """q [rows, H, hd] normed per head (qNorm [hd] or None) and rotated into `result` (None: a new tensor; q itself is allowed); k, v [rows, Hkv, hd] (k
        normed and rotated) to their slots of cacheK, cacheV [pages, Hkv, page, hd].  Rows of slot -1 are left out.  ropeStyle 0 none, 1 pairs (2i, 2i + 1), 2 pairs
        (i, i + ropeDims / 2).  Strides are free but for the elements of a head."""
        dt, hd = q.dtype, q.shape[-1]
        if dt not in _MODEL_DT:
            raise N.TSB200Error("QKNormRopePaged: unsupported dtype %s" % dt)
        dev = _placed("QKNormRopePaged", q, result=(result, dt), k=(k, dt), v=(v, dt), qNorm=(qNorm, dt), kNorm=(kNorm, dt), positions=(positions, torch.int32),
                      slots=(slots, torch.int32), cacheK=(cacheK, dt), cacheV=(cacheV, dt))
        (pages, Hkv, page, c_hd), c_str = _cache("QKNormRopePaged", cacheK, cacheV)
        rows, H = q.shape[0], q.shape[1] if q.dim() == 3 else 0
        strides = [_heads("QKNormRopePaged", "q", q, H, c_hd)]
        r = torch.empty((rows, H, hd), dtype=dt, device=q.device) if result is None else result
        for name, t, heads in (("k", k, Hkv), ("v", v, Hkv), ("result", r, H)):
            strides.append(_heads("QKNormRopePaged", name, t, heads, c_hd))
            if t.shape[0] != rows:
                raise N.TSB200Error("QKNormRopePaged: %s has %d rows, q %d" % (name, t.shape[0], rows))
        _plain("QKNormRopePaged", qNorm=(qNorm, (hd,)), kNorm=(kNorm, (hd,)), positions=(positions, (rows,)), slots=(slots, (rows,)))
        N.call("TSB200_QKNormRopePaged", dev, _MODEL_DT[dt], r.data_ptr(), *strides[3], q.data_ptr(), *strides[0], k.data_ptr(), *strides[1],
               v.data_ptr(), *strides[2], None if qNorm is None else qNorm.data_ptr(), None if kNorm is None else kNorm.data_ptr(), eps,
               positions.data_ptr(), slots.data_ptr(), rows, H, Hkv, hd, ropeStyle, hd if ropeDims is None else ropeDims, base, cacheK.data_ptr(), cacheV.data_ptr(),
               *c_str, pages, page, _queue(dev))
        return r

    @staticmethod
    def PagedAttention(result, q, cacheK, cacheV, table, starts, lens, maxNew, scale=None, window=0):
        """Attention of packed new rows q [rows, H, hd] over cacheK, cacheV [pages, Hkv, page, hd]: rows starts[b] .. starts[b + 1] are the last tokens of the lens[b]
        of sequence b, whose pages are table[b]; each sees the keys up to its own (window > 0: the last `window` of them).  maxNew: the most rows of a
        sequence.  scale None: 1 / sqrt(hd).  Rows of no sequence keep what `result` held."""
        dt, i32 = q.dtype, torch.int32
        if dt not in _MODEL_DT:
            raise N.TSB200Error("PagedAttention: unsupported dtype %s" % dt)
        dev = _placed("PagedAttention", q, result=(result, dt), cacheK=(cacheK, dt), cacheV=(cacheV, dt), table=(table, i32), starts=(starts, i32), lens=(lens, i32))
        (pages, Hkv, page, hd), c_str = _cache("PagedAttention", cacheK, cacheV)
        rows, H = q.shape[0], q.shape[1] if q.dim() == 3 else 0
        q_str = _heads("PagedAttention", "q", q, H, hd)
        r = torch.empty((rows, H, hd), dtype=dt, device=q.device) if result is None else result
        r_str = _heads("PagedAttention", "result", r, H, hd)
        if r.shape[0] != rows:
            raise N.TSB200Error("PagedAttention: result has %d rows, q %d" % (r.shape[0], rows))
        B = table.shape[0]
        if table.dim() != 2 or table.stride(1) != 1:
            raise N.TSB200Error("PagedAttention: table is %s, [sequences, pages of a sequence] with entries side by side is wanted" % (tuple(table.shape),))
        _plain("PagedAttention", starts=(starts, (B + 1,)), lens=(lens, (B,)))
        ws_bytes = N.lib().TSB200_PagedAttentionWorkspaceBytes(_MODEL_DT[dt], H, Hkv, hd, maxNew)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device)
        N.call("TSB200_PagedAttention", dev, _MODEL_DT[dt], r.data_ptr(), *r_str, q.data_ptr(), *q_str, cacheK.data_ptr(), cacheV.data_ptr(), *c_str, pages, page, table.data_ptr(), table.stride(0), table.shape[1], starts.data_ptr(), lens.data_ptr(), B, rows, maxNew, H, Hkv, hd,
               hd ** -0.5 if scale is None else scale, window, ws.data_ptr(), ws_bytes, _queue(dev))
        return r

    @staticmethod
    def VerifyDraft(targetProbs, draftProbs, draftTokens, u, starts=None):
        """targetProbs [rows, V], draftProbs [B * K, V] (None: the drafts were certain), draftTokens [B, K], u [B, K + 1] uniform numbers; rows starts[b] ..
        starts[b + 1] (None: K + 1 each) of sequence b.  Returns tokens [B, K + 1] (accepted drafts, one drawn token, -1 behind) and counts [B]."""
        f32, i32 = torch.float32, torch.int32
        dev = _placed("VerifyDraft", targetProbs, targetProbs=(targetProbs, f32), draftProbs=(draftProbs, f32), draftTokens=(draftTokens, i32), u=(u, f32), starts=(starts, i32))
        if targetProbs.dim() != 2 or draftTokens.dim() != 2:
            raise N.TSB200Error("VerifyDraft: targetProbs [rows, words] and draftTokens [sequences, drafts] are wanted")
        (rows, V), (B, K) = targetProbs.shape, draftTokens.shape
        _plain("VerifyDraft", draftTokens=(draftTokens, (B, K)), u=(u, (B, K + 1)), starts=(starts, (B + 1,)))
        for name, t, n in (("targetProbs", targetProbs, rows), ("draftProbs", draftProbs, B * K)):
            if t is not None and (tuple(t.shape) != (n, V) or (V > 1 and t.stride(1) != 1)):
                raise N.TSB200Error("VerifyDraft: %s is %s, [%d, %d] with words side by side is wanted" % (name, tuple(t.shape), n, V))
        tokens, counts = torch.empty((B, K + 1), dtype=i32, device=u.device), torch.empty(B, dtype=i32, device=u.device)
        N.call("TSB200_VerifyDraft", dev, tokens.data_ptr(), counts.data_ptr(), targetProbs.data_ptr(), targetProbs.stride(0), None if draftProbs is None else draftProbs.data_ptr(),
               0 if draftProbs is None else draftProbs.stride(0), draftTokens.data_ptr(), None if starts is None else starts.data_ptr(), u.data_ptr(), B, K, V, rows, _queue(dev))
        return tokens, counts
