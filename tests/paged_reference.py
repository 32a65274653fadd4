"""The operators of the paged cache restated plainly: the plan sequence by sequence, the rest in 64 bits."""
import math

import torch


def pages(tokens, page):
    return -(-tokens // page)


def plan(cached, fresh, table, held, free, page, rows):
    """Lists in, lists out; `free`: the free pages, the next one to be taken last.  table, held and free are changed."""
    width, given, out, left, stop_pages, stop_rows = len(table[0]), [], [], rows, False, False
    stock, taken = list(free), 0
    for b, (old, new) in enumerate(zip(cached, fresh)):
        fits = old >= 0 and new >= 0 and old + new <= width * page
        if not fits:
            out.append(0)
            continue
        need = max(0, pages(old + new, page) - held[b]) if new > 0 else 0
        if need and (stop_pages or need > len(stock) - taken):
            stop_pages, new = True, 0
        if new and (stop_rows or new > left):
            stop_rows, new = True, 0
        need = need if new else 0
        left -= new
        for j in range(need):
            taken += 1
            table[b][held[b] + j] = stock[-taken]
        keep = pages(old + new, page) if new else min(held[b], pages(old, page))
        for j in range(keep, held[b]):
            given.append(table[b][j])
            table[b][j] = -1
        held[b] = keep
        out.append(new)
    free[:] = stock[: len(stock) - taken] + given[::-1]
    starts, slots, positions = [0], [], []
    for b, new in enumerate(out):
        starts.append(starts[-1] + new)
        for i in range(new):
            pos = cached[b] + i
            positions.append(pos)
            slots.append(table[b][pos // page] * page + pos % page)
    lens = [old + new for old, new in zip(cached, out)]
    behind = [-1] * (rows - starts[-1])
    return lens, starts, slots + behind, positions + behind


def norm_rope(x, w, eps, positions, style, rot, base):
    """x [rows, heads, hd] in 64 bits -> (result, sum of the magnitudes that meet in an element)."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x ** 2).mean(-1, keepdim=True) + eps) * w.double()
    y, met = x.clone(), x.abs()
    if style:
        i = torch.arange(rot // 2, device=x.device)
        lo, hi = (2 * i, 2 * i + 1) if style == 1 else (i, i + rot // 2)
        angle = positions.double()[:, None, None] * torch.exp(-2.0 * i.double() / rot * math.log(base))
        a, b, c, s = x[..., lo], x[..., hi], angle.cos(), angle.sin()
        y[..., lo], y[..., hi] = a * c - b * s, b * c + a * s
        met[..., lo] = met[..., hi] = a.abs() + b.abs()
    return y, met


def attention(q, K, V, table, starts, lens, scale, window=0):
    """(out, sum of weight * |value|, largest sum of |q k| * scale) per row and head, in 64 bits; rows of no sequence NaN."""
    rows, H, hd = q.shape
    count, Hkv, page, _ = K.shape
    G = H // Hkv
    out, mass = (torch.full((rows, H, hd), float("nan"), dtype=torch.float64, device=q.device) for _ in range(2))
    size = torch.zeros(rows, H, 1, dtype=torch.float64, device=q.device)
    for b in range(len(lens)):
        r0, n, T = starts[b], starts[b + 1] - starts[b], min(lens[b], table.shape[1] * page)
        if n == 0:
            continue
        j = torch.arange(T, device=q.device)
        entry = table[b].long()[j // page]
        there = (entry >= 0) & (entry < count)
        entry = entry.clamp(0, count - 1)
        pos = lens[b] - n + torch.arange(n, device=q.device)
        sees = there & (j <= pos[:, None])
        if window:
            sees &= j > pos[:, None] - window
        used = sees.any(0)
        for h in range(Hkv):
            k, v = (torch.where(used[:, None], x[entry, h, j % page].double(), 0.0) for x in (K, V))
            qq = q[r0: r0 + n, h * G:(h + 1) * G].double()
            s = torch.einsum("igd,td->igt", qq, k) * scale
            s = s.masked_fill(~sees[:, None], -math.inf)
            w = torch.softmax(s, -1).nan_to_num(0.0) if T else s
            if T:
                w = torch.where(sees.any(1)[:, None, None], torch.softmax(torch.where(sees.any(1)[:, None, None], s, 0.0), -1), 0.0)
                size[r0: r0 + n, h * G:(h + 1) * G, 0] = (torch.einsum("igd,td->igt", qq.abs(), k.abs()) * abs(scale)).masked_fill(~sees[:, None], 0.0).amax(-1)
            out[r0: r0 + n, h * G:(h + 1) * G] = torch.einsum("igt,td->igd", w, v)
            mass[r0: r0 + n, h * G:(h + 1) * G] = torch.einsum("igt,td->igd", w, v.abs())
    return out, mass, size


def verify(p, q, draft, u, starts, K):
    """Plain lists of rows (64-bit numpy arrays) -> tokens, counts."""
    import numpy as np
    tokens, counts = [], []
    for b in range(len(draft)):
        n = min(starts[b + 1] - starts[b], K + 1)
        if n <= 0:
            tokens.append([-1] * (K + 1))
            counts.append(0)
            continue
        V, got = p.shape[1], []
        weights = None
        for i in range(n - 1):
            x, row = draft[b][i], p[starts[b] + i]
            inside = 0 <= x < V
            if inside and u[b][i] * (q[b * K + i][x] if q is not None else 1.0) < row[x]:
                got.append(x)
                continue
            less = q[b * K + i] if q is not None else np.eye(1, V, x if inside else V)[0]
            weights = np.maximum(row - less, 0.0)
            break
        if weights is None or not weights.sum() > 0:
            weights = np.maximum(p[starts[b] + len(got)], 0.0)
        sums = np.cumsum(weights)
        if sums[-1] > 0:
            got.append(int(min(np.searchsorted(sums, u[b][K] * sums[-1], side="right"), np.flatnonzero(weights)[-1])))
        else:
            got.append(-1)
        tokens.append(got + [-1] * (K + 1 - len(got)))
        counts.append(len(got))
    return tokens, counts
