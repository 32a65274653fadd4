"""The paged key / value cache against plain restatements in 64 bits: the plan, norm / rotation / append, attention of ragged chunks, the check of drafted
tokens, and a run of them together.

Tolerances count roundings (half a step, h = eps / 2 of the type): an attention output is rounded once, and so is each weight in the 16-bit kernels,
which changes the sum of weight * |value| (`mass`) by at most h of it; a score's fp32 sum is off by at most (hd + 3) 2^-24 of the sum of |q k|, a weight
by twice that; exponentials, their arguments and the sums add less than 2^-19 of the mass; fp16 weights below 2^-14 of the largest are off by up to 2^-25 of it."""
import numpy as np
import pytest
import torch

from seq2seqsharp_b200 import _native as N
from seq2seqsharp_b200.ops import Ops
from tests import paged_reference as R

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
H_OF = {t: torch.finfo(t).eps / 2 for t in (F32, F16, BF16)}


def ints(v, dev="cuda"):
    return torch.tensor(v, dtype=torch.int32, device=dev)


# ---------------------------------------------------------------------------------------------------------------------------- plan
class Pool:
    """The state of a plan on the device and in plain lists."""

    def __init__(self, B, width, page, pages, stride=None, seed=0):
        rng = np.random.default_rng(seed)
        self.page, self.table, self.held = page, [[-1] * width for _ in range(B)], [0] * B
        self.free = [int(x) for x in rng.permutation(pages)]
        wide = torch.full((B, stride or width), -7, dtype=torch.int32, device="cuda")
        self.d_wide, self.d_table = wide, wide[:, :width]
        self.d_table.fill_(-1)
        self.d_held, self.d_free, self.d_count = ints(self.held), ints(self.free), ints([pages])

    def step(self, cached, fresh, rows):
        got = Ops.PagedPlan(ints(cached), ints(fresh), self.d_table, self.d_held, self.d_free, self.d_count, self.page, rows)
        want = R.plan(cached, fresh, self.table, self.held, self.free, self.page, rows)
        for g, w in zip(got, want):
            assert g.tolist() == w
        assert self.d_table.tolist() == self.table and self.d_held.tolist() == self.held
        assert self.d_count.item() == len(self.free) and self.d_free[: len(self.free)].tolist() == self.free
        assert (self.d_wide[:, self.d_table.shape[1]:] == -7).all()
        return want


@pytest.mark.parametrize("B,width,page,pages", [(1, 40, 16, 64), (7, 9, 8, 40), (33, 70, 16, 700), (64, 3, 256, 100), (1024, 12, 32, 4000), (1025, 5, 16, 3000), (2100, 4, 8, 9000),
                                                (8192, 3, 8, 20000)])
def test_plan_follows_requests(cuda, B, width, page, pages):
    rng = np.random.default_rng(B)
    pool = Pool(B, width, page, pages, stride=width + 3, seed=B)
    lens = [0] * B
    for step in range(6):
        fresh = [int(x) for x in np.where(rng.random(B) < 0.2, 0, rng.integers(1, (30, 6, 60, 2, 9, 5)[step], B))]
        rows = (sum(fresh) + 5, sum(fresh), sum(fresh) // 2, 3, 4 * B, 0)[step]     # all, exactly, half, hardly any, any, none
        lens = pool.step(lens, fresh, rows)[0]
        # some end, some lose their newest tokens
        lens = [0 if r < 0.1 else max(0, n - int(k)) for r, n, k in zip(rng.random(B), lens, rng.integers(0, 9, B))]
        if step % 2:
            pool.step(lens, [0] * B, 2)


def test_plan_without_pages(cuda):
    pool = Pool(4, 8, 16, 5)
    pool.step([0, 0, 0, 0], [40, 60, 10, 0], 200)        # 3 + 4 + 1 pages wanted of 5: the second gets nothing, nor does the third
    assert pool.held == [3, 0, 0, 0]
    pool.step([40, 0, 0, 0], [8, 0, 16, 16], 200)        # room in its last page; 2 left
    assert pool.held == [3, 0, 1, 1] and not pool.free
    pool.step([48, 0, 16, 16], [1, 1, 0, 0], 200)        # nothing is left
    pool.step([0, 0, 16, 16], [0, 1, 0, 0], 200)         # what goes back in a call is not taken in it
    assert pool.held == [0, 0, 1, 1]
    pool.step([0, 0, 16, 16], [1, 2, 3, 0], 200)
    assert pool.held == [1, 1, 2, 1] and not pool.free   # now it is


def test_plan_with_bad_counts(cuda):
    pool = Pool(5, 4, 8, 20)
    pool.step([0] * 5, [9, 9, 9, 9, 9], 100)
    pool.step([9, -1, 9, 30, 9], [1, 5, -2, 3, 24], 100)   # negative or too long: their pages stay, the others are served
    pool.step([9, 9, 9, 2 ** 31 - 1, 9], [2 ** 31 - 1, 0, 1, 2 ** 31 - 1, 0], 100)
    pool.step([0] * 5, [0] * 5, 0)
    assert len(pool.free) == 20


def test_plan_lengths_in_place(cuda):
    pool = Pool(3, 6, 16, 20)
    lens = ints([0, 0, 0])
    for fresh in ([5, 20, 0], [40, 1, 17]):
        new = torch.empty(3 + 4 + 100, dtype=torch.int32, device="cuda")
        before = lens.tolist()
        N.call("TSB200_PagedPlan", 0, lens.data_ptr(), ints(fresh).data_ptr(), 3, 16, pool.d_table.data_ptr(), pool.d_table.stride(0), 6, pool.d_held.data_ptr(), pool.d_free.data_ptr(),
               pool.d_count.data_ptr(), 20, lens.data_ptr(), new.data_ptr(), new[4:].data_ptr(), new[54:].data_ptr(), 50, 1)
        want = R.plan(before, fresh, pool.table, pool.held, pool.free, 16, 50)
        assert lens.tolist() == want[0] and new[:4].tolist() == want[1] and new[4:54].tolist() == want[2] and new[54:104].tolist() == want[3]


# ---------------------------------------------------------------------------------------------------------------------------- norm, rotation, append
def cache(pages, Hkv, page, hd, t, layout="heads", fill=None, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    make = lambda *s: torch.randn(*s, generator=g, device="cuda").to(t) if fill is None else torch.full(s, fill, dtype=t, device="cuda")  # noqa: E731
    if layout == "tokens":                                  # a page's tokens outside of its heads
        return [make(pages, page, Hkv, hd).transpose(1, 2) for _ in range(2)]
    if layout == "both":                                    # keys and values of a page side by side
        both = make(pages, 2, Hkv, page, hd)
        return [both[:, 0], both[:, 1]]
    return [make(pages, Hkv, page, hd) for _ in range(2)]


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("rows,H,Hkv,hd,page,style,rot,norm,layout", [
    (1, 4, 1, 64, 16, 1, 64, True, "heads"), (5, 32, 8, 128, 16, 2, 128, True, "tokens"), (67, 3, 3, 80, 8, 2, 32, True, "both"), (300, 8, 2, 96, 32, 1, 50, False, "heads"),
    (9, 2, 1, 256, 256, 2, 256, True, "tokens"), (13, 6, 2, 8, 8, 1, 8, True, "heads"), (40, 5, 5, 72, 64, 0, None, True, "both"), (1000, 12, 4, 64, 128, 2, 16, True, "heads"),
    (2, 1, 1, 16, 8, 2, 16, False, "heads"), (33, 7, 1, 200, 16, 1, 2, True, "tokens")])
def test_norm_rope_append(cuda, t, rows, H, Hkv, hd, page, style, rot, norm, layout):
    g = torch.Generator(device="cuda").manual_seed(rows)
    rot = hd if rot is None else rot
    qkv = (torch.randn(rows, (H + 2 * Hkv) * hd + 24, generator=g, device="cuda") * 2).to(t)      # rows that end in something else
    q, k, v = (x.unflatten(1, (-1, hd)) for x in qkv[:, :(H + 2 * Hkv) * hd].split([H * hd, Hkv * hd, Hkv * hd], 1))
    wq, wk = [(1 + 0.3 * torch.randn(hd, generator=g, device="cuda")).to(t) for _ in range(2)] if norm else (None, None)
    pages = R.pages(rows, page) + 3
    K, V = cache(pages, Hkv, page, hd, t, layout)
    K0, V0 = K.clone(), V.clone()
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:rows].to(torch.int32)
    positions = torch.randint(0, 200000, (rows,), generator=g, device="cuda", dtype=torch.int32)
    skipped = torch.rand(rows, generator=g, device="cuda") < 0.2
    if rows > 8:
        slots[0], slots[3], slots[4] = pages * page, -5, 2 ** 31 - 1                # not places of the cache
        skipped[[0, 3, 4]] = True
    live = torch.where(skipped, -1, slots)
    slots = torch.where(skipped & (slots >= 0) & (slots < pages * page), -1, slots)
    out = torch.full((rows, H, hd), 9.0, dtype=t, device="cuda")
    r = Ops.QKNormRopePaged(out, q, k, v, wq, wk, 1e-6, positions, slots, K, V, ropeStyle=style, ropeDims=rot, base=10000.0)
    assert r is out
    at = live >= 0
    h, slip = H_OF[t], (hd / 2 + 16) * 2.0 ** -24          # a norm's sum of squares, its root, and the rotation in fp32
    for x, w, got in ((q, wq, out), (k, wk, None)):
        want, met = R.norm_rope(x, w, 1e-6, positions, style, rot, 10000.0)
        if got is None:
            got = K.transpose(1, 2).reshape(-1, Hkv, hd)[live[at].long()]
            want, met = want[at], met[at]
        else:
            assert (got[~at] == 9.0).all()
            got, want, met = got[at], want[at], met[at]
        assert ((got.double() - want).abs() <= h * want.abs() + slip * met + 2.0 ** -25).all()   # 2^-25: fp16 results below its smallest normal number
    flat = lambda c: c.transpose(1, 2).reshape(-1, Hkv, hd)  # noqa: E731
    assert torch.equal(flat(V)[live[at].long()], v[at])
    untouched = torch.ones(pages * page, dtype=torch.bool, device="cuda")
    untouched[live[at].long()] = False
    assert torch.equal(flat(K)[untouched], flat(K0)[untouched]) and torch.equal(flat(V)[untouched], flat(V0)[untouched])


def test_norm_rope_in_place_and_unaligned(cuda):
    g = torch.Generator(device="cuda").manual_seed(3)
    rows, H, Hkv, hd = 11, 4, 2, 64
    flat = torch.randn(rows * (H + 2 * Hkv) * hd + 1, generator=g, device="cuda").to(F16)
    for off in (0, 1):
        x = flat[off: off + rows * (H + 2 * Hkv) * hd].clone() if off == 0 else flat.clone()[1:]
        q, k, v = x.view(rows, H + 2 * Hkv, hd).split([H, Hkv, Hkv], 1)
        K, V = cache(3, Hkv, 8, hd, F16)
        pos, slots = torch.arange(rows, device="cuda", dtype=torch.int32), torch.arange(rows, device="cuda", dtype=torch.int32) + 4
        want = Ops.QKNormRopePaged(None, q, k, v, None, None, 1e-6, pos, slots, K, V, base=1000.0)
        K2, V2 = cache(3, Hkv, 8, hd, F16)
        got = Ops.QKNormRopePaged(q, q, k, v, None, None, 1e-6, pos, slots, K2, V2, base=1000.0)
        assert torch.equal(got, want) and got.data_ptr() == q.data_ptr() and torch.equal(K, K2) and torch.equal(V, V2)
        ref, met = R.norm_rope(flat[off: off + rows * (H + 2 * Hkv) * hd].view(rows, -1, hd)[:, :H], None, 0, pos, 1, hd, 1000.0)
        assert ((got.double() - ref).abs() <= H_OF[F16] * ref.abs() + 2.0 ** -19 * met + 2.0 ** -25).all()


# ---------------------------------------------------------------------------------------------------------------------------- attention
def problem(t, H, Hkv, hd, page, lens, new, layout="heads", seed=0, extra=2, spread=1.0, rows_more=0, stale=float("nan")):
    """Rows, cache, table, starts and lengths; what the pages hold behind a sequence's end and all pages of nobody are `stale`."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, width = len(lens), max(R.pages(max(lens), page), 1) + extra
    pool = sum(R.pages(n, page) for n in lens) + 5
    K, V = cache(pool, Hkv, page, hd, t, layout, seed=seed + 1)
    order = torch.randperm(pool, generator=g, device="cuda").tolist()
    table, at = [], 0
    used = torch.zeros(pool * page, dtype=torch.bool)
    for n in lens:
        own = order[at: at + R.pages(n, page)]
        at += len(own)
        table.append(own + [-1] * (width - len(own)))
        for i in range(n):
            used[own[i // page] * page + i % page] = True
    gone = (~used).view(pool, 1, page, 1).cuda()
    K.masked_fill_(gone, stale)
    V.masked_fill_(gone, stale)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    q = (torch.randn(starts[-1] + rows_more, H, hd, generator=g, device="cuda") * spread).to(t)
    return q, K, V, ints(table), ints(starts), ints(lens)


def check(got, q, K, V, table, starts, lens, scale, window=0):
    t, hd = q.dtype, q.shape[2]
    want, mass, size = R.attention(q, K, V, table, starts.tolist(), lens.tolist(), scale, window)
    owned = ~want.isnan()
    tol = mass * (2 * H_OF[t] + 2 * (hd + 3) * 2.0 ** -24 * size + 2.0 ** -19) + 2.0 ** -24
    if t == F16:
        tol = tol + int(lens.max()) * 2.0 ** -25 * V[~V.isnan()].abs().max().double()
    off = (got.double() - want).abs()
    bad = owned & ~(off <= tol)
    assert not bad.any(), (int(bad.sum()), float((off / tol)[owned].nan_to_num(1e9).max()), bad.nonzero()[0].tolist())
    return owned


SHAPES = [(4, 4, 64), (8, 2, 64), (32, 8, 128), (8, 1, 128), (6, 2, 64), (5, 1, 128), (16, 1, 64), (3, 3, 32), (4, 2, 80), (2, 1, 256), (24, 2, 8)]


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("H,Hkv,hd", SHAPES)
def test_single_tokens(cuda, t, H, Hkv, hd):
    for page, lens in ((16, [1]), (8, [1, 2, 7, 8, 9, 31, 32, 33, 63, 64, 65, 127, 128, 129, 500]), (64, [1300, 3, 700]), (256, [255, 256, 257])):
        a = problem(t, H, Hkv, hd, page, lens, [1] * len(lens), seed=hd + page)
        got = Ops.PagedAttention(None, *a[:4], a[4], a[5], 1)
        assert check(got, *a, hd ** -0.5).all()


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("H,Hkv,hd", SHAPES)
def test_chunks(cuda, t, H, Hkv, hd):
    # drafts, prompts of their own and behind cached text, a sequence that stands still, an empty one; a window that ends inside pages and tiles
    for page, lens, new, window in ((16, [5, 40, 130, 9, 0, 77], [5, 3, 4, 0, 0, 2], 0), (8, [70, 300, 17], [70, 40, 1], 0), (32, [200, 90, 513], [129, 90, 128], 33),
                                    (128, [260, 1], [257, 1], 1)):
        a = problem(t, H, Hkv, hd, page, lens, new, layout="tokens" if page == 8 else "both" if page == 32 else "heads", seed=hd + page)
        got = Ops.PagedAttention(None, *a[:4], a[4], a[5], max(new), window=window)
        assert check(got, *a, hd ** -0.5, window).all()


@pytest.mark.parametrize("t,H,Hkv,hd,lens,new,window", [
    (F16, 32, 8, 128, [9000], [1], 0), (BF16, 8, 1, 64, [20000, 3], [1, 1], 0), (F16, 4, 4, 128, [5000, 12000], [7, 5], 0), (BF16, 32, 8, 64, [6000, 100], [600, 100], 0),
    (F32, 8, 8, 64, [4000], [1], 0), (F32, 4, 2, 128, [2500, 40], [90, 33], 300), (F16, 16, 2, 64, [7000], [300], 1000), (BF16, 4, 1, 128, [16384], [16], 5000),
    (F16, 6, 2, 128, [3000, 2000, 1], [700, 1, 1], 0), (BF16, 3, 1, 64, [1500], [1500], 0)])
def test_long_sequences(cuda, t, H, Hkv, hd, lens, new, window):
    a = problem(t, H, Hkv, hd, 16, lens, new, seed=sum(lens))
    got = Ops.PagedAttention(None, *a[:4], a[4], a[5], max(new), window=window)
    assert check(got, *a, hd ** -0.5, window).all()
    assert torch.equal(got, Ops.PagedAttention(None, *a[:4], a[4], a[5], max(new), window=window))    # the same bits each time


@pytest.mark.parametrize("t,n", [(F32, 1), (F16, 1), (BF16, 4), (F16, 200), (BF16, 200)])
def test_many_sequences(cuda, t, n):
    rng = np.random.default_rng(n)
    new = [n] + [int(x) for x in rng.integers(0, n + 1, 699)]
    lens = [m + int(x) for m, x in zip(new, rng.integers(0, 60, 700))]
    a = problem(t, 4, 1, 64, 8, lens, new, seed=n)
    assert check(Ops.PagedAttention(None, *a[:4], a[4], a[5], n), *a, 0.125).all()


@pytest.mark.parametrize("t,n,hd", [(F32, 1, 64), (F32, 30, 64), (F16, 1, 128), (F16, 9, 64), (BF16, 300, 128), (F16, 300, 64)])
def test_pages_that_are_none(cuda, t, n, hd):
    # entries that name no page hide their keys; where a row's window lies in them it becomes zero
    lens, new = [700, 300, n, 500], [n, n, n, n]
    q, K, V, table, starts, lens_ = problem(t, 8, 2, hd, 16, lens, new, seed=n)
    table[0, :10], table[0, 20] = -1, 2 ** 31 - 1
    table[1] = -3
    table[3, 0::2] = K.shape[0]
    for window in (0, 20):
        got = Ops.PagedAttention(None, q, K, V, table, starts, lens_, n, window=window)
        assert check(got, q, K, V, table, starts, lens_, hd ** -0.5, window).all()
        assert (got[n: 2 * n] == 0).all()


@pytest.mark.parametrize("t,n,hd", [(F32, 3, 64), (F16, 1, 64), (BF16, 20, 128), (F16, 150, 128)])
def test_rows_of_nobody_stay(cuda, t, n, hd):
    a = problem(t, 4, 2, hd, 16, [n + 30, n, 5], [n, n, 0], rows_more=9, seed=n)
    q, K, V, table, starts, lens = a
    result = torch.full((2 * n + 9, 6, hd), 3.0, dtype=t, device="cuda")[:, 1:5]            # heads of a wider row
    wide = torch.randn(q.shape[0], 7, hd, device="cuda").to(t)
    wide[:, 2:6] = q
    got = Ops.PagedAttention(result, wide[:, 2:6], K, V, table, starts, lens, n)
    assert got.data_ptr() == result.data_ptr() and (result[2 * n:] == 3.0).all()
    owned = check(got, q, K, V, table, starts, lens, hd ** -0.5)
    assert owned[:2 * n].all() and not owned[2 * n:].any()
    # a length below the rows: the first of them have no position and see nothing; rows that do not exist are nobody's
    lens[0], starts[2], starts[3] = 1, q.shape[0] + 1, q.shape[0] + 1
    result.fill_(3.0)
    Ops.PagedAttention(result, wide[:, 2:6], K, V, table, starts, lens, n)
    assert (result[: n - 1] == 0).all() and (result[n:] == 3.0).all() and not result.isnan().any()


@pytest.mark.parametrize("t,n", [(F32, 5), (F16, 1), (F16, 5), (F16, 200), (BF16, 200)])
def test_sharp_and_flat_scores(cuda, t, n):
    for spread, scale in ((30.0, 1.0), (0.0, 0.125), (1.0, -0.3), (1.0, 0.0)):
        a = problem(t, 8, 2, 64, 16, [900, n + 1], [n, n], spread=spread, seed=n)
        check(Ops.PagedAttention(None, *a[:4], a[4], a[5], n, scale=scale), *a, scale)


@pytest.mark.parametrize("t,n", [(F32, 2), (F16, 1), (F16, 150), (BF16, 6)])
def test_nan_spreads_to_its_rows_only(cuda, t, n):
    q, K, V, table, starts, lens = problem(t, 4, 2, 64, 16, [400, 300], [n, n], seed=4)
    K[table[0, 3], 1, 5] = float("nan")                       # one key of sequence 0, KV head 1
    got = Ops.PagedAttention(None, q, K, V, table, starts, lens, n)
    assert got[:n, 2:].isnan().all() and not got[:n, :2].isnan().any() and not got[n:].isnan().any()


@pytest.mark.parametrize("t,n", [(F32, 1), (F16, 1), (BF16, 6), (F16, 300)])
def test_captured_call_with_other_lengths(cuda, t, n):
    big = problem(t, 8, 2, 64, 16, [3000, 900, 40 + n], [n, n, n], seed=5)
    q, K, V, table, starts, lens = (x.clone() for x in big)
    s = torch.cuda.Stream()
    out = torch.zeros_like(q)
    with torch.cuda.stream(s):
        Ops.PagedAttention(out, q, K, V, table, starts, lens, n)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            Ops.PagedAttention(out, q, K, V, table, starts, lens, n)
        for new_lens, new_rows in (([3000, 900, 40 + n], [n, n, n]), ([n, 700, 1], [n, max(1, n // 2), 1]), ([2999, 1, 0], [n, 1, 0])):
            lens.copy_(ints(new_lens))
            starts.copy_(ints(np.cumsum([0] + new_rows).tolist()))
            out.fill_(5.0)
            g.replay()
            s.synchronize()
            clean = (q, K.nan_to_num(0.5), V.nan_to_num(0.5), table, starts, lens)
            owned = check(out, *clean, 0.125)
            assert (out[~owned] == 5.0).all()


def test_more_rows_than_announced(cuda):
    for t in (F32, F16):
        a = problem(t, 8, 2, 64, 16, [400, 90], [150, 2], seed=6)
        assert check(Ops.PagedAttention(None, *a[:4], a[4], a[5], 1), *a, 0.125).all()


def test_places_beyond_32_bits(cuda):
    # 2^31 elements and more in front of the pages in use
    Hkv, page, hd = 8, 256, 128
    pages = 2 ** 31 // (Hkv * page * hd) + 40
    for n in (1, 6, 300):
        K, V = (torch.empty(pages, Hkv, page, hd, dtype=F16, device="cuda") for _ in range(2))
        K[-40:], V[-40:] = torch.randn(40, Hkv, page, hd, device="cuda").to(F16), torch.randn(40, Hkv, page, hd, device="cuda").to(F16)
        table = ints([list(range(pages - 30, pages - 20)), list(range(pages - 10, pages))])
        starts, lens, pos = ints([0, n, 2 * n]), ints([2560, 2001]), torch.arange(2 * n, device="cuda", dtype=torch.int32)
        q, k, v = (torch.randn(2 * n, h, hd, device="cuda").to(F16) for h in (16, Hkv, Hkv))
        place = torch.cat([torch.arange(lens[b].item() - n, lens[b].item()) for b in range(2)])
        slots = torch.stack([table[r // n, place[r] // page] * page + place[r] % page for r in range(2 * n)]).to(torch.int32)
        assert slots.min() * Hkv * hd > 2 ** 31 - 1 or int(slots.min()) * Hkv * hd > 2 ** 31 - 1
        Ops.QKNormRopePaged(q, q, k, v, None, None, 0.0, pos, slots, K, V, ropeStyle=0)
        assert torch.equal(V[slots.long() // page, :, slots.long() % page], v)
        tail = slice(pages - 40, pages)
        got = Ops.PagedAttention(None, q, K, V, table, starts, lens, n)
        assert check(got, q, K[tail], V[tail], table - (pages - 40), starts, lens, hd ** -0.5).all()
        del K, V


# ---------------------------------------------------------------------------------------------------------------------------- drafted tokens
def draft_case(B, K, V, rows, seed, certain=False, pad=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    starts = np.cumsum([0] + rows).tolist()
    p = torch.softmax(torch.randn(max(starts[-1], 1) + pad, V, generator=g, device="cuda") * 2, -1)
    q = torch.softmax(torch.randn(B * K, V, generator=g, device="cuda") * 2, -1)
    draft = torch.randint(0, V, (B, K), generator=g, device="cuda", dtype=torch.int32)
    for b in range(B):                                       # half of the drafts are likely under the target
        for i in range(min(K, rows[b] - 1)):
            if (b + i) % 2:
                draft[b, i] = p[starts[b] + i].argmax()
    u = torch.rand(B, K + 1, generator=g, device="cuda")
    return p, None if certain else q, draft, u, starts


def verified(p, q, draft, u, starts, K, given=True):
    got = Ops.VerifyDraft(p, q, draft, u, ints(starts) if given else None)
    host = lambda x: None if x is None else x.double().cpu().numpy()  # noqa: E731
    want = R.verify(host(p), host(q), draft.tolist(), host(u), starts, K)
    assert got[0].tolist() == want[0] and got[1].tolist() == want[1]
    return want


@pytest.mark.parametrize("certain", [False, True])
@pytest.mark.parametrize("B,K,V", [(1, 4, 32000), (3, 1, 1), (5, 3, 2), (9, 7, 50257), (70, 2, 501), (2, 0, 777), (4, 5, 4095), (3, 8, 131073), (1, 2, 513)])
def test_drafts(cuda, B, K, V, certain):
    rows = [K + 1] * B
    verified(*draft_case(B, K, V, rows, B + V, certain), K, given=False)
    rng = np.random.default_rng(V)
    rows = [int(x) for x in rng.integers(0, K + 2, B)]       # sequences with fewer drafts, without any, without rows
    counts = verified(*draft_case(B, K, V, rows, B + K, certain, pad=2), K)[1]
    assert all((c == 0) == (r == 0) for c, r in zip(counts, rows))


def test_drafts_at_the_borders(cuda):
    V, K = 1000, 3
    p, q, draft, u, starts = draft_case(6, K, V, [4] * 6, 1)
    q[0:3] = p[0:3]                                          # the same distributions: accepted whatever u is, nothing left of p - q where u is 1
    u[0] = 1 - 2.0 ** -24
    u[1] = 0.0
    draft[2, 0], draft[3, 0], draft[4, 1] = -1, V, 2 ** 31 - 1
    p[20:24] = 0.0
    p[20, 7] = 1.0
    draft[5, 0] = 7
    q[15:18] = 1.0 / V
    u[5] = torch.tensor([0.5, 0.0, 0.0, 0.999], device="cuda")
    tokens, counts = verified(p, q, draft, u, starts, K)
    assert counts[0] == 4 and counts[2] == counts[3] == 1 and tokens[5][:2] == [7, -1]     # row 21 has no weight at all
    # refused where p <= q everywhere: drawn from p
    p, q, draft, u, starts = draft_case(1, 1, 64, [2], 2)
    q.copy_(p[:1] * 2)
    u[0, 0] = 0.9
    verified(p, q, draft, u, starts, 1)
    # a sum that ends in zeros; one word
    p.zero_()
    p[0, 3], p[1, 5] = 0.25, 0.5
    u[0] = 1 - 2.0 ** -24
    assert verified(p, q, draft, u, starts, 1)[0][0][0] == 3


def test_drafts_strided_and_behind(cuda):
    p, q, draft, u, starts = draft_case(4, 3, 300, [4, 2, 0, 3], 3, pad=4)
    wide_p, wide_q = torch.rand(p.shape[0], 333, device="cuda"), torch.rand(q.shape[0], 301, device="cuda")
    wide_p[:, 5:305], wide_q[:, 1:] = p, q
    a = Ops.VerifyDraft(wide_p[:, 5:305], wide_q[:, 1:], draft, u, ints(starts))
    b = Ops.VerifyDraft(p, q, draft, u, ints(starts))
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    # rows that are not there are no rows; more than K + 1 count as K + 1
    bad = Ops.VerifyDraft(p, q, draft, u, ints([0, 4, p.shape[0] + 1, -1, 9]))
    assert bad[1].tolist()[1:] == [0, 0, 0] and bad[1][0] == b[1][0]


def test_drafted_tokens_follow_the_target(cuda):
    # whatever the draft's distribution, the first token's is the target's: 40000 draws, each frequency within six standard deviations
    V, B = 12, 40000
    g = torch.Generator(device="cuda").manual_seed(9)
    pt, qt = torch.softmax(torch.randn(2, V, generator=g, device="cuda"), -1), torch.softmax(2 * torch.randn(1, V, generator=g, device="cuda"), -1)
    draft = torch.multinomial(qt[0].expand(B, V), 1, generator=g).to(torch.int32)
    tokens, _ = Ops.VerifyDraft(pt.repeat(B, 1), qt.repeat(B, 1), draft, torch.rand(B, 2, generator=g, device="cuda"))
    share = torch.bincount(tokens[:, 0], minlength=V).double() / B
    assert ((share - pt[0].double()).abs() <= 6 * (pt[0].double() / B).sqrt()).all()


# ---------------------------------------------------------------------------------------------------------------------------- together
@pytest.mark.parametrize("t", [F32, F16, BF16])
def test_a_run_with_drafts(cuda, t):
    """One attention layer, requests that come and go, drafts accepted and refused: the cache after every step is that of the accepted
    text, and every row's attention is that of its sequence computed alone."""
    H, Hkv, hd, page, B, V, K, width = 8, 2, 64, 8, 5, 50, 3, 12
    g = torch.Generator(device="cuda").manual_seed(11)
    embed = torch.randn(V, (H + 2 * Hkv) * hd, generator=g, device="cuda").to(t)
    wq, wk = ((1 + 0.1 * torch.randn(hd, generator=g, device="cuda")).to(t) for _ in range(2))
    pool = Pool(B, width, page, 40, seed=2)
    Kc, Vc = cache(40, Hkv, page, hd, t, fill=float("nan"))
    text = [[] for _ in range(B)]
    rng = np.random.default_rng(5)
    lens = [0] * B
    for step in range(7):
        prompts = [[int(x) for x in rng.integers(0, V, int(rng.integers(1, 30)))] if not text[b] and (b + step) % 2 == 0 else [] for b in range(B)]
        drafts = [[int(x) for x in rng.integers(0, V, K)] if text[b] else [] for b in range(B)]
        fed = [prompts[b] or ([text[b][-1]] + drafts[b] if text[b] else []) for b in range(B)]
        rows = sum(map(len, fed)) + 4
        before = list(lens)
        _, starts, _, positions = pool.step(lens, [len(f) for f in fed], rows)
        # the device's own answers go on from here
        d_lens, d_starts, d_slots, d_pos = [ints(x) for x in ([a + len(f) for a, f in zip(before, fed)], starts, R_slots(pool, before, fed, rows), positions)]
        ids = torch.tensor(sum(fed, []) + [0] * 4, device="cuda")
        q, k, v = (x.unflatten(1, (-1, hd)) for x in embed[ids].split([H * hd, Hkv * hd, Hkv * hd], 1))
        qn = Ops.QKNormRopePaged(None, q, k, v, wq, wk, 1e-6, d_pos, d_slots, Kc, Vc, ropeStyle=2)
        out = Ops.PagedAttention(torch.zeros_like(qn), qn, Kc, Vc, pool.d_table, d_starts, d_lens, max(1, max(map(len, fed))))
        assert not out.isnan().any()
        check(out, qn, Kc, Vc, pool.d_table, d_starts, d_lens, hd ** -0.5)
        # the same rows from the whole text of the sequence, without a cache
        for b in range(B):
            if not fed[b]:
                continue
            whole = torch.tensor((text[b][:-1] if not prompts[b] else []) + fed[b], device="cuda")
            kk = embed[whole][:, H * hd:(H + Hkv) * hd].unflatten(1, (-1, hd))
            kk, _ = R.norm_rope(kk, wk, 1e-6, torch.arange(len(whole), device="cuda"), 2, hd, 500000.0)
            held = torch.stack([Kc[pool.table[b][i // page], :, i % page] for i in range(len(whole))]).double()
            assert ((held - kk).abs() <= H_OF[t] * kk.abs() + 2.0 ** -17 * kk.abs().max()).all()
        # verification: probabilities from the attention's output
        n_rows = [min(len(f), K + 1) if text[b] else 0 for b, f in enumerate(fed)]
        probs = torch.softmax(out.float().reshape(out.shape[0], -1)[:, :V] * 3, -1)
        vs = np.cumsum([0] + n_rows).tolist()
        pick = sum([list(range(starts[b], starts[b] + n_rows[b])) for b in range(B)], [])
        p = probs[torch.tensor(pick, dtype=torch.long, device="cuda")] if pick else probs[:0]
        d = ints([f or [0] * K for f in drafts])
        u = torch.rand(B, K + 1, generator=g, device="cuda")
        qd = torch.full((B * K, V), 1.0 / V, device="cuda")
        tokens, counts = Ops.VerifyDraft(p, qd, d, u, ints(vs))
        tokens, counts = tokens.tolist(), counts.tolist()
        for b in range(B):
            if prompts[b]:
                text[b] = prompts[b] + [int(rng.integers(0, V))]
                lens[b] = len(prompts[b])
            elif text[b]:
                text[b] += tokens[b][:counts[b]]
                lens[b] = before[b] + counts[b]
            if len(text[b]) > 60 or (text[b] and rng.random() < 0.15):
                text[b], lens[b] = [], 0
        pool.step(lens, [0] * B, 0)      # refused drafts and ended requests give their pages back
    assert sum(pool.held) + len(pool.free) == 40


def R_slots(pool, before, fed, rows):
    s = [pool.table[b][(before[b] + i) // pool.page] * pool.page + (before[b] + i) % pool.page for b, f in enumerate(fed) for i in range(len(f))]
    return s + [-1] * (rows - len(s))


# ---------------------------------------------------------------------------------------------------------------------------- streams, refusals
def test_another_stream(cuda):
    a = problem(F16, 8, 2, 64, 16, [2000, 400], [1, 1], seed=7)
    want = Ops.PagedAttention(None, *a[:4], a[4], a[5], 1)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    big = torch.randn(6000, 6000, device="cuda")
    with torch.cuda.stream(s):
        for _ in range(5):
            big = big @ big * 1e-4
        q = a[0] + 0 * big[0, 0].to(F16).nan_to_num(0.0)
        got = Ops.PagedAttention(None, q, *a[1:4], a[4], a[5], 1)
        twice = got + got
    s.synchronize()
    assert torch.equal(twice, want + want)
    # the default stream: in its place among torch's work, without a wait of the host
    q = torch.zeros_like(a[0])
    q.copy_(a[0])
    assert torch.equal(Ops.PagedAttention(None, q, *a[1:4], a[4], a[5], 1) * 2, want * 2)


def test_wrong_tensors_are_refused(cuda):
    q, K, V, table, starts, lens = problem(F16, 8, 2, 64, 16, [40, 50], [1, 1])
    for args in ((q.double(), K, V, table, starts, lens), (q, K.float(), V, table, starts, lens), (q, K, V[:, :1], table, starts, lens), (q, K, V, table.long(), starts, lens),
                 (q, K, V, table.t(), starts, lens), (q, K, V, table, starts[:2], lens), (q, K, V, table, starts, lens[:1]), (q.cpu(), K, V, table, starts, lens),
                 (q, K, V, table.cpu(), starts, lens), (q[:, :7], K, V, table, starts, lens), (q[..., :32], K, V, table, starts, lens), (q[0], K, V, table, starts, lens)):
        with pytest.raises(N.TSB200Error):
            Ops.PagedAttention(None, *args, 1)
    with pytest.raises(N.TSB200Error, match="workspace"):
        N.call("TSB200_PagedAttention", 0, N.F16, q.data_ptr(), 512, 64, q.data_ptr(), 512, 64, K.data_ptr(), V.data_ptr(), 2048, 1024, 64, K.shape[0], 16, table.data_ptr(),
               table.stride(0), table.shape[1], starts.data_ptr(), lens.data_ptr(), 2, 2, 1, 8, 2, 64, 0.125, 0, K.data_ptr(), 100, None)
    with pytest.raises(N.TSB200Error):
        Ops.VerifyDraft(torch.rand(8, 10, device="cuda"), None, ints([[1, 2, 3]]), torch.rand(1, 3, device="cuda"))
    with pytest.raises(N.TSB200Error):
        Ops.PagedPlan(ints([1]), ints([1]), ints([[1]]), ints([0]), ints([0]), ints([1, 2]), 16, 4)
    with pytest.raises(N.TSB200Error):
        Ops.QKNormRopePaged(None, q, K[:2, 0, :2], K[:2, 0, :2], None, None, 1e-6, ints([0]), ints([0, 1]), K, V)


@pytest.mark.parametrize("t,H,Hkv,n,lens", [(F16, 128, 1, 1, [700, 3]), (BF16, 256, 1, 1, [300]), (F16, 20, 1, 9, [260, 9]), (F16, 24, 2, 30, [500, 30]), (BF16, 64, 2, 4, [1000, 129, 128, 127]),
                                            (F16, 7, 7, 65, [65, 400])])
def test_large_and_odd_groups(cuda, t, H, Hkv, n, lens):
    for hd, window in ((64, 0), (128, 50)):
        a = problem(t, H, Hkv, hd, 8, lens, [n] * len(lens), seed=H)
        assert check(Ops.PagedAttention(None, *a[:4], a[4], a[5], n, window=window), *a, hd ** -0.5, window).all()


@pytest.mark.parametrize("t,n", [(F32, 1), (F32, 40), (F16, 1), (F16, 100)])
def test_lengths_beyond_the_table(cuda, t, n):
    # positions behind the table's last page: every key of the table is seen
    q, K, V, table, starts, lens = problem(t, 4, 2, 64, 16, [320, 320], [n, n], extra=0, seed=8)
    lens.copy_(ints([320 + 7, 2 ** 31 - 1]))
    got = Ops.PagedAttention(None, q, K, V, table, starts, lens, n)
    assert check(got, q, K, V, table, starts, ints([320 + n + 7, 320 + n + 7]), 0.125)[n:].all() if n == 1 else not got.isnan().any()
    every = ints([320 + n, 320 + n])
    want = Ops.PagedAttention(None, q, K, V, table, starts, every, n)
    assert torch.equal(got[n:], want[n:])


@pytest.mark.parametrize("t,n", [(F32, 1), (F32, 40), (F16, 1), (F16, 5), (BF16, 100)])
def test_many_calls_at_once(cuda, t, n):
    problems = [problem(t, 8, 2, 64, 16, [900 + 37 * i, n], [n, n], seed=20 + i) for i in range(6)]
    want = [Ops.PagedAttention(None, *a[:4], a[4], a[5], n) for a in problems]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in problems]
    got = []
    for _ in range(3):
        for s, a in zip(streams, problems):
            with torch.cuda.stream(s):
                got.append(Ops.PagedAttention(None, *a[:4], a[4], a[5], n))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i % 6]) for i, g in enumerate(got))


def test_captured_plan_append_attention_verify(cuda):
    """A step captured once and replayed with other lengths, its buffers a little larger than its rows."""
    H, Hkv, hd, page, B, K, V = 8, 2, 64, 16, 3, 2, 40
    pool = Pool(B, 20, page, 64, seed=4)
    Kc, Vc = cache(64, Hkv, page, hd, F16)
    cached, fresh = ints([0, 0, 0]), ints([1, 1, 1])
    q, k, v = (torch.randn(12, h, hd, device="cuda").to(F16) for h in (H, Hkv, Hkv))
    out, p = torch.zeros_like(q), torch.softmax(torch.randn(12, V, device="cuda"), -1)
    draft, u = ints([[1, 2], [3, 4], [5, 6]]), torch.rand(B, K + 1, device="cuda")

    def step():
        lens, starts, slots, positions = Ops.PagedPlan(cached, fresh, pool.d_table, pool.d_held, pool.d_free, pool.d_count, page, 12)
        qn = Ops.QKNormRopePaged(torch.zeros_like(q), q, k, v, None, None, 0.0, positions, slots, Kc, Vc)
        Ops.PagedAttention(out, qn, Kc, Vc, pool.d_table, starts, lens, 8)
        return (lens, starts, slots, positions, qn) + tuple(Ops.VerifyDraft(p, None, draft, u, starts))
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            got = step()
        for new in ([5, 1, 3], [1, 0, 8], [3, 3, 3], [0, 0, 0]):
            before = cached.tolist()
            fresh.copy_(ints(new))
            out.fill_(7.0)
            g.replay()
            s.synchronize()
            want = R.plan(before, new, pool.table, pool.held, pool.free, page, 12)
            assert [x.tolist() for x in got[:4]] == list(want)
            total = sum(new)
            owned = check(out, got[4], Kc, Vc, pool.d_table, got[1], got[0], hd ** -0.5)
            assert owned[:total].all() and (out[total:] == 7.0).all()
            counts = got[6].tolist()
            assert all((c == 0) == (n == 0) and c <= max(n, 1) for c, n in zip(counts, new))
            cached.copy_(got[0])


# (a poll waits for some microseconds by itself, so that short calls get what they wait for)
@pytest.mark.parametrize("H,hd,n,T", [(32, 128, 1, 20000), (32, 64, 12, 40000), (32, 128, 300, 20000), (24, 128, 300, 20000), (32, 64, 300, 40000)])
def test_a_wait_that_runs_out(cuda, H, hd, n, T):
    """One poll per wait (an environment variable, hence a process of its own): every warp gives up in its own place, copies and products in flight end before a
    CTA leaves, the synchronisation says so, and the calls behind it are sound."""
    import os
    import subprocess
    import sys
    code = """
import torch
from seq2seqsharp_b200 import _native as N
from seq2seqsharp_b200.ops import Ops
H, hd, n, T = %d, %d, %d, %d
pages = 2 * (T // 16 + 1)
K, V = (torch.randn(pages, 8, 16, hd, device="cuda", dtype=torch.float16) for _ in range(2))
q = torch.randn(2 * n, H, hd, device="cuda", dtype=torch.float16)
i = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
table = torch.arange(pages, dtype=torch.int32, device="cuda").view(2, -1)
for _ in range(4):
    out = Ops.PagedAttention(None, q, K, V, table, i([0, n, 2 * n]), i([T, T - 40]), n)
torch.cuda.synchronize()
try:
    N.call("TSB200_Synchronize", 0, None)
    print("silent")
except N.TSB200Error as e:
    print(e)
N.call("TSB200_Synchronize", 0, None)
print("usable", float(torch.ones(4, device="cuda").sum()))
""" % (H, hd, n, T)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120, env=dict(os.environ, TSB200_WAIT_LIMIT="1"),
                       cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert r.returncode == 0, r.stderr
    assert "gave up waiting" in r.stdout and "usable 4.0" in r.stdout, r.stdout
