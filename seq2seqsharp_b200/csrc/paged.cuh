// Attention of packed rows over a paged key / value cache: what its kernels share.
//
// Rows of several sequences lie one after the other (starts[b] .. starts[b + 1]); those of sequence b are the last ones of its lens[b] cached tokens,
// so row i of n sees the keys j <= lens[b] - n + i, and with a window only j > that position - window.  Key j lies in page table[b][j / page]
// at place j % page.  Entries that name no page hide their keys, and a row that sees no key is written as zeros.
//
// Work: an item is (sequence, tile of RT of its n * G (query, head) pairs, KV head), a unit a tile of KT of the item's keys, or the time of one: an item
// begins with `start` units for what it costs beside its keys.  What is known on the
// host are bounds only (a captured call is replayed with other lengths), so each CTA reads the lengths, numbers all units and takes an equal run of
// them: one sequence of any length, or sequences of very different lengths, keep every SM busy.  A run may begin or end inside an item; such a
// CTA leaves its maximum, sum and accumulator in the workspace and paged_combine_kernel joins them in the order of the runs (the same
// order whatever CTA ends first).  Ends within a 32nd of a run of an item's end, or within `snap` units, are moved there: a record has to be written and read.
#pragma once
#include <cuda.h>

#include "kernels.cuh"

namespace tsb {

// division of numbers below 2^31 by one that the host knows
struct PagedDiv {
  uint32_t mul, shift;
  void set(uint32_t d) {
    shift = 0;
    while ((1ull << shift) < d) ++shift;
    mul = (uint32_t)((((1ull << shift) - d) << 32) / d + 1);
  }
  __device__ __forceinline__ int operator()(int n) const { return (int)((__umulhi(mul, (uint32_t)n) + (uint32_t)n) >> shift); }
};
struct PagedArgs {
  void* out;                       // [rows, H, hd], strides o_row, o_head
  const void* q;                   // [rows, H, hd], strides q_row, q_head
  const void *K, *V;               // page, KV head, place: strides c_page, c_head, c_tok
  int64_t o_row, o_head, q_row, q_head, c_page, c_head, c_tok;
  const int* table;
  int64_t table_stride;
  int max_blocks, num_pages, page_shift;
  const int *starts, *lens;
  int B, rows, H, Hkv, G, hd;
  PagedDiv by_G;
  float c;                         // scale * log2(e)
  int window;                      // 0: none
  float* part;                     // records: paged_record_floats() each, two per CTA
  int4* joins;                     // two per CTA: the item that the run's beginning is the first to fall into (PagedJoin)
  int min_units, snap;             // no run is shorter; ends this near to an item's are moved there (at least `start`)
  int most;                        // (query, head) pairs of a KV head that a sequence may have, as far as the host knows
  int start;                       // units that an item costs beside those of its keys
  unsigned wait_limit;
  int* error;
};

// 16 bytes to shared memory, zeros where there is nothing
__device__ __forceinline__ void paged_cp16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void paged_cp16(void* dst, const void* src, bool there) { paged_cp16((uint32_t)__cvta_generic_to_shared(dst), src, there); }

// a record: (maximum, sum) of RT rows, then their accumulators
__host__ __device__ inline int64_t paged_record_floats(int RT, int hd) { return (int64_t)RT * (hd + 2); }

struct PagedSeq {
  int row0, n, len;
};
__device__ __forceinline__ PagedSeq paged_seq(const PagedArgs& a, int b) {
  const int r0 = a.starts[b], r1 = a.starts[b + 1];
  PagedSeq s;
  s.row0 = r0;
  s.n = r0 >= 0 && r1 > r0 && r1 <= a.rows ? r1 - r0 : 0;   // rows that are not there are nobody's
  s.len = min(max(a.lens[b], 0), 0x7fff0000);   // positions and what is added to them stay below 2^31
  return s;
}
// the first key that a tile of pairs sees, the first of which is p0
__device__ __forceinline__ int paged_front(const PagedArgs& a, const PagedSeq& s, int p0) {
  const int first = s.len - s.n + a.by_G(p0);
  return a.window > 0 && a.window <= first ? first - a.window + 1 : 0;
}
struct PagedTile {
  int k0, units;   // first key tile, how many
};
__device__ __forceinline__ PagedTile paged_tile(const PagedArgs& a, const PagedSeq& s, int t, int RT, int KT) {
  const int p1 = min(s.n * a.G, (t + 1) * RT) - 1;
  const int last = s.len - s.n + a.by_G(p1);   // its position
  const int hi = min(last + 1, a.max_blocks << a.page_shift);
  PagedTile r;
  r.k0 = paged_front(a, s, t * RT) / KT;
  r.units = max(1, (hi + KT - 1) / KT - r.k0);   // a tile without keys is still written
  return r;
}
// where a run begins or ends: key tile `off` (0 .. units) of an item whose first unit is number `s` of all
struct PagedLoc {
  int b, t, h, off, units;
  long long s;
};
// (records, first row of the sequence, first pair of the item, its pairs), (KV head, -, -, -)
struct PagedJoin {
  int records, row0, p0, pairs, h, pad[3];
};
static_assert(sizeof(PagedJoin) == 2 * sizeof(int4), "a join is written as two pieces");
struct PagedPlanShared {
  long long warp[32];
  PagedLoc loc[2];
};

template <int NT>
__device__ __forceinline__ long long paged_block_scan(long long v, PagedPlanShared& sh, long long& all) {   // exclusive
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  long long x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) sh.warp[w] = x;
  __syncthreads();
  long long before = 0, total = 0;
#pragma unroll
  for (int i = 0; i < NT / 32; ++i) {
    const long long y = sh.warp[i];
    if (i < w) before += y;
    total += y;
  }
  all = total;
  return before + x - v;
}
// Units of this lane's sequence (b, or none).  Few tiles are added up by the lane, many (a chunk) by the warp.
constexpr int kPagedFewTiles = 4;
__device__ __forceinline__ long long paged_seq_units(const PagedArgs& a, int b, int RT, int KT) {
  PagedSeq s{0, 0, 0};
  if (b < a.B) s = paged_seq(a, b);
  const int tiles = (s.n * a.G + RT - 1) / RT, lane = threadIdx.x & 31;
  int u = 0;
  if (tiles <= kPagedFewTiles)
    for (int t = 0; t < tiles; ++t) u += paged_tile(a, s, t, RT, KT).units + a.start;
  long long mine = u;
  for (unsigned many = __ballot_sync(0xffffffffu, tiles > kPagedFewTiles); many; many &= many - 1) {
    const int src = __ffs(many) - 1, nt = __shfl_sync(0xffffffffu, tiles, src);
    const PagedSeq q{0, __shfl_sync(0xffffffffu, s.n, src), __shfl_sync(0xffffffffu, s.len, src)};
    long long x = 0;
    for (int t = lane; t < nt; t += 32) x += paged_tile(a, q, t, RT, KT).units + a.start;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    if (lane == src) mine = x;
  }
  return mine * a.Hkv;
}
// Unit x of all, where sequence b's first is s: tile, head and place in the item.  By a whole warp, for its lane `src`'s sequence.
__device__ __forceinline__ PagedLoc paged_find(const PagedArgs& a, int b, long long s, long long x, long long tol, int RT, int KT) {
  const int lane = threadIdx.x & 31;
  const PagedSeq q = paged_seq(a, b);
  auto place = [&](int t, int cost, long long at) {
    PagedLoc l;
    l.b = b;
    l.t = t;
    // below 65536: the quotient in fp32 is off by one at most
    l.h = (int)__fdividef((float)(x - at), (float)max(cost, 1));
    if ((long long)l.h * cost > x - at) --l.h;
    else if ((long long)(l.h + 1) * cost <= x - at) ++l.h;
    l.s = at + (long long)l.h * cost;
    l.units = cost - a.start;
    const int in_item = (int)(x - l.s), rest = cost - in_item;
    if (in_item <= a.start || (in_item <= tol && in_item <= rest)) l.off = 0;
    else l.off = rest <= tol ? l.units : in_item - a.start;
    return l;
  };
  if (q.n * a.G <= RT) return place(0, paged_tile(a, q, 0, RT, KT).units + a.start, s);   // a single tile: tokens, drafts
  for (int t0 = 0;; t0 += 32) {
    const bool there = (long long)(t0 + lane) * RT < (long long)q.n * a.G;
    const int u = there ? paged_tile(a, q, t0 + lane, RT, KT).units + a.start : 0;   // of one head
    long long end = (long long)u * a.Hkv;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, end, o);
      if (lane >= o) end += y;
    }
    const unsigned in = __ballot_sync(0xffffffffu, there && x < s + end);
    if (in == 0 && __any_sync(0xffffffffu, there)) {
      s += __shfl_sync(0xffffffffu, end, 31);
      continue;
    }
    const int src = in ? __ffs(in) - 1 : 0;
    const int cost = __shfl_sync(0xffffffffu, u, src);
    return place(t0 + src, cost, s + __shfl_sync(0xffffffffu, end, src) - (long long)cost * a.Hkv);
  }
}
// The runs: `rest` of each + 1 units, then the others of each.  (Divisions of 64 bits, four one after the other, were half of the time to find a run's place.)
struct PagedRuns {
  long long each;
  int rest;
  __device__ __forceinline__ PagedRuns(long long all, int runs) {
    if (all < 1ll << 31) {
      each = (uint32_t)all / (uint32_t)runs;
    } else {
      each = all / runs;
    }
    rest = (int)(all - each * runs);
  }
  __device__ __forceinline__ long long begin(int c) const { return each * c + min(c, rest); }
};
// Run `c` of the plan: sh.loc[0] and sh.loc[1] where it begins and ends.  Returns whether there is such a run.  `all` / `runs`: units and runs of
// the whole call.  All threads of the CTA.
template <int NT, int RT, int KT>
__device__ __forceinline__ bool paged_locate(const PagedArgs& a, int c, int ctas, PagedPlanShared& sh, long long& all, int& runs) {
  const int tid = threadIdx.x, w = tid >> 5;
  // few sequences: every warp adds them up for itself, the first two look for an end each
  const bool few = a.B <= 32;
  // the last run ends where no warp finds a unit; in front of the scans' barriers, behind which the other runs' ends are found by whichever warp has them
  if (!few && tid == 0) sh.loc[1] = PagedLoc{a.B, 0, 0, 0, 0, 0};
  long long mine = paged_seq_units(a, few ? tid & 31 : tid, RT, KT), before = 0;
  if (few) {
    long long to = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, to, o);
      if ((tid & 31) >= o) to += y;
    }
    before = to - mine;
    all = __shfl_sync(0xffffffffu, to, 31);
  } else if (a.B <= NT) {
    before = paged_block_scan<NT>(mine, sh, all);
  } else {
    long long total = mine;
    for (int b0 = NT; b0 < a.B; b0 += NT) total += paged_seq_units(a, b0 + tid, RT, KT);
    paged_block_scan<NT>(total, sh, all);
  }
  runs = all >= (long long)a.min_units * ctas ? ctas : max(1, (int)all / a.min_units);
  if (all == 0 || c >= runs) {
    if (tid == 0) a.joins[2 * c] = make_int4(0, 0, 0, 0);
    return false;
  }
  const PagedRuns split(all, runs);
  const long long tol = max(split.each >> 5, (long long)a.snap);
  const long long x[2] = {split.begin(c), split.begin(c + 1)};
  if (few) {
    if (w < 2) {
      const long long y = x[w];
      const unsigned hit = __ballot_sync(0xffffffffu, mine > 0 && y >= before && y < before + mine);
      PagedLoc l{a.B, 0, 0, 0, 0, all};
      if (hit) {
        const int src = __ffs(hit) - 1;
        l = paged_find(a, src, __shfl_sync(0xffffffffu, before, src), y, tol, RT, KT);
      }
      if ((tid & 31) == 0) sh.loc[w] = l;
    }
  }
  long long base = 0;
  for (int b0 = few ? a.B : 0; b0 < a.B && base <= x[1]; b0 += NT) {
    const int b = b0 + tid;
    if (b0 > 0) mine = paged_seq_units(a, b, RT, KT);
    long long here = all;
    const long long s = a.B <= NT ? before : base + paged_block_scan<NT>(mine, sh, here);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const unsigned hit = __ballot_sync(0xffffffffu, mine > 0 && x[i] >= s && x[i] < s + mine);
      if (hit) {
        const int src = __ffs(hit) - 1;
        const PagedLoc l = paged_find(a, __shfl_sync(0xffffffffu, b, src), __shfl_sync(0xffffffffu, s, src), x[i], tol, RT, KT);
        if ((tid & 31) == 0) sh.loc[i] = l;
      }
    }
    base += here;
  }
  __syncthreads();
  if (tid == 0) {
    // the records of an item that runs end in: those of the run in front of the first such end (its last) and of the runs behind, up to the one
    // that has the item's end (their first)
    const PagedLoc l = sh.loc[0];
    PagedJoin j{};
    if (l.off > 0 && l.off < l.units && split.begin(c - 1) - l.s <= max(tol, (long long)a.start)) {
      const PagedSeq q = paged_seq(a, l.b);
      j.records = 2;
      while (c + j.records - 1 < runs && l.s + a.start + l.units - split.begin(c + j.records - 1) > tol) ++j.records;
      j.row0 = q.row0;
      j.p0 = l.t * RT;
      j.pairs = min(RT, q.n * a.G - l.t * RT);
      j.h = l.h;
    }
    a.joins[2 * c] = make_int4(j.records, j.row0, j.p0, j.pairs);
    a.joins[2 * c + 1] = make_int4(j.h, 0, 0, 0);
  }
  return true;
}
// Items of a run, one after the other: begin(), then next() for each, which is false when there is none left, and step() behind it.  [k0, k1): the key tiles of the
// item that are this run's.
struct PagedRun {
  int b, t, h, tiles;
  int k0, k1;            // key tiles
  bool first, last;      // whether the run has the item's first / last unit
  PagedSeq seq;
  int off;
  __device__ __forceinline__ void begin(const PagedArgs& a, const PagedPlanShared& sh, int RT) {
    const PagedLoc& l = sh.loc[0];
    b = l.b; t = l.t; h = l.h; off = l.off;
    seq = paged_seq(a, b);
    tiles = (seq.n * a.G + RT - 1) / RT;
    if (off == l.units) step(a);
  }
  __device__ __forceinline__ void step(const PagedArgs& a) {
    off = 0;
    if (++h < a.Hkv) return;
    h = 0;
    ++t;
  }
  // the next item with work of this run; false: none
  __device__ __forceinline__ bool next(const PagedArgs& a, const PagedPlanShared& sh, int RT, int KT) {
    while (t >= tiles) {
      if (++b >= a.B) return false;
      t = 0;
      seq = paged_seq(a, b);
      tiles = (seq.n * a.G + RT - 1) / RT;
    }
    const PagedLoc& e = sh.loc[1];
    if (b > e.b) return false;
    const PagedTile p = paged_tile(a, seq, t, RT, KT);
    int stop = p.units;
    if (b == e.b) {
      if (t > e.t || (t == e.t && h > e.h)) return false;
      if (t == e.t && h == e.h) stop = e.off;
    }
    if (off >= stop) return false;
    first = off == 0;
    last = stop == p.units;
    k0 = p.k0 + off;
    k1 = p.k0 + stop;
    return true;
  }
};

int launch_paged_combine(int device, int dtype, const PagedArgs& a, int RT, int ctas, cudaStream_t s);
// kernels for 16-bit types and head sizes 64 and 128: rows of few pairs per sequence on mma.sync, chunks on tcgen05
int paged_map(CUtensorMap* map, int dtype, const void* base, const PagedArgs& a, int keys);
int launch_paged_mma(int device, DeviceState* st, int dtype, PagedArgs a, int RT, cudaStream_t s);
bool paged_tc_strides(const PagedArgs& a);
int launch_paged_tc(int device, DeviceState* st, int dtype, PagedArgs a, cudaStream_t s);

}  // namespace tsb
