// Attention of packed rows over a paged key / value cache: what its kernels share.
//
// Rows of several sequences lie one after the other (starts[b] .. starts[b + 1]); those of sequence b are the last ones of its lens[b] cached tokens,
// so row i of n sees the keys j <= lens[b] - n + i, and with a window only j > that position - window.  Key j lies in page table[b][j / page]
// at place j % page.  Entries that name no page hide their keys, and a row that sees no key is written as zeros.
//
// Work: an item is (sequence, tile of RT of its n * G (query, head) pairs, KV head), a unit a tile of KT of the item's keys.  What is known on the
// host are bounds only (a captured call is replayed with other lengths), so each CTA reads the lengths, numbers all units and takes an equal run of
// them: one sequence of any length, or sequences of very different lengths, keep every SM busy.  A run may begin or end inside an item; such a
// CTA leaves its maximum, sum and accumulator in the workspace and paged_combine_kernel joins them in the order of the runs (the same
// order whatever CTA ends first).  Ends within an eighth of a run of an item's end are moved there, since a record costs about a unit to write and to read.
#pragma once
#include "kernels.cuh"

namespace tsb {

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
  float c;                         // scale * log2(e)
  int window;                      // 0: none
  float* part;                     // records: paged_record_floats() each, two per CTA
  int min_units;                   // no run is shorter
  unsigned wait_limit;
  int* error;
};

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
  s.len = max(a.lens[b], 0);
  return s;
}
struct PagedTile {
  int k0, units;   // first key tile, how many
};
__device__ __forceinline__ PagedTile paged_tile(const PagedArgs& a, const PagedSeq& s, int t, int RT, int KT) {
  const int p1 = min(s.n * a.G, (t + 1) * RT) - 1;
  const int first = s.len - s.n + t * RT / a.G, last = s.len - s.n + p1 / a.G;   // positions of the tile
  const int hi = min(last + 1, a.max_blocks << a.page_shift);
  const int lo = a.window > 0 && a.window <= first ? first - a.window + 1 : 0;
  PagedTile r;
  r.k0 = lo / KT;
  r.units = max(1, (hi + KT - 1) / KT - r.k0);   // a tile without keys is still written
  return r;
}
// where a run begins or ends: unit `off` (0 .. units) of an item whose first unit is number `s` of all
struct PagedLoc {
  int b, t, h, off, units;
  long long s;
};
struct PagedPlanShared {
  long long warp[32], base[2];
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
__device__ __forceinline__ long long paged_seq_units(const PagedArgs& a, int b, int RT, int KT) {
  if (b >= a.B) return 0;
  const PagedSeq s = paged_seq(a, b);
  const int tiles = (s.n * a.G + RT - 1) / RT;
  long long u = 0;
  for (int t = 0; t < tiles; ++t) u += paged_tile(a, s, t, RT, KT).units;
  return u * a.Hkv;
}
// Run `c` of the plan: sh.loc[0] and sh.loc[1] where it begins and ends.  Returns whether there is such a run.  `all` / `runs`: units and runs of
// the whole call.  All threads of the CTA.
template <int NT, int RT, int KT>
__device__ __forceinline__ bool paged_locate(const PagedArgs& a, int c, int ctas, PagedPlanShared& sh, long long& all, int& runs) {
  const int tid = threadIdx.x;
  long long mine = paged_seq_units(a, tid, RT, KT), total = mine;
  for (int b = tid + NT; b < a.B; b += NT) total += paged_seq_units(a, b, RT, KT);
  paged_block_scan<NT>(total, sh, all);
  if (all == 0) return false;
  const long long most = all / a.min_units;
  runs = (int)(most < 1 ? 1 : (most < ctas ? most : ctas));
  if (c >= runs) return false;
  const long long tol = all / runs / 8;
  const long long x[2] = {all * c / runs, all * (c + 1) / runs};
  if (tid == 0) sh.loc[1] = PagedLoc{a.B, 0, 0, 0, 0, all};
  long long base = 0;
  for (int b0 = 0; b0 < a.B && base <= x[1]; b0 += NT) {
    const int b = b0 + tid;
    if (b0 > 0) mine = paged_seq_units(a, b, RT, KT);
    long long here;
    const long long s = base + paged_block_scan<NT>(mine, sh, here);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (mine > 0 && x[i] >= s && x[i] < s + mine) {
        const PagedSeq q = paged_seq(a, b);
        long long at = s;
        for (int t = 0;; ++t) {
          const int u = paged_tile(a, q, t, RT, KT).units;
          if (x[i] < at + (long long)u * a.Hkv) {
            const int h = (int)((x[i] - at) / u);
            PagedLoc l{b, t, h, (int)(x[i] - at - (long long)h * u), u, at + (long long)h * u};
            if (l.off <= tol) l.off = 0;
            else if (u - l.off <= tol) l.off = u;
            sh.loc[i] = l;
            break;
          }
          at += (long long)u * a.Hkv;
        }
      }
    base += here;
  }
  __syncthreads();
  return true;
}
// Items of a run, one after the other.  done() when there is none left; [k0, k1) the key tiles of the item that are this run's.
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
  __device__ __forceinline__ void step(const PagedArgs& a, int RT = 0) {
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

int launch_paged_combine(int device, int dtype, const PagedArgs& a, int RT, int KT, int ctas, cudaStream_t s);
// kernels for 16-bit types and head sizes 64 and 128: rows of few pairs per sequence on mma.sync, chunks on tcgen05
int launch_paged_mma(int device, DeviceState* st, int dtype, PagedArgs a, int pairs, cudaStream_t s);
int launch_paged_tc(int device, DeviceState* st, int dtype, PagedArgs a, cudaStream_t s);

}  // namespace tsb
