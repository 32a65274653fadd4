// A key / value cache in pages: the plan that hands pages out and maps rows to places, the norm / rotation / append of new rows, and the attention over
// the pages (kernel for every type and head size; attn_paged_mma.cu and attn_paged_tc.cu for 16-bit types and head sizes 64 and 128).
#include <cfloat>
#include <cmath>

#include "paged.cuh"

namespace tsb {

// ------------------------------------------------------------------------------------------------------------------------ plan
// want = ceil((cached + fresh) / page);  need = max(0, want - held), taken from the top of the stack of free pages in the order of the sequences;
// held - want pages of a sequence that wants fewer go back, so that taking and giving back leaves the stack as it was;
// starts = exclusive sum of the granted rows;  slot(row) = table[pos / page] * page + pos % page.
// What bounds it: latency (three block scans, a few hundred KB at most; 8 sequences 5.4 us, 1024 sequences with 92500 rows 13, where the search of each row's sequence takes half).  Sums of rows and pages over sequences are 64-bit: their bounds are the caller's.
struct PlanArgs {
  const int *cached, *fresh;
  int B, page_shift, max_blocks, num_pages, rows;
  int* table;
  int64_t table_stride;
  int *held, *free_pages, *free_count, *lens, *starts, *slots, *positions;
};
constexpr int kPlanThreads = 1024, kPlanMaxB = 8192;

__device__ __forceinline__ long long plan_scan(long long v, long long* warps, long long& all) {   // exclusive, kPlanThreads
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  long long x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) warps[w] = x;
  __syncthreads();
  long long y = warps[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long z = __shfl_up_sync(0xffffffffu, y, o);
    if (lane >= o) y += z;
  }
  all = __shfl_sync(0xffffffffu, y, 31);
  const long long before = __shfl_sync(0xffffffffu, y, w > 0 ? w - 1 : 0);
  return (w > 0 ? before : 0) + x - v;
}
// the last i of [0, n) with first[i] <= v (first ascending, first[0] <= v)
__device__ __forceinline__ int plan_find(const int* first, int n, int v) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int m = (lo + hi) >> 1;
    if (first[m] <= v) lo = m;
    else hi = m;
  }
  return lo;
}

// One cluster.  Every CTA makes the scans for itself; the pages to move and the rows are shared out over all threads.
__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(PlanArgs a, int ctas) {
  extern __shared__ int plan_sm[];
  __shared__ long long warps[32];
  __shared__ int granted;
  const int B = a.B, tid = threadIdx.x, page = 1 << a.page_shift;
  // of every sequence: pages held before, cached tokens, pages kept; number of its first new row, first page taken, first page given back
  int *have_s = plan_sm, *old_s = have_s + B, *keep_s = old_s + B, *row_s = keep_s + B, *take_s = row_s + B, *give_s = take_s + B;
  const int avail = min(max(*a.free_count, 0), a.num_pages);
  if (tid == 0) granted = 0;
  long long rows = 0, asked = 0, moved = 0;   // over the sequences so far; moved: pages taken in the upper, given back in the lower half
  for (int b0 = 0; b0 < B; b0 += kPlanThreads) {
    const int b = b0 + tid;
    int old = 0, fresh = 0, have = 0;
    if (b < B) {
      old = a.cached[b];
      fresh = a.fresh[b];
      have = min(max(a.held[b], 0), a.max_blocks);
    }
    const bool fits = b < B && old >= 0 && fresh >= 0 && (long long)old + fresh <= ((long long)a.max_blocks << a.page_shift);
    int now = fits ? fresh : 0;
    const int kept = fits ? (int)(((long long)old + page - 1) >> a.page_shift) : have;
    const int want = fits ? (int)(((long long)old + now + page - 1) >> a.page_shift) : have;
    int need = now > 0 ? max(0, want - have) : 0;
    long long all;
    const long long need_before = asked + plan_scan(need, warps, all);
    asked += all;
    if (need > 0 && need_before + need > avail) now = 0;
    const long long rows_before = rows + plan_scan(now, warps, all);
    rows += all;
    if (rows_before + now > a.rows) now = 0;   // nor is any row behind granted: the sums only grow
    if (now == 0) need = 0;
    const int keep = now > 0 ? want : min(have, kept);
    const long long move = ((long long)need << 32) | (unsigned)max(0, have - keep);
    const long long move_before = moved + plan_scan(move, warps, all);
    moved += all;
    if (b < B) {
      have_s[b] = have;
      old_s[b] = old;
      keep_s[b] = keep;
      row_s[b] = (int)min(rows_before, (long long)a.rows);
      take_s[b] = (int)(move_before >> 32);
      give_s[b] = (int)(move_before & 0xffffffffLL);
      if (now > 0) atomicMax(&granted, (int)(rows_before + now));
    }
  }
  __syncthreads();
  const int total = granted, taken = (int)(moved >> 32), given = (int)(moved & 0xffffffffLL);
  for (int b = tid; b < B; b += kPlanThreads) row_s[b] = min(row_s[b], total);
  const int first = (int)blockIdx.x * kPlanThreads + tid, step = ctas * kPlanThreads;
  for (int m = first; m < taken; m += step) {
    const int b = plan_find(take_s, B, m);
    a.table[b * a.table_stride + have_s[b] + (m - take_s[b])] = a.free_pages[avail - 1 - m];
  }
  cluster_sync();   // all that other CTAs read of the state has been read, and the pages taken are in the table
  const int height = avail - taken + given;
  for (int m = first; m < given; m += step) {
    const int b = plan_find(give_s, B, m), at = height - 1 - m;
    int* entry = a.table + b * a.table_stride + keep_s[b] + (m - give_s[b]);
    if (at >= 0 && at < a.num_pages) a.free_pages[at] = *entry;
    *entry = -1;
  }
  for (int b = first; b <= B; b += step) {
    a.starts[b] = b < B ? row_s[b] : total;
    if (b == B) continue;
    const int now = (b + 1 < B ? row_s[b + 1] : total) - row_s[b];
    a.held[b] = keep_s[b];
    a.lens[b] = old_s[b] + now;
  }
  if (first == 0) *a.free_count = min(height, a.num_pages);
  for (int r = first; r < a.rows; r += step) {
    int pos = -1, slot = -1;
    if (r < total) {
      const int b = plan_find(row_s, B, r);
      pos = old_s[b] + (r - row_s[b]);
      const int entry = a.table[b * a.table_stride + (pos >> a.page_shift)];
      if (entry >= 0 && entry < a.num_pages) slot = entry * page + (pos & (page - 1));
    }
    a.slots[r] = slot;
    a.positions[r] = pos;
  }
}

// ------------------------------------------------------------------------------------------------------------------------ norm, rotation, append
//   y = x / sqrt(mean(x^2) + eps) * w;   (y_a, y_b) -> (y_a cos - y_b sin, y_b cos + y_a sin),   angle = position * base^(-2 i / rot)
// for every query and key head of a row; queries go to `out`, keys and values to the row's place in the cache.  Norm and rotation in fp32, rounded once;
// angles in 64 bits (fp32 loses the angle of position 10^5 from the third digit on) as half turns, which are brought to [-1, 1] before they are rounded to fp32 for the sine
// and cosine: off by up to pi 2^-25, which 16-bit results do not show (the rotation's own fp32 sums are off by as much), and which is turned back for fp32.
// L = 2^k lanes hold a head, 8 C elements each; the cos / sin of a row are made once per CTA.  What bounds it: issue slots and bytes about equally.  Of 16384 rows
// of 32 + 16 heads of 64 in bf16 (201 MB, 30.8 us at the rate of a copy): C = 1, six CTAs per SM 54.5 us; C = 2, four 44.4 (five 49.1, three 47.6); C = 4, two 63.
// Rows first and heads second, with a head's addresses and weights kept in registers, is slower (61: a warp's lines lie in two places).
struct RopePagedArgs {
  void* out;
  const void *q, *k, *v, *q_norm, *k_norm;
  int o_row, o_head, q_row, q_head, k_row, k_head, v_row, v_head;   // 32 bits: one multiplication for an address
  float eps;
  const int *positions, *slots;
  int rows, H, Hkv, hd, rot, style;   // style 0: no rotation, 1: pairs (2i, 2i + 1), 2: pairs (i, i + rot / 2)
  double first, ratio;                // half turns per position of pair 0; of pair i: first * ratio^i
  void *K, *V;
  int c_page, c_head, c_tok;
  int num_pages, page_shift;
  int rows_here;                      // rows per CTA
};
constexpr int kRopeThreads = 256, kRopeMaxHd = 256, kRopeTurns = 1024;

// eight elements as they lie in memory, four at p0 and four at p1: WIDE by 8 or 16 bytes, else one by one
template <typename T, bool WIDE>
struct Eight {
  static constexpr int N = WIDE ? (sizeof(T) == 4 ? 8 : 4) : 8;   // registers
  uint32_t r[N];
  template <bool WHOLE>   // p1 = p0 + 4
  __device__ __forceinline__ void load(const T* p0, const T* p1) {
    if constexpr (!WIDE) {
#pragma unroll
      for (int e = 0; e < 4; ++e) r[e] = __float_as_uint(to_f<T>(p0[e])), r[4 + e] = __float_as_uint(to_f<T>(p1[e]));
    } else if constexpr (N == 8) {
      const uint4 x = *reinterpret_cast<const uint4*>(p0), y = *reinterpret_cast<const uint4*>(p1);
      r[0] = x.x; r[1] = x.y; r[2] = x.z; r[3] = x.w;
      r[4] = y.x; r[5] = y.y; r[6] = y.z; r[7] = y.w;
    } else if constexpr (WHOLE) {
      const uint4 x = *reinterpret_cast<const uint4*>(p0);
      r[0] = x.x; r[1] = x.y; r[2] = x.z; r[3] = x.w;
    } else {
      const uint2 x = *reinterpret_cast<const uint2*>(p0), y = *reinterpret_cast<const uint2*>(p1);
      r[0] = x.x; r[1] = x.y; r[2] = y.x; r[3] = y.y;
    }
  }
  __device__ __forceinline__ void get(float* f) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (N == 8) {
        f[i] = __uint_as_float(r[i]);
      } else {
        const float2 t = Pair16<T>::get(r[i]);
        f[2 * i] = t.x;
        f[2 * i + 1] = t.y;
      }
    }
  }
  template <bool WHOLE>
  static __device__ __forceinline__ void store(T* p0, T* p1, const float* f) {
    if constexpr (!WIDE) {
#pragma unroll
      for (int e = 0; e < 4; ++e) p0[e] = from_f<T>(f[e]), p1[e] = from_f<T>(f[4 + e]);
    } else if constexpr (N == 8) {
      *reinterpret_cast<float4*>(p0) = make_float4(f[0], f[1], f[2], f[3]);
      *reinterpret_cast<float4*>(p1) = make_float4(f[4], f[5], f[6], f[7]);
    } else if constexpr (WHOLE) {
      *reinterpret_cast<uint4*>(p0) = make_uint4(Pair16<T>::put(f[0], f[1]), Pair16<T>::put(f[2], f[3]), Pair16<T>::put(f[4], f[5]), Pair16<T>::put(f[6], f[7]));
    } else {
      *reinterpret_cast<uint2*>(p0) = make_uint2(Pair16<T>::put(f[0], f[1]), Pair16<T>::put(f[2], f[3]));
      *reinterpret_cast<uint2*>(p1) = make_uint2(Pair16<T>::put(f[4], f[5]), Pair16<T>::put(f[6], f[7]));
    }
  }
};

// STYLE as in RopePagedArgs; LT: lanes of a head, 0: as many as its size needs; C: pieces of eight elements per lane, L apart
template <typename T, bool WIDE, int STYLE, int LT, int C>
__global__ void __launch_bounds__(kRopeThreads, 4) qk_norm_rope_paged_kernel(const __grid_constant__ RopePagedArgs a) {
  constexpr bool WHOLE = STYLE != 2;
  __shared__ __align__(16) float wq[kRopeMaxHd], wk[kRopeMaxHd];
  __shared__ __align__(16) float2 turn[kRopeTurns];
  __shared__ int place[kRopeTurns];
  const int tid = threadIdx.x, half = a.rot / 2;
  // angles of a row, filled up to whole fours of pairs with turns by nothing; a pass: as many rows as there is room for
  const int slots = STYLE ? (half + 3) / 4 * 4 : 0, rows_pass = STYLE ? kRopeTurns / slots : kRopeTurns;
  // a thread makes the angles of one pair, of every (256 / slots)-th row
  const int turn_rows = STYLE ? kRopeThreads / slots : 1, ar = STYLE ? tid / slots : 0, ai = STYLE ? tid - ar * slots : 0;
  const double rate = STYLE && ai < half ? a.first * pow(a.ratio, (double)ai) : 0.0;   // half turns per position
  for (int e = tid; e < a.hd; e += kRopeThreads) {
    wq[e] = a.q_norm ? to_f<T>(reinterpret_cast<const T*>(a.q_norm)[e]) : 1.0f;
    wk[e] = a.k_norm ? to_f<T>(reinterpret_cast<const T*>(a.k_norm)[e]) : 1.0f;
  }
  int L = LT ? LT : 1;
  if (LT == 0)
    while (L * C * 8 < a.hd) L <<= 1;
  const int li = tid & (L - 1), per = kRopeThreads / L, heads = a.H + 2 * a.Hkv;
  const bool norms = a.q_norm || a.k_norm;
  const float inv_hd = 1.0f / (float)a.hd;
  // C times, a lane has four elements and the four that they turn with (pairs (i, i + rot / 2)), or eight neighbours
  bool on[C], turned[C];
  int e0[C], e1[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int i = c * L + li;
    on[c] = i * 8 < a.hd;
    turned[c] = STYLE && i * 8 < a.rot;
    e0[c] = STYLE == 2 && turned[c] ? i * 4 : i * 8;
    e1[c] = STYLE == 2 && turned[c] ? half + i * 4 : e0[c] + 4;
  }
  const int places = a.num_pages << a.page_shift;
  auto place_of = [&](int row) {   // in the cache, or -1
    const int slot = a.slots[row];
    return slot >= 0 && slot < places ? slot : -1;
  };
  const int row_first = (int)blockIdx.x * a.rows_here, row_end = row_first + min(a.rows_here, a.rows - row_first);
  for (int row0 = row_first; row0 < row_end; row0 += rows_pass) {
    const int n = min(rows_pass, row_end - row0);
    // (row, head) pairs go round the groups of L lanes; the next one is on its way while one is turned
    const int stride = per * (int)gridDim.y, passes = (n * heads + stride - 1) / stride;
    int head = (int)blockIdx.y * per + tid / L, r = 0;
    Eight<T, WIDE> ahead[C];
    int slot = -1;
    auto fetch = [&](bool known) {
      while (head >= heads) {
        head -= heads;
        ++r;
      }
      slot = r >= n ? -1 : known ? place[r] : place_of(row0 + r);
      if (slot < 0) return;
      const int64_t row = row0 + r;
      const T* p = head < a.H ? reinterpret_cast<const T*>(a.q) + row * a.q_row + (int64_t)head * a.q_head
                              : (head < a.H + a.Hkv ? reinterpret_cast<const T*>(a.k) + row * a.k_row + (int64_t)(head - a.H) * a.k_head
                                                    : reinterpret_cast<const T*>(a.v) + row * a.v_row + (int64_t)(head - a.H - a.Hkv) * a.v_head);
#pragma unroll
      for (int c = 0; c < C; ++c)
        if (on[c]) ahead[c].template load<WHOLE>(p + e0[c], p + e1[c]);
    };
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < Eight<T, WIDE>::N; ++i) ahead[c].r[i] = 0u;
    fetch(false);   // of the first pass before the angles are made
    __syncthreads();   // the pass before is done with both
    if (STYLE && ar < turn_rows)
      for (int r = ar; r < n; r += turn_rows) {
        double x = (double)a.positions[row0 + r] * rate;
        x -= 2.0 * rint(0.5 * x);
        const float near = (float)x;
        float s, c;
        sincospif(near, &s, &c);
        if constexpr (sizeof(T) == 4) {   // turned on by what the rounding took from the angle, below pi 2^-25
          const float d = (float)((x - (double)near) * 3.14159265358979323846), t = s;
          s = fmaf(c, d, s);
          c = fmaf(-t, d, c);
        }
        turn[r * slots + ai] = make_float2(c, s);
      }
    for (int r = tid; r < n; r += kRopeThreads) place[r] = place_of(row0 + r);
    __syncthreads();
#pragma unroll 1
    for (int pass = 0; pass < passes; ++pass) {
      float x[C][8];
#pragma unroll
      for (int c = 0; c < C; ++c) ahead[c].get(x[c]);
      const int head_now = head, r_now = r, slot_now = slot;
      const bool is_q = head_now < a.H, is_v = head_now >= a.H + a.Hkv;
      head += stride;
      fetch(true);
      if (norms) {
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < 8 * C; ++e) ss += x[e / 8][e & 7] * x[e / 8][e & 7];
        if constexpr (LT > 0) {
#pragma unroll
          for (int o = LT / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        } else {
          for (int o = L >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        }
        if (!is_v && (is_q ? a.q_norm : a.k_norm)) {
          const float f = rsqrtf(ss * inv_hd + a.eps);   // off by 2^-22.9 of itself at most: the fp32 roundings of a root and a quotient would be 2^-23
          const float* w = is_q ? wq : wk;
#pragma unroll
          for (int c = 0; c < C; ++c)
            if (C == 1 || on[c]) {
              const float4 w0 = *reinterpret_cast<const float4*>(w + e0[c]), w1 = *reinterpret_cast<const float4*>(w + e1[c]);
              x[c][0] *= f * w0.x; x[c][1] *= f * w0.y; x[c][2] *= f * w0.z; x[c][3] *= f * w0.w;
              x[c][4] *= f * w1.x; x[c][5] *= f * w1.y; x[c][6] *= f * w1.z; x[c][7] *= f * w1.w;
            }
        }
      }
      if (slot_now >= 0) {
        if (STYLE && !is_v)
#pragma unroll
          for (int c = 0; c < C; ++c)
            if (turned[c]) {
              const float4* t = reinterpret_cast<const float4*>(turn + r_now * slots + (c * L + li) * 4);
              const float4 t0 = t[0], t1 = t[1];
              const float co[4] = {t0.x, t0.z, t1.x, t1.z}, si[4] = {t0.y, t0.w, t1.y, t1.w};
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                float &u = x[c][STYLE == 2 ? i : 2 * i], &v = x[c][STYLE == 2 ? 4 + i : 2 * i + 1];
                const float y0 = u * co[i] - v * si[i], y1 = v * co[i] + u * si[i];
                u = y0;
                v = y1;
              }
            }
        T* dst;
        if (is_q) dst = reinterpret_cast<T*>(a.out) + (int64_t)(row0 + r_now) * a.o_row + (int64_t)head_now * a.o_head;
        else
          dst = reinterpret_cast<T*>(is_v ? a.V : a.K) + (int64_t)(slot_now >> a.page_shift) * a.c_page + (int64_t)(slot_now & ((1 << a.page_shift) - 1)) * a.c_tok +
                (int64_t)(head_now - (is_v ? a.H + a.Hkv : a.H)) * a.c_head;
#pragma unroll
        for (int c = 0; c < C; ++c)
          if (on[c]) Eight<T, WIDE>::template store<WHOLE>(dst + e0[c], dst + e1[c], x[c]);
      }
    }
  }
}

template <typename T, bool WIDE, int STYLE>
static void launch_rope_paged_l(const RopePagedArgs& a, dim3 grid, cudaStream_t s) {
  constexpr int C = WIDE && sizeof(T) == 2 ? 2 : 1;   // fp32: two pieces are no faster (7.8 us for 2036 rows of 8 + 16 heads of 64)
  if (WIDE && a.hd > 32 && a.hd <= 64) qk_norm_rope_paged_kernel<T, WIDE, STYLE, WIDE ? 8 / C : 0, C><<<grid, kRopeThreads, 0, s>>>(a);
  else if (WIDE && a.hd > 64 && a.hd <= 128) qk_norm_rope_paged_kernel<T, WIDE, STYLE, WIDE ? 16 / C : 0, C><<<grid, kRopeThreads, 0, s>>>(a);
  else qk_norm_rope_paged_kernel<T, WIDE, STYLE, 0, 1><<<grid, kRopeThreads, 0, s>>>(a);
}
template <typename T, bool WIDE>
static void launch_rope_paged(const RopePagedArgs& a, dim3 grid, cudaStream_t s) {
  if (a.style == 0) launch_rope_paged_l<T, WIDE, 0>(a, grid, s);
  else if (a.style == 1) launch_rope_paged_l<T, WIDE, 1>(a, grid, s);
  else launch_rope_paged_l<T, WIDE, 2>(a, grid, s);
}

// ------------------------------------------------------------------------------------------------------------------------ attention, every type
// Four warps of RW rows; a tile of 32 keys and values is brought to shared memory by cp.async while the one before is used (places
// that hold no visible key, behind the sequence's end, in front of every window or in no page, are filled with zeros, whatever the cache has there).  Scores: a lane per key; values: a lane per hd / 32 elements.
// fp32 throughout: the products run on the FMA pipe, which is what bounds chunks; single tokens are bound by bytes.  It serves what the kernels for tensor cores
// do not: fp32 tokens, other head sizes, strides that no tensor map takes (8 fp32 tokens over 6000 keys, 8 / 8 heads of 64: 17.6 us; 8 fp16 tokens over up to 4096, heads of 96: 47.5).
constexpr int kFmaThreads = 128, kFmaKeys = 32;
template <typename T>
constexpr int fma_row_bytes(int NH) { return NH * 32 * (int)sizeof(T) + 16; }   // odd in units of 16 bytes: lanes of neighbouring keys meet no bank twice
template <typename T>
constexpr int fma_smem(int NH, int RW) { return 4 * kFmaKeys * fma_row_bytes<T>(NH) + 4 * RW * NH * 32 * 4; }

template <typename T, int NH, int RW>
__global__ void __launch_bounds__(kFmaThreads) paged_fma_kernel(const __grid_constant__ PagedArgs a) {
  constexpr int RT = 4 * RW, KT = kFmaKeys, D = NH * 32, RB = fma_row_bytes<T>(NH), EV = 16 / (int)sizeof(T);
  extern __shared__ __align__(16) unsigned char fma_sm[];
  __shared__ PagedPlanShared plan;
  float* qs = reinterpret_cast<float*>(fma_sm + 4 * KT * RB);   // [RT][D]
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  pdl_trigger();
  long long all;
  int runs;
  if (!paged_locate<kFmaThreads, RT, KT>(a, blockIdx.x, gridDim.x, plan, all, runs)) return;
  const int pieces = a.hd / EV, mask = (1 << a.page_shift) - 1;
  PagedRun run;
  run.begin(a, plan, RT);
  for (; run.next(a, plan, RT, KT); run.step(a)) {
    const PagedSeq& s = run.seq;
    const int p0 = run.t * RT, pairs = s.n * a.G;
    const int cap = min(s.len, a.max_blocks << a.page_shift), front = paged_front(a, s, p0);
    const int* table = a.table + run.b * a.table_stride;
    auto fetch = [&](int kt) {
      unsigned char* ks = fma_sm + (kt & 1) * 2 * KT * RB;
      for (int i = tid; i < KT * (D / EV); i += kFmaThreads) {
        const int k = i / (D / EV), e = i % (D / EV), j = kt * KT + k;
        bool there = j < cap && j >= front && e < pieces;
        const int page = there ? table[j >> a.page_shift] : 0;
        there = there && page >= 0 && page < a.num_pages;
        const int64_t at = there ? page * a.c_page + run.h * a.c_head + (j & mask) * a.c_tok + e * EV : 0;
        paged_cp16(ks + k * RB + e * 16, reinterpret_cast<const T*>(a.K) + at, there);
        paged_cp16(ks + (KT + k) * RB + e * 16, reinterpret_cast<const T*>(a.V) + at, there);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    __syncthreads();   // the item before has been read
    fetch(run.k0);
    for (int i = tid; i < RT * D; i += kFmaThreads) {
      const int r = i / D, e = i % D, p = p0 + r;
      float v = 0.0f;
      if (p < pairs && e < a.hd) v = to_f<T>(reinterpret_cast<const T*>(a.q)[(int64_t)(s.row0 + a.by_G(p)) * a.q_row + (run.h * a.G + (p - a.by_G(p) * a.G)) * a.q_head + e]) * a.c;
      qs[i] = v;
    }
    float m[RW], l[RW], acc[RW][NH];
    int lo[RW], hi[RW];
#pragma unroll
    for (int r = 0; r < RW; ++r) {
      m[r] = -INFINITY;
      l[r] = 0.0f;
      const int p = p0 + w * RW + r, pos = s.len - s.n + a.by_G(p);
      hi[r] = p < pairs ? min(pos + 1, cap) : 0;
      lo[r] = a.window > 0 ? pos - a.window + 1 : 0;
#pragma unroll
      for (int e = 0; e < NH; ++e) acc[r][e] = 0.0f;
    }
    for (int kt = run.k0; kt < run.k1; ++kt) {
      if (kt + 1 < run.k1) fetch(kt + 1);
      else asm volatile("cp.async.commit_group;" ::: "memory");
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      __syncthreads();
      const unsigned char* ks = fma_sm + (kt & 1) * 2 * KT * RB;
      const int j = kt * KT + lane;
      bool seen = j < cap;
      if (seen) {
        const int page = table[j >> a.page_shift];
        seen = page >= 0 && page < a.num_pages;
      }
      float sc[RW];
#pragma unroll
      for (int r = 0; r < RW; ++r) sc[r] = 0.0f;
#pragma unroll 4
      for (int e = 0; e < D / EV; ++e) {
        float kf[EV];
        if constexpr (sizeof(T) == 4) {
          const float4 k4 = *reinterpret_cast<const float4*>(ks + lane * RB + e * 16);
          kf[0] = k4.x; kf[1] = k4.y; kf[2] = k4.z; kf[3] = k4.w;
        } else {
          Eight<T, true> k8;
          k8.template load<true>(reinterpret_cast<const T*>(ks + lane * RB + e * 16), nullptr);
          k8.get(kf);
        }
#pragma unroll
        for (int r = 0; r < RW; ++r) {
#pragma unroll
          for (int g = 0; g < EV; g += 4) {
            const float4 q4 = *reinterpret_cast<const float4*>(qs + (w * RW + r) * D + e * EV + g);
            sc[r] += q4.x * kf[g] + q4.y * kf[g + 1] + q4.z * kf[g + 2] + q4.w * kf[g + 3];
          }
        }
      }
#pragma unroll
      for (int r = 0; r < RW; ++r) {
        if (!(seen && j < hi[r] && j >= lo[r])) sc[r] = -INFINITY;
        const float up = fmaxf(m[r], warp_max(sc[r]));
        const float from = fmaxf(up, -FLT_MAX);   // no key seen yet: every weight is exp2(-inf)
        const float f = exp2f(m[r] - from);
        sc[r] = exp2f(sc[r] - from);
        m[r] = up;
        l[r] = l[r] * f + sc[r];   // this lane's keys
#pragma unroll
        for (int e = 0; e < NH; ++e) acc[r][e] *= f;
      }
#pragma unroll 4
      for (int k = 0; k < KT; ++k) {
        float vf[NH];
        const T* v = reinterpret_cast<const T*>(ks + (KT + k) * RB) + lane * NH;
#pragma unroll
        for (int e = 0; e < NH; ++e) vf[e] = to_f<T>(v[e]);
#pragma unroll
        for (int r = 0; r < RW; ++r) {
          const float p = __shfl_sync(0xffffffffu, sc[r], k);
#pragma unroll
          for (int e = 0; e < NH; ++e) acc[r][e] += p * vf[e];
        }
      }
      __syncthreads();
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    const bool whole = run.first && run.last;
    float* rec = a.part + (2 * (int64_t)blockIdx.x + (run.first ? 1 : 0)) * paged_record_floats(RT, a.hd);
#pragma unroll
    for (int r = 0; r < RW; ++r) {
      const float sum = warp_sum(l[r]);
      const int row = w * RW + r, p = p0 + row;
      if (p >= pairs) continue;
      if (whole) {
        T* o = reinterpret_cast<T*>(a.out) + (int64_t)(s.row0 + a.by_G(p)) * a.o_row + (run.h * a.G + (p - a.by_G(p) * a.G)) * a.o_head;
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
        for (int e = 0; e < NH; ++e)
          if (lane * NH + e < a.hd) o[lane * NH + e] = from_f<T>(acc[r][e] * inv);
      } else {
        if (lane == 0) {
          rec[2 * row] = m[r];
          rec[2 * row + 1] = sum;
        }
#pragma unroll
        for (int e = 0; e < NH; ++e)
          if (lane * NH + e < a.hd) rec[2 * RT + row * a.hd + lane * NH + e] = acc[r][e];
      }
    }
  }
}

// fp32 chunks: 64 rows and 64 keys at a time, a thread has 4 x 4 scores and 4 x D / 16 outputs (four elements of a row from shared memory feed 16 products).  What
// bounds it: the FMA pipe and shared memory, about even.  2 x 512 rows over 3000, 32 / 8 heads of 128: 991 us (47 TFLOP/s with what the mask leaves out); 1090 with one product to an
// instruction, 1890 with 16 rows and a lane per key (shared memory alone).
constexpr int kTileThreads = 256, kTileRows = 64, kTileKeys = 64;
// d += x y of two pairs: one instruction
__device__ __forceinline__ void paged_fma2(float2& d, float2 x, float2 y) {
  uint64_t a, b, c;
  asm("mov.b64 %0, {%1, %2};" : "=l"(a) : "f"(x.x), "f"(x.y));
  asm("mov.b64 %0, {%1, %2};" : "=l"(b) : "f"(y.x), "f"(y.y));
  asm("mov.b64 %0, {%1, %2};" : "=l"(c) : "f"(d.x), "f"(d.y));
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(c) : "l"(a), "l"(b));
  asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(c));
}
template <int D>
constexpr int tile_smem() { return (kTileRows * (D + 4) + 2 * kTileKeys * (D + 4) + 2 * kTileKeys * D + kTileRows * (kTileKeys + 4)) * 4; }

template <int D>
__global__ void __launch_bounds__(kTileThreads, D == 64 ? 2 : 1) paged_f32_kernel(const __grid_constant__ PagedArgs a) {
  constexpr int RT = kTileRows, KT = kTileKeys, C = D / 64, PS = KT + 4;
  extern __shared__ __align__(16) float tile_sm[];
  __shared__ PagedPlanShared plan;
  __shared__ int there_s[2][KT / 8];   // whether eight keys have a page
  float *qs = tile_sm, *ks = qs + RT * (D + 4), *vs = ks + 2 * KT * (D + 4), *ps = vs + 2 * KT * D;
  const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
  pdl_trigger();
  long long all;
  int runs;
  if (!paged_locate<kTileThreads, RT, KT>(a, blockIdx.x, gridDim.x, plan, all, runs)) return;
  const int pieces = a.hd / 4, mask = (1 << a.page_shift) - 1;
  PagedRun run;
  run.begin(a, plan, RT);
  for (; run.next(a, plan, RT, KT); run.step(a)) {
    const PagedSeq& s = run.seq;
    const int p0 = run.t * RT, pairs = s.n * a.G, cap = min(s.len, a.max_blocks << a.page_shift), front = paged_front(a, s, p0);
    const int* table = a.table + run.b * a.table_stride;
    auto fetch = [&](int kt) {
      float *k = ks + (kt & 1) * KT * (D + 4), *v = vs + (kt & 1) * KT * D;
      const int e = tid % (D / 4);
#pragma unroll
      for (int r = tid / (D / 4); r < KT; r += kTileThreads / (D / 4)) {
        const int j = kt * KT + r, page = j < cap ? table[j >> a.page_shift] : -1;
        const bool there = page >= 0 && page < a.num_pages;
        if (e == 0 && (r & 7) == 0) there_s[kt & 1][r >> 3] = there;
        const bool get = there && j >= front && e < pieces;
        const int64_t at = get ? page * a.c_page + run.h * a.c_head + (j & mask) * a.c_tok + e * 4 : 0;
        paged_cp16(k + r * (D + 4) + e * 4, reinterpret_cast<const float*>(a.K) + at, get);
        paged_cp16(v + r * D + e * 4, reinterpret_cast<const float*>(a.V) + at, get);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    __syncthreads();   // the item before has been read
    fetch(run.k0);
    for (int i = tid; i < RT * (D / 4); i += kTileThreads) {
      const int r = i / (D / 4), e = i % (D / 4), p = p0 + r, query = a.by_G(p);
      float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (p < pairs && e < pieces) x = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(a.q) + (int64_t)(s.row0 + query) * a.q_row + (run.h * a.G + p - query * a.G) * a.q_head + e * 4);
      *reinterpret_cast<float4*>(qs + r * (D + 4) + e * 4) = make_float4(x.x * a.c, x.y * a.c, x.z * a.c, x.w * a.c);
    }
    float m[4], l[4];
    float2 acc[4][C][2];
    int lo[4], hi[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int p = p0 + ty * 4 + i, pos = s.len - s.n + a.by_G(p);
      m[i] = -INFINITY;
      l[i] = 0.0f;
      hi[i] = p < pairs ? min(pos + 1, cap) : 0;
      lo[i] = a.window > 0 ? pos - a.window + 1 : 0;
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int e = 0; e < 2; ++e) acc[i][c][e] = make_float2(0.0f, 0.0f);
    }
    for (int kt = run.k0; kt < run.k1; ++kt) {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      __syncthreads();   // this tile has landed, the one before has been used
      if (kt + 1 < run.k1) fetch(kt + 1);
      const float *k = ks + (kt & 1) * KT * (D + 4), *v = vs + (kt & 1) * KT * D;
      float2 x2[4][4];   // rows 4 ty + i, keys tx + 16 j: sums of the even and of the odd elements
      float x[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) x2[i][j] = make_float2(0.0f, 0.0f);
#pragma unroll 4
      for (int e = 0; e < D; e += 4) {
        float4 q4[4], k4[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) q4[i] = *reinterpret_cast<const float4*>(qs + (ty * 4 + i) * (D + 4) + e);
#pragma unroll
        for (int j = 0; j < 4; ++j) k4[j] = *reinterpret_cast<const float4*>(k + (tx + 16 * j) * (D + 4) + e);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            paged_fma2(x2[i][j], make_float2(q4[i].x, q4[i].y), make_float2(k4[j].x, k4[j].y));
            paged_fma2(x2[i][j], make_float2(q4[i].z, q4[i].w), make_float2(k4[j].z, k4[j].w));
          }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) x[i][j] = x2[i][j].x + x2[i][j].y;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int key = tx + 16 * j, at = kt * KT + key;
          if (!(at < hi[i] && at >= lo[i] && there_s[kt & 1][key >> 3])) x[i][j] = -INFINITY;
          top = fmaxf(top, x[i][j]);
        }
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float up = fmaxf(m[i], top), from = fmaxf(up, -FLT_MAX);   // no key seen yet: every weight is exp2(-inf)
        const float f = exp2f(m[i] - from);
        m[i] = up;
        l[i] *= f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          x[i][j] = exp2f(x[i][j] - from);
          l[i] += x[i][j];
          ps[(ty * 4 + i) * PS + tx + 16 * j] = x[i][j];
        }
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int e = 0; e < 2; ++e) acc[i][c][e].x *= f, acc[i][c][e].y *= f;
      }
      __syncwarp();   // a row's weights are made and used by the same half of a warp
#pragma unroll 2
      for (int key = 0; key < KT; key += 4) {
        float4 p4[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) p4[i] = *reinterpret_cast<const float4*>(ps + (ty * 4 + i) * PS + key);
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int c = 0; c < C; ++c) {
            const float4 v4 = *reinterpret_cast<const float4*>(v + (key + u) * D + c * 64 + tx * 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float p = u == 0 ? p4[i].x : u == 1 ? p4[i].y : u == 2 ? p4[i].z : p4[i].w;
              paged_fma2(acc[i][c][0], make_float2(p, p), make_float2(v4.x, v4.y));
              paged_fma2(acc[i][c][1], make_float2(p, p), make_float2(v4.z, v4.w));
            }
          }
      }
      __syncwarp();
    }
    const bool whole = run.first && run.last;
    float* rec = a.part + (2 * (int64_t)blockIdx.x + (run.first ? 1 : 0)) * paged_record_floats(RT, a.hd);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float sum = l[i];
#pragma unroll
      for (int o = 1; o < 16; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      const int row = ty * 4 + i, p = p0 + row;
      if (p >= pairs) continue;
      const int query = a.by_G(p);
      float* out = reinterpret_cast<float*>(a.out) + (int64_t)(s.row0 + query) * a.o_row + (int64_t)(run.h * a.G + p - query * a.G) * a.o_head;
      const float inv = whole ? (sum == 0.0f ? 0.0f : 1.0f / sum) : 1.0f;
      if (!whole && tx == 0) *reinterpret_cast<float2*>(rec + 2 * row) = make_float2(m[i], sum);
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int e = c * 64 + tx * 4;
        if (e >= a.hd) continue;
        *reinterpret_cast<float4*>((whole ? out : rec + 2 * RT + row * a.hd) + e) = make_float4(acc[i][c][0].x * inv, acc[i][c][0].y * inv, acc[i][c][1].x * inv, acc[i][c][1].y * inv);
      }
    }
  }
}

// Joins the records of the items that runs end in, four elements of a row per thread.  What bounds it: latency of dependent reads, then the records.
// W warps share the records of 32 x 4 elements: an item of few rows may have a record of every run (one token of 16384, 8 KV heads: 37 each; W = 1 took 16 us,
// W = 8 takes 6), one of many rows has few.
constexpr int kJoinThreads = 256;
template <typename T, int W>
__global__ void __launch_bounds__(kJoinThreads) paged_combine_kernel(const __grid_constant__ PagedArgs a, int RT) {
  constexpr int Q = kJoinThreads / W;   // quads of a CTA
  __shared__ float4 shared_acc[W > 1 ? W : 1][W > 1 ? Q : 1];
  __shared__ float2 shared_ml[W > 1 ? W : 1][W > 1 ? Q : 1];
  const int c = (int)blockIdx.x + 1, share = W > 1 ? (int)threadIdx.x / Q : 0, at = (int)threadIdx.x % Q;
  pdl_wait();
  const int4 j = __ldcg(&a.joins[2 * c]);
  const int h = __ldcg(&a.joins[2 * c + 1]).x, n = j.x, quads = a.hd / 4;
  if (n == 0) return;
  const int64_t rf = paged_record_floats(RT, a.hd);
  // of run c - 1: its last; of the runs behind: their first
  auto record = [&](int k) { return a.part + (k == 0 ? 2 * (int64_t)(c - 1) + 1 : 2 * (int64_t)(c - 1 + k)) * rf; };
  for (int i0 = (int)blockIdx.y * Q; i0 < j.w * quads; i0 += Q * (int)gridDim.y) {
    const int i = i0 + at, row = i / quads, e = (i - row * quads) * 4;
    const bool live = row < j.w;
    float m = -INFINITY, sum = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (live)
      for (int k0 = share; k0 < n; k0 += 4 * W) {
        // four records on their way at a time, both parts of them
        float2 ml[4];
        float4 x[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const float* r = record(min(k0 + u * W, n - 1));
          ml[u] = __ldcg(reinterpret_cast<const float2*>(r + 2 * row));
          x[u] = __ldcg(reinterpret_cast<const float4*>(r + 2 * RT + (int64_t)row * a.hd + e));
          if (k0 + u * W >= n) ml[u] = make_float2(-INFINITY, 0.0f), x[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
        const float up = fmaxf(fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x)), m), from = fmaxf(up, -FLT_MAX), f0 = exp2f(m - from);
        m = up;
        sum *= f0;
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[q] *= f0;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const float f = exp2f(ml[u].x - from);
          sum += ml[u].y * f;
          acc[0] += x[u].x * f;
          acc[1] += x[u].y * f;
          acc[2] += x[u].z * f;
          acc[3] += x[u].w * f;
        }
      }
    if constexpr (W > 1) {
      __syncthreads();   // the elements before have been read
      if (share > 0) {
        shared_acc[share][at] = make_float4(acc[0], acc[1], acc[2], acc[3]);
        shared_ml[share][at] = make_float2(m, sum);
      }
      __syncthreads();
      if (share > 0) continue;
      const int most = min(n, W);
      float up = m;
      for (int k = 1; k < most; ++k) up = fmaxf(up, shared_ml[k][at].x);
      const float from = fmaxf(up, -FLT_MAX), f0 = exp2f(m - from);
      sum *= f0;
#pragma unroll
      for (int q = 0; q < 4; ++q) acc[q] *= f0;
      for (int k = 1; k < most; ++k) {
        const float f = exp2f(shared_ml[k][at].x - from);
        const float4 x = shared_acc[k][at];
        sum += shared_ml[k][at].y * f;
        acc[0] += x.x * f;
        acc[1] += x.y * f;
        acc[2] += x.z * f;
        acc[3] += x.w * f;
      }
    }
    if (!live) continue;
    const int p = j.z + row, query = a.by_G(p);
    T* out = reinterpret_cast<T*>(a.out) + (int64_t)(j.y + query) * a.o_row + (int64_t)(h * a.G + p - query * a.G) * a.o_head + e;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[k] *= inv;
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(out) = make_float4(acc[0], acc[1], acc[2], acc[3]);
    else *reinterpret_cast<uint2*>(out) = make_uint2(Pair16<T>::put(acc[0], acc[1]), Pair16<T>::put(acc[2], acc[3]));
  }
}

template <typename T>
static cudaError_t launch_join(const PagedArgs& a, int RT, int ctas, cudaStream_t s) {
  const int W = RT <= 32 ? 8 : RT <= 64 ? 2 : 1, rows = a.most < RT ? a.most : RT, parts = (rows * a.hd / 4 * W + kJoinThreads - 1) / kJoinThreads;
  const dim3 grid(ctas - 1, parts < 16 ? parts : 16);   // most runs end between items: few CTAs each, which go round
  return launch_k(W == 8 ? paged_combine_kernel<T, 8> : W == 2 ? paged_combine_kernel<T, 2> : paged_combine_kernel<T, 1>, grid, dim3(kJoinThreads), 0, s, a, RT);
}
int launch_paged_combine(int device, int dtype, const PagedArgs& a, int RT, int ctas, cudaStream_t s) {
  if (ctas < 2) return 1;
  PdlScope chained(true);
  if (dtype == TSB200_F32) TSB_CUDA(launch_join<float>(a, RT, ctas, s));
  else if (dtype == TSB200_F16) TSB_CUDA(launch_join<__half>(a, RT, ctas, s));
  else TSB_CUDA(launch_join<__nv_bfloat16>(a, RT, ctas, s));
  count_launch(device);
  return check_launch("paged_combine");
}

// The kernel that serves a call, its rows of a tile and its CTAs, by the most (query, head) pairs of a KV head that a sequence may have.  us at both sides of the rules, 8 KV heads:
//   16-bit, mma.sync | tcgen05      1 sequence of 500   1 of 16000      8 of 4000      32 of 4000
//     heads of 128, 32 pairs           14.7 | 19.5     30.0 | 31.7    35.5 | 34.5    79.5 | 79.9
//                   64 (two tiles)     16.4 | 20.1     35.5 | 32.4    47.8 | 37.9     127 | 93
//     heads of  64, 32 pairs           12.3 | 17.1     21.8 | 27.3    24.2 | 29.3    50.5 | 68.6
//                   64 (two tiles)     13.0 | 17.1     25.3 | 27.6    31.7 | 31.7    79.9 | 79.2
//   fp32, a lane per key | tiles     1 of 300            1 of 4000       8 of 1000      32 of 4000
//     heads of  64, 16 pairs           25.6 | 13.7     28.3 | 32.4    30.0 | 31.1     217 | 366
//                   32                 25.9 | 14.0     34.5 | 33.8    37.9 | 31.7     422 | 374
//     heads of 128, 16 pairs           34.5 | 17.1     42.0 | 46.4    43.7 | 53.6     324 | 718
//                   32                 35.1 | 18.4     51.9 | 47.1    58.0 | 55.0     627 | 721
// One number each, between the sides that most sizes have: short single sequences of 33 pairs and more lose up to 5 us in 16 bits, of 16 and fewer in fp32 up to 18.
struct PagedChoice {
  enum { FMA, TILE, MMA, TC } kind;
  int RT, KT, ctas;
};
static PagedChoice paged_choose(int sm_count, int dtype, int64_t pairs, int hd, bool positive) {
  PagedChoice c;
  if (is_16bit(dtype) && (hd == 64 || hd == 128) && positive) {
    if (pairs <= 32) {
      c.kind = PagedChoice::MMA;
      c.RT = pairs <= 16 ? 16 : 32;
      c.KT = 64;
      c.ctas = 2 * sm_count;
      return c;
    }
    c.kind = PagedChoice::TC;
    c.RT = 256;
    c.KT = 128;
    c.ctas = sm_count;
    return c;
  }
  if (dtype == TSB200_F32 && hd <= 128 && pairs > 16) {
    c.kind = PagedChoice::TILE;
    c.RT = kTileRows;
    c.KT = kTileKeys;
    c.ctas = sm_count * (hd <= 64 ? 2 : 1);
    return c;
  }
  c.kind = PagedChoice::FMA;
  c.KT = kFmaKeys;
  c.RT = pairs <= 4 ? 4 : 16;
  c.ctas = sm_count * (hd <= 128 ? 3 : 1);
  return c;
}
constexpr int kSmCountMost = 160;   // of a compute capability 10.x device: workspace sizes must not need one
static int64_t paged_ws_bytes(int dtype, int64_t pairs, int hd) {
  int64_t most = 0;
  for (int positive = 0; positive < 2; ++positive) {
    const PagedChoice c = paged_choose(kSmCountMost, dtype, pairs, hd, positive);
    const int64_t n = 2LL * c.ctas * (paged_record_floats(c.RT, hd) * 4 + (int64_t)sizeof(int4));
    if (n > most) most = n;
  }
  return most;
}

template <typename T, int NH>
static int launch_paged_fma_n(int device, DeviceState* st, const PagedArgs& a, const PagedChoice& c, cudaStream_t s) {
  static bool done[kMaxDevices] = {};
  if (!done[device]) {
    TSB_CUDA(cudaFuncSetAttribute(paged_fma_kernel<T, NH, 1>, cudaFuncAttributeMaxDynamicSharedMemorySize, fma_smem<T>(NH, 1)));
    TSB_CUDA(cudaFuncSetAttribute(paged_fma_kernel<T, NH, 4>, cudaFuncAttributeMaxDynamicSharedMemorySize, fma_smem<T>(NH, 4)));
    done[device] = true;
  }
  if (c.RT == 4) {
    paged_fma_kernel<T, NH, 1><<<c.ctas, kFmaThreads, fma_smem<T>(NH, 1), s>>>(a);
  } else {
    paged_fma_kernel<T, NH, 4><<<c.ctas, kFmaThreads, fma_smem<T>(NH, 4), s>>>(a);
  }
  count_launch(device);
  return check_launch("paged_fma");
}
template <int D>
static int launch_paged_tile(int device, const PagedArgs& a, const PagedChoice& c, cudaStream_t s) {
  static bool done[kMaxDevices] = {};
  if (!done[device]) {
    TSB_CUDA(cudaFuncSetAttribute(paged_f32_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, tile_smem<D>()));
    done[device] = true;
  }
  paged_f32_kernel<D><<<c.ctas, kTileThreads, tile_smem<D>(), s>>>(a);
  count_launch(device);
  return check_launch("paged_f32");
}
template <typename T>
static int launch_paged_fma(int device, DeviceState* st, const PagedArgs& a, const PagedChoice& c, cudaStream_t s) {
  if (a.hd <= 32) return launch_paged_fma_n<T, 1>(device, st, a, c, s);
  if (a.hd <= 64) return launch_paged_fma_n<T, 2>(device, st, a, c, s);
  if (a.hd <= 128) return launch_paged_fma_n<T, 4>(device, st, a, c, s);
  return launch_paged_fma_n<T, 8>(device, st, a, c, s);
}

static bool page_size_ok(int page, int* shift) {
  for (int i = 3; i <= 8; ++i)
    if (page == 1 << i) {
      *shift = i;
      return true;
    }
  return false;
}

}  // namespace tsb

using namespace tsb;

extern "C" {

int TSB200_PagedPlan(int device, const int32_t* cached, const int32_t* fresh, int B, int page, int32_t* table, int64_t table_stride, int max_blocks, int32_t* held,
                     int32_t* free_pages, int32_t* free_count, int num_pages, int32_t* lens, int32_t* starts, int32_t* slots, int32_t* positions, int rows,
                     void* stream) {
  PlanArgs a{};
  TSB_CHECK(cached && fresh && table && held && free_pages && free_count && lens && starts && (rows == 0 || (slots && positions)), "paged_plan: null pointer");
  TSB_CHECK(B >= 1 && B <= kPlanMaxB, "paged_plan: %d sequences, 1 to %d are served", B, kPlanMaxB);
  TSB_CHECK(page_size_ok(page, &a.page_shift), "paged_plan: pages of %d tokens, a power of two from 8 to 256 is wanted", page);
  TSB_CHECK(max_blocks >= 1 && table_stride >= max_blocks && (int64_t)B * max_blocks <= 0x7fffffff && (int64_t)max_blocks * page <= 0x7fffffff,
            "paged_plan: a table of %d rows of %d pages (stride %lld)", B, max_blocks, (long long)table_stride);
  TSB_CHECK(num_pages >= 0 && (int64_t)num_pages * page <= 0x7fffffff, "paged_plan: %d pages of %d tokens", num_pages, page);
  TSB_CHECK(rows >= 0, "paged_plan: %d rows", rows);
  KeepDevice keep;
  DeviceState* st;
  TSB_TRY(use_device(device, &st));
  a.cached = cached; a.fresh = fresh; a.B = B; a.max_blocks = max_blocks; a.num_pages = num_pages; a.rows = rows; a.table = table; a.table_stride = table_stride;
  a.held = held; a.free_pages = free_pages; a.free_count = free_count; a.lens = lens; a.starts = starts; a.slots = slots; a.positions = positions;
  // a cluster for many rows
  const int smem = 6 * B * (int)sizeof(int), ctas = rows > 2048 ? 8 : 1;
  static bool done[kMaxDevices] = {};
  if (!done[device]) {
    TSB_CUDA(cudaFuncSetAttribute(paged_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 6 * kPlanMaxB * (int)sizeof(int)));
    done[device] = true;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kPlanThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = pick_stream(st, stream);
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = ctas;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  TSB_CUDA(cudaLaunchKernelEx(&cfg, paged_plan_kernel, a, ctas));
  count_launch(device);
  return check_launch("paged_plan");
}

int TSB200_QKNormRopePaged(int device, int dtype, void* q_out, int64_t o_row, int64_t o_head, const void* q, int64_t q_row, int64_t q_head, const void* k,
                           int64_t k_row, int64_t k_head, const void* v, int64_t v_row, int64_t v_head, const void* q_norm, const void* k_norm, float eps,
                           const int32_t* positions, const int32_t* slots, int rows, int H, int Hkv, int hd, int rope_style, int rope_dims, double rope_base,
                           void* cacheK, void* cacheV, int64_t c_page, int64_t c_head, int64_t c_tok, int num_pages, int page, void* stream) {
  RopePagedArgs a{};
  TSB_CHECK(rows >= 0 && H >= 1 && Hkv >= 1 && (int64_t)H + 2LL * Hkv <= 65536, "qk_norm_rope_paged: %d rows of %d and %d heads", rows, H, Hkv);
  TSB_CHECK(dtype == TSB200_F32 || dtype == TSB200_F16 || dtype == TSB200_BF16, "qk_norm_rope_paged: unsupported dtype %d", dtype);
  TSB_CHECK(hd >= 8 && hd % 8 == 0 && hd <= kRopeMaxHd, "qk_norm_rope_paged: head size %d, a multiple of 8 up to %d is wanted", hd, kRopeMaxHd);
  TSB_CHECK(rope_style >= 0 && rope_style <= 2, "qk_norm_rope_paged: rotation style %d", rope_style);
  TSB_CHECK(rope_style == 0 || (rope_dims >= 2 && rope_dims <= hd && rope_dims % (rope_style == 2 ? 16 : 2) == 0),
            "qk_norm_rope_paged: %d rotated elements of %d (pairs: an even number, halves: a multiple of 16)", rope_dims, hd);
  TSB_CHECK(rope_style == 0 || (rope_base > 0 && std::isfinite(rope_base)), "qk_norm_rope_paged: rotation base %g", rope_base);
  TSB_CHECK(page_size_ok(page, &a.page_shift), "qk_norm_rope_paged: pages of %d tokens, a power of two from 8 to 256 is wanted", page);
  TSB_CHECK(num_pages >= 0 && (int64_t)num_pages * page <= 0x7fffffff, "qk_norm_rope_paged: %d pages of %d tokens", num_pages, page);
  if (rows == 0) return 1;
  TSB_CHECK(q_out && q && k && v && slots && (positions || rope_style == 0) && cacheK && cacheV, "qk_norm_rope_paged: null pointer");
  KeepDevice keep;
  DeviceState* st;
  TSB_TRY(use_device(device, &st));
  for (const int64_t stride : {o_row, o_head, q_row, q_head, k_row, k_head, v_row, v_head, c_page, c_head, c_tok})
    TSB_CHECK(stride >= 0 && stride <= 0x7fffffff, "qk_norm_rope_paged: a stride of %lld elements", (long long)stride);
  a.out = q_out; a.q = q; a.k = k; a.v = v; a.q_norm = q_norm; a.k_norm = k_norm;
  a.o_row = (int)o_row; a.o_head = (int)o_head; a.q_row = (int)q_row; a.q_head = (int)q_head; a.k_row = (int)k_row; a.k_head = (int)k_head; a.v_row = (int)v_row; a.v_head = (int)v_head;
  a.eps = eps; a.positions = positions; a.slots = slots; a.rows = rows; a.H = H; a.Hkv = Hkv; a.hd = hd; a.rot = rope_style ? rope_dims : 0; a.style = rope_style;
  a.first = 1.0 / 3.14159265358979323846;
  a.ratio = rope_style ? std::pow(rope_base, -2.0 / rope_dims) : 1.0;
  a.K = cacheK; a.V = cacheV; a.c_page = (int)c_page; a.c_head = (int)c_head; a.c_tok = (int)c_tok; a.num_pages = num_pages;
  const int V = 16 / (int)dtype_size(dtype);
  const bool wide = ((o_row | o_head | q_row | q_head | k_row | k_head | v_row | v_head | c_page | c_head | c_tok) % V) == 0 &&
                    (((uintptr_t)q_out | (uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)cacheK | (uintptr_t)cacheV) % 16) == 0;
  // Few rows: a CTA each, or several, so that every head has its lanes at once; many: four CTAs of an SM share them, at least a pass of angles each
  const int L = hd <= 8 ? 1 : hd <= 16 ? 2 : hd <= 32 ? 4 : hd <= 64 ? 8 : hd <= 128 ? 16 : 32, heads = H + 2 * Hkv;
  const int pieces = wide && dtype != TSB200_F32 && hd > 32 && hd <= 128 ? 2 : 1, parts = (heads * L / pieces + kRopeThreads - 1) / kRopeThreads;
  const int ctas = 4 * st->sm_count;
  dim3 grid;
  if (rows <= ctas / 2) {
    a.rows_here = 1;
    grid = dim3(rows, (int64_t)rows * parts <= ctas ? parts : 1);
  } else {
    a.rows_here = (rows + ctas - 1) / ctas;
    grid = dim3((rows + a.rows_here - 1) / a.rows_here);
  }
  cudaStream_t s = pick_stream(st, stream);
#define TSB_ROPE_PAGED(T)                                                                 \
  do {                                                                                    \
    if (wide) launch_rope_paged<T, true>(a, grid, s);                                     \
    else launch_rope_paged<T, false>(a, grid, s);                                         \
  } while (0)
  if (dtype == TSB200_F32) TSB_ROPE_PAGED(float);
  else if (dtype == TSB200_F16) TSB_ROPE_PAGED(__half);
  else TSB_ROPE_PAGED(__nv_bfloat16);
#undef TSB_ROPE_PAGED
  count_launch(device);
  return check_launch("qk_norm_rope_paged");
}

int64_t TSB200_PagedAttentionWorkspaceBytes(int dtype, int H, int Hkv, int hd, int max_new) {
  if (H < 1 || Hkv < 1 || H % Hkv || hd < 8 || hd > 256 || max_new < 1) return 0;
  return paged_ws_bytes(dtype, (int64_t)max_new * (H / Hkv), hd);
}

int TSB200_PagedAttention(int device, int dtype, void* out, int64_t o_row, int64_t o_head, const void* q, int64_t q_row, int64_t q_head, const void* cacheK,
                          const void* cacheV, int64_t c_page, int64_t c_head, int64_t c_tok, int num_pages, int page, const int32_t* table, int64_t table_stride,
                          int max_blocks, const int32_t* starts, const int32_t* lens, int B, int rows, int max_new, int H, int Hkv, int hd, float scale, int window,
                          void* workspace, int64_t workspace_bytes, void* stream) {
  PagedArgs a{};
  TSB_CHECK(dtype == TSB200_F32 || dtype == TSB200_F16 || dtype == TSB200_BF16, "paged_attention: unsupported dtype %d", dtype);
  TSB_CHECK(B >= 0 && rows >= 0 && max_new >= 1, "paged_attention: %d sequences, %d rows, at most %d new", B, rows, max_new);
  TSB_CHECK(H >= 1 && H <= 65536 && Hkv >= 1 && H % Hkv == 0, "paged_attention: %d query heads over %d key / value heads", H, Hkv);
  TSB_CHECK(hd >= 8 && hd % 8 == 0 && hd <= 256, "paged_attention: head size %d, a multiple of 8 up to 256 is wanted", hd);
  TSB_CHECK(page_size_ok(page, &a.page_shift), "paged_attention: pages of %d tokens, a power of two from 8 to 256 is wanted", page);
  TSB_CHECK(max_blocks >= 1 && table_stride >= max_blocks && (int64_t)max_blocks * page <= 0x7fffff00, "paged_attention: %d pages per sequence (stride %lld)", max_blocks,
            (long long)table_stride);
  TSB_CHECK(num_pages >= 0 && (int64_t)num_pages * page <= 0x7fffffff, "paged_attention: %d pages of %d tokens", num_pages, page);
  TSB_CHECK((int64_t)rows * H <= 0x7fff0000, "paged_attention: %d rows of %d heads", rows, H);
  TSB_CHECK(window >= 0, "paged_attention: window %d", window);
  if (B == 0 || rows == 0) return 1;
  TSB_CHECK(out && q && cacheK && cacheV && table && starts && lens, "paged_attention: null pointer");
  const int V = 16 / (int)dtype_size(dtype);
  TSB_CHECK(((o_row | o_head | q_row | q_head | c_page | c_head | c_tok) % V) == 0 && (((uintptr_t)out | (uintptr_t)q | (uintptr_t)cacheK | (uintptr_t)cacheV) % 16) == 0,
            "paged_attention: pointers and strides must be multiples of 16 bytes");
  KeepDevice keep;
  DeviceState* st;
  TSB_TRY(use_device(device, &st));
  const int64_t pairs = (int64_t)max_new * (H / Hkv), need = paged_ws_bytes(dtype, pairs, hd);
  TSB_CHECK(workspace && workspace_bytes >= need && (uintptr_t)workspace % 16 == 0, "paged_attention: a workspace of %lld bytes on a boundary of 16 is needed (%lld given)",
            (long long)need, (long long)(workspace ? workspace_bytes : 0));
  a.out = out; a.q = q; a.K = cacheK; a.V = cacheV; a.o_row = o_row; a.o_head = o_head; a.q_row = q_row; a.q_head = q_head;
  a.c_page = c_page; a.c_head = c_head; a.c_tok = c_tok; a.table = table; a.table_stride = table_stride; a.max_blocks = max_blocks; a.num_pages = num_pages;
  a.starts = starts; a.lens = lens; a.B = B; a.rows = rows; a.H = H; a.Hkv = Hkv; a.G = H / Hkv; a.hd = hd;
  a.by_G.set((uint32_t)a.G);
  a.c = scale * 1.44269504088896340736f;
  a.window = window;
  a.most = (int)(pairs < 0x7fffffff ? pairs : 0x7fffffff);
  cudaStream_t s = pick_stream(st, stream);
  // the kernels on tensor cores look for the largest score before it is scaled
  const PagedChoice c = paged_choose(st->sm_count, dtype, pairs, hd, scale > 0 && paged_tc_strides(a));
  TSB_CHECK(st->sm_count <= kSmCountMost, "paged_attention: %d SMs", st->sm_count);
  a.joins = reinterpret_cast<int4*>(workspace);
  a.part = reinterpret_cast<float*>(a.joins + 2 * c.ctas);
  a.min_units = c.kind == PagedChoice::TILE ? 1 : 4;   // a unit of the fp32 tiles takes as long as eight of a lane per key
  a.snap = c.kind == PagedChoice::TILE ? 0 : 1;
  a.start = 1;
  if (c.kind == PagedChoice::MMA) return launch_paged_mma(device, st, dtype, a, c.RT, s);
  if (c.kind == PagedChoice::TC) return launch_paged_tc(device, st, dtype, a, s);
  if (c.kind == PagedChoice::TILE) {
    if (hd <= 64) TSB_TRY(launch_paged_tile<64>(device, a, c, s));
    else TSB_TRY(launch_paged_tile<128>(device, a, c, s));
  } else if (dtype == TSB200_F32) TSB_TRY(launch_paged_fma<float>(device, st, a, c, s));
  else if (dtype == TSB200_F16) TSB_TRY(launch_paged_fma<__half>(device, st, a, c, s));
  else TSB_TRY(launch_paged_fma<__nv_bfloat16>(device, st, a, c, s));
  return launch_paged_combine(device, dtype, a, c.RT, c.ctas, s);
}

}  // extern "C"
