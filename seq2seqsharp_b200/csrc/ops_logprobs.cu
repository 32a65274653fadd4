// Log probabilities of given tokens, with the entropy of their rows, their rank and the most likely alternatives:
//   m = max x,  S = sum e^(x - m),  T = sum (x - m) e^(x - m):  lp(t) = x_t - m - log S,  H = log S - T / S,
//   rank = #{j: x_j > x_t, or x_j = x_t and j < t},  best = the `top` largest logits, the lower index first among equal ones.
//
// One pass over the logits.  A thread keeps a running maximum and both sums of its share in fp32, with powers of two (x log2 e is taken against the rounded m log2 e, any
// reference being as good as the maximum itself); what threads have is joined in 64 bits, so that a probability near 1 keeps its digits (log S of a sum a little over 1).
// The threads' maxima are also a bound for the alternatives: where r = ceil(top / warps) lanes of ceil(top / r) warps have a logit of at least B, `top` words have, and only threads
// whose maximum is at least B have one, nearly always in the piece of their maximum alone, which is read again.  What they find (some 40 words for random logits) is ordered by counting.
// Should that be over kLpRoom (many equal logits), the bound is raised to the top-th largest (logit, index) by eight histograms of eight bits.
//
// What bounds it: issue slots, about ten instructions a 16-bit logit (28.7 before two at a time, counts in the type's own numbers and rows' ends apart: 4096 rows of 50257 bf16 327 us, now 86, floor 63),
// and bytes; for few rows two dependent reads, the words' second look and a cluster barrier (one row of 32000 fp32, 5 alternatives 6.6 us).
//
// Few rows: a cluster of up to eight CTAs shares a row, and the first one joins what all have pushed to it.  Many rows: a CTA per row.
#include <cmath>
#include <type_traits>

#include "kernels.cuh"

namespace tsb {

constexpr int kLpTop = 32;       // most alternatives
constexpr int kLpRoom = 1024;    // words that a CTA orders
constexpr int kLpCluster = 8;
constexpr int kLpUnroll = 4;     // loads of 16 bytes in flight per thread
constexpr float kLog2e = 1.44269504088896341f;

struct LogProbArgs {
  const void* x;         // rows of stride x_row
  const int* tokens;     // [rows]
  int64_t x_row;
  int V, top, parts;     // parts: CTAs of a row
  float* lp;             // [rows]
  float* entropy;        // [rows]
  int* rank;             // [rows]
  int* best;             // [rows, top]
  float* best_lp;        // [rows, top]
};

__device__ __forceinline__ float lp_max_nan(float a, float b) {   // a NaN stays one
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float lp_exp2(float v) {   // off by 2 ulp; 0 below 2^-126
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// whole numbers that order as the numbers do, a zero having one sign; NaN comes last
__device__ __forceinline__ uint32_t lp_order(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  return v != v ? 0u : (b & 0x80000000u ? ~b : b | 0x80000000u);
}
__device__ __forceinline__ float lp_value(uint32_t o) { return o == 0u ? NAN : __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }
__device__ __forceinline__ uint64_t lp_key(float v, int j) { return ((uint64_t)lp_order(v) << 32) | (uint32_t)~j; }

__device__ __forceinline__ uint64_t lp_two(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 lp_apart(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t lp_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t lp_add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// 16 bytes of logits.  What needs no wider type (largest, smallest, count of those at least some value) is done for two 16-bit ones at a time.
template <typename T> struct LpVec {
  static constexpr int N = 8;
  typedef typename std::conditional<Pair16<T>::kBf16, __nv_bfloat162, __half2>::type Two;
  uint4 raw;
  __device__ __forceinline__ uint32_t word(int i) const { return i == 0 ? raw.x : i == 1 ? raw.y : i == 2 ? raw.z : raw.w; }
  __device__ __forceinline__ Two two(int i) const { const uint32_t r = word(i); return *reinterpret_cast<const Two*>(&r); }
  __device__ __forceinline__ float2 pair(int i) const { return Pair16<T>::get(word(i)); }   // elements 2 i, 2 i + 1
  __device__ __forceinline__ float get(int e) const { const float2 f = pair(e >> 1); return e & 1 ? f.y : f.x; }
};
template <> struct LpVec<float> {
  static constexpr int N = 4;
  uint4 raw;
  __device__ __forceinline__ float get(int e) const { return __uint_as_float(e == 0 ? raw.x : e == 1 ? raw.y : e == 2 ? raw.z : raw.w); }
  __device__ __forceinline__ float2 pair(int i) const { return make_float2(get(2 * i), get(2 * i + 1)); }
};
// largest of some vectors; a NaN is passed over
template <typename T> struct LpLargest {
  typename LpVec<T>::Two hi;
  __device__ __forceinline__ LpLargest() {
    const uint32_t h = Pair16<T>::put(-INFINITY, -INFINITY);
    hi = *reinterpret_cast<const typename LpVec<T>::Two*>(&h);
  }
  __device__ __forceinline__ void add(const LpVec<T>& x) { hi = __hmax2(hi, __hmax2(__hmax2(x.two(0), x.two(1)), __hmax2(x.two(2), x.two(3)))); }
  __device__ __forceinline__ float get() const { const float2 f = Pair16<T>::get(*reinterpret_cast<const uint32_t*>(&hi)); return fmaxf(f.x, f.y); }
};
template <> struct LpLargest<float> {
  float hi;
  __device__ __forceinline__ LpLargest() : hi(-INFINITY) {}
  __device__ __forceinline__ void add(const LpVec<float>& x) { hi = fmaxf(fmaxf(hi, fmaxf(x.get(0), x.get(1))), fmaxf(x.get(2), x.get(3))); }
  __device__ __forceinline__ float get() const { return hi; }
};
// how many logits are at least `v`: counted in the type's own numbers (at most 16 in each half, which they hold), added up by total()
template <typename T> struct LpCount {
  typename LpVec<T>::Two n;
  __device__ __forceinline__ LpCount() {
    const uint32_t zero = 0u;
    n = *reinterpret_cast<const typename LpVec<T>::Two*>(&zero);
  }
  __device__ __forceinline__ void add(const LpVec<T>& x, uint32_t v) {
    const typename LpVec<T>::Two a = *reinterpret_cast<const typename LpVec<T>::Two*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) n = __hadd2(n, __hge2(x.two(i), a));
  }
  __device__ __forceinline__ int total() const { const float2 f = Pair16<T>::get(*reinterpret_cast<const uint32_t*>(&n)); return (int)(f.x + f.y); }
};
template <> struct LpCount<float> {
  int n = 0;
  __device__ __forceinline__ void add(const LpVec<float>& x, uint32_t v) {
#pragma unroll
    for (int e = 0; e < 4; ++e) n += x.get(e) >= __uint_as_float(v);
  }
  __device__ __forceinline__ int total() const { return n; }
};
// a number of the type for LpCount::add (twice in 32 bits for 16-bit types), and the next larger one (of infinity and NaN: a NaN, which nothing reaches)
__device__ __forceinline__ uint32_t lp_bits(float v) { return __float_as_uint(v); }
__device__ __forceinline__ uint32_t lp_bits(__half v) { return (uint32_t)__half_as_ushort(v) * 0x10001u; }
__device__ __forceinline__ uint32_t lp_bits(__nv_bfloat16 v) { return (uint32_t)__bfloat16_as_ushort(v) * 0x10001u; }
template <typename T>
__device__ __forceinline__ uint32_t lp_bits_above(T v) {
  const float f = to_f<T>(v);
  const uint32_t one = sizeof(T) == 4 ? 1u : 0x10001u, b = lp_bits(v);
  return f != f ? b : f == 0.0f ? one : f > 0.0f ? b + one : b - one;
}

// A row as pieces of 16 bytes on their boundaries, `head` elements in front of the first and `tail` behind the last
template <typename T>
struct LpRow {
  static constexpr int N = LpVec<T>::N;
  const T* x;
  int head, pieces, tail;
  __device__ __forceinline__ LpRow(const T* p, int V) : x(p) {
    head = min(V, (int)((-(uintptr_t)p & 15) / sizeof(T)));
    pieces = (V - head) / N;
    tail = V - head - pieces * N;
  }
  __device__ __forceinline__ int first(int v) const { return head + v * N; }   // index of a piece's first element
  __device__ __forceinline__ LpVec<T> load(int v) const {
    LpVec<T> r;
    r.raw = *reinterpret_cast<const uint4*>(x + first(v));
    return r;
  }
};

// Exponents are taken as x log2 e - m log2 e with the second product rounded, one instruction a logit.  What that product's rounding leaves is an exponent that all logits of
// a share have more: below 2^20 at most a sixteenth, but whole powers where a step of m log2 e is no longer small (440 at -1e10, so that sums of words masked by that are infinite).  From
// 2^20 on, and for infinities, the difference comes first.
__device__ __forceinline__ bool lp_far(float m) { return !(fabsf(m) < 0x1p20f); }
// what the rounding of m log2 e leaves, exact (a product and its rounding differ by a number of fp32)
__device__ __forceinline__ float lp_left(float m) { return lp_far(m) ? 0.0f : fmaf(m, kLog2e, -__fmul_rn(m, kLog2e)); }
// exponent of 2 between two maxima, at most 0, as their sums have them; 2^-1000 is 0, and so is its product with the exponent
__device__ __forceinline__ float lp_gap(float m, float to) { return lp_max_nan(fmaf(m - to, kLog2e, lp_left(to) - lp_left(m)), -1000.0f); }
struct LpSums {
  float m, s, t;   // maximum; sums, over the logits, of 2^exponent and of the exponent times it
  __device__ __forceinline__ void raise(float to) {   // to > m
    if (m > -INFINITY) {
      const float d = lp_gap(m, to), f = lp_exp2(d);
      t = f * fmaf(d, s, t);
      s *= f;
    }
    m = to;
  }
};
// the same joined, in 64 bits
struct __align__(16) LpJoined {
  double s, t;
  float m;
  int rank;
};
__device__ __forceinline__ void lp_rebase(double& s, double& t, float m, float to) {   // both are maxima, m <= to
  if (m == to || !(m > -INFINITY)) return;   // (a share of -infinity has sums of 0, or NaN)
  const float d = lp_gap(m, to);
  const double f = (double)lp_exp2(d);
  t = f * (t + (double)d * s);
  s *= f;
}
template <int LANES>
__device__ __forceinline__ double lp_sum(double v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// `n` of them (at most LANES) by a whole warp; every lane has the result
template <int LANES>
__device__ __forceinline__ LpJoined lp_join(const LpJoined* from, int n) {
  const int lane = (int)threadIdx.x & 31;
  LpJoined c{0.0, 0.0, -INFINITY, 0};
  if ((lane & (LANES - 1)) < n) c = from[lane & (LANES - 1)];
  const float m = lp_value(__reduce_max_sync(0xffffffffu, lp_order(c.m)));
  lp_rebase(c.s, c.t, c.m, m);
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) c.rank += __shfl_xor_sync(0xffffffffu, c.rank, o);
  return LpJoined{lp_sum<LANES>(c.s), lp_sum<LANES>(c.t), m, c.rank};
}

// what the joined sums of a row make of a logit
struct LpWhole {
  double log_s, entropy;
  float m;
  int rank;
  __device__ __forceinline__ LpWhole() {}
  __device__ __forceinline__ explicit LpWhole(LpJoined c) : m(c.m), rank(c.rank) {
    const bool none = !(m > -INFINITY);   // nothing but -infinity and NaN
    if (!none && c.s < 1.5) {
      // The maximum's own exponent is what rounding left of it, and its power of two is off by 2 ulp of 1: as much as all other words have where it is nearly certain
      const float own = lp_left(m);
      c.s += exp2((double)own) - (double)lp_exp2(own);
    }
    log_s = none ? (double)NAN : log(c.s);
    entropy = log_s - c.t / c.s * kLn2;
  }
  static constexpr double kLn2 = 0.693147180559945309417;
  // rounding may leave a little over 0 of a certain token
  __device__ __forceinline__ float value(float v) const {
    const double l = (lp_far(m) ? (double)v - (double)m : ((double)v * (double)kLog2e - (double)__fmul_rn(m, kLog2e)) * kLn2) - log_s;
    return (float)(l > 0.0 ? 0.0 : l);
  }
};

// kTrack: several alternatives; which piece a thread's maximum lies in is kept
template <typename T, int kLpThreads, bool kTrack>
__global__ void __launch_bounds__(kLpThreads, 1024 / kLpThreads) log_probs_kernel(LogProbArgs a) {
  constexpr int kLpWarps = kLpThreads / 32;
  __shared__ LpJoined s_join[kLpWarps];
  __shared__ LpJoined s_part[kLpCluster];            // (first CTA) of every CTA of the row
  __shared__ uint32_t s_bound[kLpWarps];
  __shared__ uint64_t s_words[kLpRoom];
  __shared__ uint64_t s_best[kLpCluster * kLpTop];   // (first CTA) of every CTA of the row, 0: none
  __shared__ uint32_t s_hist[256];
  __shared__ uint8_t s_lane[kLpWarps][32];
  __shared__ uint64_t s_prefix;
  __shared__ int s_count, s_need;
  __shared__ LpWhole s_whole;

  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const int parts = a.parts, part = (int)(blockIdx.x % parts);
  const int64_t r = (int64_t)(blockIdx.x / parts);
  if (parts > 1) {   // the first CTA runs; waited for in front of the pushes
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  }
  const LpRow<T> row(reinterpret_cast<const T*>(a.x) + r * a.x_row, a.V);
  constexpr int N = LpVec<T>::N;
  const int v0 = (int)((int64_t)row.pieces * part / parts), v1 = (int)((int64_t)row.pieces * (part + 1) / parts);
  const int token = a.tokens[r];

  struct Group { LpVec<T> of[kLpUnroll]; };
  Group next;   // on its way while one is added up
  auto fetch = [&](int v) {
#pragma unroll
    for (int u = 0; u < kLpUnroll; ++u)
      if (v + u * kLpThreads < v1) next.of[u] = row.load(v + u * kLpThreads);
  };
  fetch(v0 + tid);
  // one element more for some threads: of the row's ends
  int end_j = -1;
  if (part == 0 && tid < row.head + row.tail) end_j = tid < row.head ? tid : row.pieces * N + tid;
  const float end_x = end_j >= 0 ? to_f<T>(row.x[end_j]) : -INFINITY;
  // what the token's rank is counted against: in pieces in front of its own x >= xt, in those behind it x >= the next larger number (a NaN: never)
  const bool given = token >= 0 && token < a.V;
  const T given_x = given ? row.x[token] : from_f<T>(NAN);
  const float xt = to_f<T>(given_x);
  const uint32_t from = lp_bits(given_x), above = lp_bits_above<T>(given_x), never = lp_bits(from_f<T>(NAN));
  const int own = token < row.head ? -1 : (token - row.head) / N;   // the token's piece
  auto outranks = [&](float y, int j) { return y > xt || (y == xt && j < token); };
  int rank = end_j >= 0 && outranks(end_x, end_j);
  if (tid < N && given && own >= v0 && own < v1) rank += outranks(to_f<T>(row.x[row.first(own) + tid]), row.first(own) + tid);

  auto tell = [&](const LpWhole& whole) {
    a.lp[r] = given ? whole.value(xt) : token < 0 ? 0.0f : NAN;
    a.rank[r] = given ? whole.rank : -1;
    a.entropy[r] = (float)(whole.entropy < 0.0 ? 0.0 : whole.entropy);
  };

  LpSums mine{-INFINITY, 0.0f, 0.0f};
  int highest = -1;            // the piece of the maximum (-1: an end's, or none)
  float second = -INFINITY;    // the largest of what is not in it
  auto add = [&](float y, float m, float ref) {   // -infinity, and products that leave fp32, too
    const float d = lp_max_nan(lp_far(m) ? (y - m) * kLog2e : fmaf(y, kLog2e, -ref), -1000.0f), p = lp_exp2(d);
    mine.s += p;
    mine.t = fmaf(d, p, mine.t);
  };
  if (end_j >= 0) {
    mine.m = end_x > -INFINITY ? end_x : -INFINITY;   // (not a NaN)
    const float m = mine.m > -INFINITY ? mine.m : 0.0f;
    add(end_x, m, __fmul_rn(m, kLog2e));
  }
  // the pieces v, v + kLpThreads, .. of a group: all of them, or those in front of v1
  auto group = [&](const LpVec<T>* x, int v, auto all) {
    constexpr bool kAll = decltype(all)::value;
    LpLargest<T> largest;
#pragma unroll
    for (int u = 0; u < kLpUnroll; ++u)
      if (kAll || v + u * kLpThreads < v1) largest.add(x[u]);
    const float top = largest.get();
    if (top > mine.m) {
      if constexpr (kTrack) {   // rarely
        bool found = false;
        second = mine.m;
#pragma unroll
        for (int u = 0; u < kLpUnroll; ++u) {
          if (!kAll && v + u * kLpThreads >= v1) break;
          LpLargest<T> one;
          one.add(x[u]);
          const float y = one.get();
          if (!found && y == top) {
            found = true;
            highest = v + u * kLpThreads;
          } else {
            second = fmaxf(second, y);
          }
        }
      }
      mine.raise(top);
    } else if constexpr (kTrack) {
      second = fmaxf(second, top);
    }
    const float m = mine.m > -INFINITY ? mine.m : 0.0f, ref = __fmul_rn(m, kLog2e);   // nothing but -infinity (and NaN) yet: sums of 0 (of NaN)
    // two at a time
    const uint64_t scale = lp_two(kLog2e, kLog2e), minus = lp_two(-ref, -ref);
    uint64_t gs = 0u, gt = 0u;
    LpCount<T> count;
#pragma unroll
    for (int u = 0; u < kLpUnroll; ++u) {
      const int at = v + u * kLpThreads;
      if (!kAll && at >= v1) break;
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        const float2 y = x[u].pair(i);
        const uint64_t d = lp_fma2(lp_two(y.x, y.y), scale, minus);
        const float2 e = lp_apart(d);
        const uint64_t p = lp_two(lp_exp2(e.x), lp_exp2(e.y));
        gs = lp_add2(gs, p);
        gt = lp_fma2(d, p, gt);
      }
      count.add(x[u], at < own ? from : at > own ? above : never);
    }
    rank += count.total();
    const float2 s = lp_apart(gs), t = lp_apart(gt);
    if (t.x + t.y == t.x + t.y && !lp_far(m)) {
      mine.s += s.x + s.y;
      mine.t += t.x + t.y;
    } else {
      // the difference first; or an exponent of -infinity is among them (0 times it is none), or a NaN.  (1024 rows of 50257 bf16, all but ten words at -1e10 or -infinity 47 us, at -1e4
      // 28; the differences taken by a second copy of the loop above, 38, cost other calls registers: 2048 rows of 50257 fp32, 20 alternatives 87 -> 90.)
#pragma unroll 1
      for (int u = 0; u < kLpUnroll && v + u * kLpThreads < v1; ++u) {
        const LpVec<T> y = row.load(v + u * kLpThreads);
#pragma unroll
        for (int e = 0; e < N; ++e) add(y.get(e), m, ref);
      }
    }
  };
  int v = v0 + tid;
  for (; v + (kLpUnroll - 1) * kLpThreads < v1; v += kLpUnroll * kLpThreads) {
    const Group now = next;
    fetch(v + kLpUnroll * kLpThreads);
    group(now.of, v, std::true_type());
  }
  if (v < v1) group(next.of, v, std::false_type());

  // ---------------- the CTA's sums, against its maximum
  const uint32_t mine_o = lp_order(mine.m), warp_o = __reduce_max_sync(0xffffffffu, mine_o);
  {
    const float m = lp_value(warp_o);
    double s = mine.s, t = mine.t;
    lp_rebase(s, t, mine.m, m);
    s = lp_sum<32>(s);
    t = lp_sum<32>(t);
    rank = __reduce_add_sync(0xffffffffu, rank);
    if (lane == 0) s_join[w] = LpJoined{s, t, m, rank};
  }
  const int top = a.top;
  if (top > 0) {
    // the r-th largest maximum of the warp's lanes
    const int times = (top + kLpWarps - 1) / kLpWarps;
    uint32_t o = mine_o, at = warp_o;
    for (int i = 1; i < times; ++i) {
      if (lane == __ffs(__ballot_sync(0xffffffffu, o == at)) - 1) o = 0u;
      at = __reduce_max_sync(0xffffffffu, o);
    }
    if (lane == 0) s_bound[w] = at;
    if (tid == 0) s_count = 0;
  }
  __syncthreads();

  if (top > 0) {
    const int times = (top + kLpWarps - 1) / kLpWarps, warps = (top + times - 1) / times;
    uint32_t bound;
    {
      const uint32_t o = s_bound[lane & (kLpWarps - 1)];
      int larger = 0;
#pragma unroll
      for (int i = 0; i < kLpWarps; ++i) larger += s_bound[i] > o || (s_bound[i] == o && i < (lane & (kLpWarps - 1)));
      bound = __shfl_sync(0xffffffffu, o, __ffs(__ballot_sync(0xffffffffu, larger == warps - 1)) - 1);
      if (bound <= lp_order(-INFINITY)) bound = 0u;   // threads without a number have this maximum too: every word counts
    }
    // f(key) of every element of piece `at` that is not below least_x.  Little code, one element at a time: there are few such pieces.
    auto each_of = [&](int at, float least_x, auto f) {
      const int j0 = row.first(at);
#pragma unroll 1
      for (int j = j0; j < j0 + N; ++j) {
        const float z = to_f<T>(row.x[j]);
        if (!(z < least_x)) f(lp_key(z, j));
      }
    };
    // The same of the whole shares of the warp's lanes with `any`, which the warp reads together, and of the ends.
    auto look = [&](bool any, float least_x, auto f) {
      const uint32_t lanes = __ballot_sync(0xffffffffu, any);
      if (any) s_lane[w][__popc(lanes & ((1u << lane) - 1u))] = (uint8_t)lane;
      __syncwarp();
      const int first = v0 + w * 32, each = v1 > first ? (v1 - first + kLpThreads - 1) / kLpThreads : 0, items = __popc(lanes) * each;   // (pieces of the first lane, the most)
      auto piece = [&](int k) {
        const int of = k / each;
        return first + (int)s_lane[w][of] + (k - of * each) * kLpThreads;
      };
#pragma unroll 1
      for (int i = lane; i < items; i += 32 * kLpUnroll) {
        LpVec<T> y[kLpUnroll];
        uint32_t hits = 0u;
#pragma unroll
        for (int u = 0; u < kLpUnroll; ++u) {
          const int k = i + 32 * u, at = k < items ? piece(k) : v1;
          if (at < v1) {
            y[u] = row.load(at);
            hits |= 1u << u;
          }
        }
#pragma unroll
        for (int u = 0; u < kLpUnroll; ++u) {
          LpLargest<T> largest;
          largest.add(y[u]);
          if (largest.get() < least_x) hits &= ~(1u << u);
        }
#pragma unroll 1
        for (; hits; hits &= hits - 1u) each_of(piece(i + 32 * (__ffs(hits) - 1)), least_x, f);
      }
      if (end_j >= 0) f(lp_key(end_x, end_j));
      __syncwarp();
    };
    uint64_t least = (uint64_t)bound << 32;
    auto take = [&](uint64_t k) {
      if (k < least) return;
      const int at = atomicAdd(&s_count, 1);
      if (at < kLpRoom) s_words[at] = k;
    };
    // Most threads above the bound have one piece that is: the others' shares alone are read again as a whole.  (Pieces lie kLpThreads apart, so that a share's are as many trips to
    // memory where L2 has let go of the row: 4096 rows of 50257 bf16, 20 alternatives 134 us when all of them read theirs.)
    const float bound_x = lp_value(bound);
    if (bound != 0u) {
      const bool whole_share = kTrack ? lp_order(second) >= bound : mine_o >= bound;
      if (!whole_share && mine_o >= bound && highest >= 0) each_of(highest, bound_x, take);
      look(whole_share, bound_x, take);
      __syncthreads();
    } else {
      // nearly all words are -infinity, or the share is short: what is larger, then, by index, as many of those as are wanted
      least = (uint64_t)(lp_order(-INFINITY) + 1u) << 32;
      look(true, -3.402823466e38f, take);
      __syncthreads();
      auto take_none = [&](uint64_t k) {
        if ((uint32_t)(k >> 32) == lp_order(-INFINITY)) s_words[atomicAdd(&s_count, 1)] = k;
      };
      int have = s_count;
      if (have < top) {
        constexpr int kSome = kLpRoom / 16;   // pieces: of at most half the room
        for (int from_v = v0; from_v < v1 && have < top; from_v += kSome) {
          __syncthreads();   // (all have read the count)
          if (tid < kSome && from_v + tid < v1) each_of(from_v + tid, -INFINITY, take_none);
          __syncthreads();
          have = s_count;
        }
        __syncthreads();
        if (end_j >= 0) take_none(lp_key(end_x, end_j));
        __syncthreads();
      }
    }
    // too many of them, or NaN among the words that are wanted
    if (s_count > kLpRoom || s_count < min(top, (v1 - v0) * N + (part == 0 ? row.head + row.tail : 0))) {
      // the top-th largest key, eight bits at a time
      if (tid == 0) {
        s_prefix = 0u;
        s_need = top;
      }
      for (int shift = 56; shift >= 0; shift -= 8) {
        for (int i = tid; i < 256; i += kLpThreads) s_hist[i] = 0u;
        __syncthreads();
        const uint64_t prefix = s_prefix;
        look(true, -INFINITY, [&](uint64_t k) {
          if (shift == 56 || (k >> (shift + 8)) == (prefix >> (shift + 8))) {
            // most often the lanes that are here have the same digit: one of them counts for all
            const int d = (int)((k >> shift) & 255);
            const uint32_t here = __activemask();
            int same;
            __match_all_sync(here, d, &same);
            if (!same) atomicAdd(&s_hist[d], 1u);
            else if (lane == __ffs(here) - 1) atomicAdd(&s_hist[d], (uint32_t)__popc(here));
          }
        });
        __syncthreads();
        if (tid == 0) {
          int need = s_need, d = 255;
          while (d > 0 && (int)s_hist[d] < need) need -= (int)s_hist[d--];
          s_prefix = prefix | ((uint64_t)d << shift);
          s_need = need;
          s_count = 0;
        }
        __syncthreads();
      }
      least = s_prefix;
      look(true, -INFINITY, take);
      __syncthreads();
    }
    if (parts > 1) cluster_wait();
    // in order: a key's place is the number of larger ones, which four lanes count.  To the first CTA of the row.
    const int n = min(s_count, kLpRoom);
    for (int i0 = w * 8; i0 < n; i0 += kLpWarps * 8) {
      const int i = i0 + (lane >> 2);
      const uint64_t k = i < n ? s_words[i] : 0u;
      int at = 0;
#pragma unroll 4
      for (int j = lane & 3; j < n; j += 4) at += s_words[j] > k;
      at += __shfl_xor_sync(0xffffffffu, at, 1);
      at += __shfl_xor_sync(0xffffffffu, at, 2);
      if (i < n && at < top && (lane & 3) == 0) {
        uint32_t to = (uint32_t)__cvta_generic_to_shared(&s_best[part * kLpTop + at]);
        if (parts > 1) asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(to) : "r"(to));
        asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(to), "l"(k) : "memory");
      }
    }
    if (n < top && tid < top && tid >= n) {   // a share of fewer words
      uint32_t to = (uint32_t)__cvta_generic_to_shared(&s_best[part * kLpTop + tid]);
      if (parts > 1) asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(to) : "r"(to));
      asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(to), "l"((uint64_t)0u) : "memory");
    }
  } else if (parts > 1) {
    cluster_wait();
  }
  if (w == kLpWarps - 1) {   // (while the first warps order words)
    const LpJoined c = lp_join<kLpWarps>(s_join, kLpWarps);
    if (parts == 1) {
      const LpWhole whole(c);
      if (lane == 0) {
        s_whole = whole;
        tell(whole);
      }
    } else if (lane == 0) {
      uint32_t to = (uint32_t)__cvta_generic_to_shared(&s_part[part]);
      asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(to) : "r"(to));
      asm volatile("st.shared::cluster.v2.f64 [%0], {%1, %2};" ::"r"(to), "d"(c.s), "d"(c.t) : "memory");
      asm volatile("st.shared::cluster.v2.b32 [%0], {%1, %2};" ::"r"(to + 16), "r"(__float_as_uint(c.m)), "r"(c.rank) : "memory");
    }
  }
  if (parts == 1) {
    if (top == 0) return;
    __syncthreads();
    if (tid < top) {   // in order already
      const uint64_t k = s_best[tid];
      if (k != 0u) {
        a.best[r * top + tid] = (int)~(uint32_t)k;
        a.best_lp[r * top + tid] = s_whole.value(lp_value((uint32_t)(k >> 32)));
      }
    }
    return;
  }
  cluster_sync();
  if (part != 0) return;

  // ---------------- the row of several CTAs
  if (w * 32 < max(1, parts * top)) {   // whole warps
    const LpWhole whole(lp_join<kLpCluster>(s_part, parts));
    if (tid == 0) tell(whole);
    if (tid < parts * top) {
      const int p = tid / top;
      const uint64_t k = s_best[p * kLpTop + tid - p * top];
      int at = 0;
      for (int q = 0; q < parts; ++q)
        for (int j = 0; j < top; ++j) at += s_best[q * kLpTop + j] > k;
      if (k != 0u && at < top) {
        a.best[r * top + at] = (int)~(uint32_t)k;
        a.best_lp[r * top + at] = whole.value(lp_value((uint32_t)(k >> 32)));
      }
    }
  }
}

template <typename T>
static int log_probs_launch(LogProbArgs a, int64_t rows, int sms, cudaStream_t s) {
  // CTAs of a row: as many as keep all rows resident at once (four per SM), each with a piece a thread at least
  const int pieces = (a.V + LpVec<T>::N - 1) / LpVec<T>::N;
  a.parts = 1;
  while (a.parts < kLpCluster && rows * a.parts * 2 <= 4 * sms && pieces / (a.parts * 2) >= 256) a.parts *= 2;
  // Threads of a CTA: 512 where CTAs are fewer than SMs (8 rows of 131072 fp32, 20 alternatives: 11.1 us against 15.2 with 256); 128 for rows that are short, or not too long and many, so that
  // a row's end, where most threads wait, holds up fewer of them (us, 128 | 256: 4096 rows of 2000 fp16, 1 alternative 23 | 38, of 8000 bf16 33 | 49, of 50257 85 | 96, with 20: 110 | 120;
  // 700 rows of 32000 fp32 22 | 27; 760 of 131072 bf16 52 | 48).
  const bool wide = rows * a.parts <= sms && pieces / a.parts >= 512;
  const bool narrow = a.parts == 1 && (pieces < 1024 || (pieces <= 8192 && rows >= 4 * (int64_t)sms));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(rows * a.parts));
  cfg.blockDim = dim3(wide ? 512 : narrow ? 128 : 256);
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = a.parts;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  auto k = a.top > 1 ? (wide ? log_probs_kernel<T, 512, true> : narrow ? log_probs_kernel<T, 128, true> : log_probs_kernel<T, 256, true>)
                     : (wide ? log_probs_kernel<T, 512, false> : narrow ? log_probs_kernel<T, 128, false> : log_probs_kernel<T, 256, false>);
  TSB_CUDA(cudaLaunchKernelEx(&cfg, k, a));
  return 1;
}

}  // namespace tsb

using namespace tsb;

extern "C" {

int TSB200_TokenLogProbs(int device, int dtype, float* logprobs, float* entropy, int32_t* ranks, int32_t* top_tokens, float* top_logprobs, int top, const void* logits,
                         int64_t logits_row, const int32_t* tokens, int64_t rows, int V, void* stream) {
  TSB_CHECK(dtype == TSB200_F32 || is_16bit(dtype), "token_log_probs: unsupported dtype %d", dtype);
  TSB_CHECK(rows >= 0 && rows < ((int64_t)1 << 31), "token_log_probs: %lld rows", (long long)rows);
  TSB_CHECK(V > 0 && V <= (1 << 30), "token_log_probs: %d words", V);
  TSB_CHECK(top >= 0 && top <= kLpTop && top <= V, "token_log_probs: %d alternatives of %d words, at most %d", top, V, kLpTop);
  TSB_CHECK(rows == 0 || (logits && tokens && logprobs && entropy && ranks && (top == 0 || (top_tokens && top_logprobs))), "token_log_probs: null pointer");
  TSB_CHECK((uintptr_t)logits % dtype_size(dtype) == 0 && ((uintptr_t)tokens | (uintptr_t)logprobs | (uintptr_t)entropy | (uintptr_t)ranks | (uintptr_t)top_tokens | (uintptr_t)top_logprobs) % 4 == 0,
            "token_log_probs: pointers lie between elements");
  if (rows == 0) return 1;
  KeepDevice keep;
  DeviceState* st;
  TSB_TRY(use_device(device, &st));
  cudaStream_t s = pick_stream(st, stream);
  LogProbArgs a{};
  a.x = logits; a.x_row = logits_row; a.tokens = tokens; a.V = V; a.top = top;
  a.lp = logprobs; a.entropy = entropy; a.rank = ranks; a.best = top_tokens; a.best_lp = top_logprobs;
  if (dtype == TSB200_F32) TSB_TRY(log_probs_launch<float>(a, rows, st->sm_count, s));
  else if (dtype == TSB200_F16) TSB_TRY(log_probs_launch<__half>(a, rows, st->sm_count, s));
  else TSB_TRY(log_probs_launch<__nv_bfloat16>(a, rows, st->sm_count, s));
  count_launch(device);
  return check_launch("token_log_probs");
}

}  // extern "C"
