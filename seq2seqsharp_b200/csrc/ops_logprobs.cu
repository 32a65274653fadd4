// Log probabilities of given tokens, with the entropy of their rows, their rank and the most likely alternatives:
//   m = max x,  S = sum e^(x - m),  T = sum (x - m) e^(x - m):  lp(t) = x_t - m - log S,  H = log S - T / S,
//   rank = #{j: x_j > x_t, or x_j = x_t and j < t},  best = the `top` largest logits, the lower index first among equal ones.
//
// One pass over the logits.  A thread keeps a running maximum and both sums of its share in fp32, with powers of two (x log2 e is taken against the rounded m log2 e, any
// reference being as good as the maximum itself); what threads have is joined in 64 bits, so that a probability near 1 keeps its digits (log S of a sum a little over 1).
// The threads' maxima are also a bound for the alternatives: where r = ceil(top / warps) lanes of ceil(top / r) warps have a logit of at least B, `top` words have, and only threads
// whose maximum is at least B look through their share again, in L2.  What they find (some 50 words for random logits) is ordered by counting.  Should that be over
// kLpRoom (many equal logits, nearly all of them -infinity), the bound is raised to the top-th largest (logit, index) by eight histograms of eight bits.
//
// Few rows: a cluster of up to eight CTAs shares a row, and the first one joins what all have pushed to it.  Many rows: a CTA per row.
#include <math_constants.h>

#include "kernels.cuh"

namespace tsb {

constexpr int kLpThreads = 256, kLpWarps = kLpThreads / 32;
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
__device__ __forceinline__ float lp_exp2(float v) {   // off by 2 ulp; 0 for -infinity
  float r;
  asm("ex2.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// whole numbers that order as the numbers do, a zero having one sign; NaN comes last
__device__ __forceinline__ uint32_t lp_order(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  return v != v ? 0u : (b & 0x80000000u ? ~b : b | 0x80000000u);
}
__device__ __forceinline__ float lp_value(uint32_t o) { return o == 0u ? CUDART_NAN_F : __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }
__device__ __forceinline__ uint64_t lp_key(float v, int j) { return ((uint64_t)lp_order(v) << 32) | (uint32_t)~j; }

template <typename T> struct LpVec {
  static constexpr int N = 16 / (int)sizeof(T);
  uint4 raw;
  __device__ __forceinline__ float get(int e) const;
};
template <> __device__ __forceinline__ float LpVec<float>::get(int e) const { return __uint_as_float(e == 0 ? raw.x : e == 1 ? raw.y : e == 2 ? raw.z : raw.w); }
template <> __device__ __forceinline__ float LpVec<__half>::get(int e) const {
  const uint32_t p = (e >> 1) == 0 ? raw.x : (e >> 1) == 1 ? raw.y : (e >> 1) == 2 ? raw.z : raw.w;
  const float2 f = Pair16<__half>::get(p);
  return e & 1 ? f.y : f.x;
}
template <> __device__ __forceinline__ float LpVec<__nv_bfloat16>::get(int e) const {
  const uint32_t p = (e >> 1) == 0 ? raw.x : (e >> 1) == 1 ? raw.y : (e >> 1) == 2 ? raw.z : raw.w;
  return __uint_as_float(e & 1 ? p & 0xffff0000u : p << 16);
}

// A row as pieces of 16 bytes on their boundaries: the first one begins `off` elements in front of the row
template <typename T>
struct LpRow {
  static constexpr int N = LpVec<T>::N;
  const T* x;
  int off, V;
  __device__ __forceinline__ LpRow(const T* p, int v) : x(p), off((int)(((uintptr_t)p & 15) / sizeof(T))), V(v) {}
  __device__ __forceinline__ int pieces() const { return (int)(((int64_t)V + off + N - 1) / N); }
  __device__ __forceinline__ int first(int v) const { return v * N - off; }   // index of a piece's first element
  __device__ __forceinline__ bool whole(int v) const { return first(v) >= 0 && (int64_t)first(v) + N <= V; }
  __device__ __forceinline__ LpVec<T> load(int v) const {
    LpVec<T> r;
    const int j0 = first(v);
    if (whole(v)) {
      r.raw = *reinterpret_cast<const uint4*>(x + j0);
    } else {
      // what is not there is -infinity
      struct __align__(16) { T e[N]; } t;
#pragma unroll
      for (int e = 0; e < N; ++e) t.e[e] = j0 + e >= 0 && j0 + e < V ? x[j0 + e] : from_f<T>(-CUDART_INF_F);
      r.raw = *reinterpret_cast<const uint4*>(&t);
    }
    return r;
  }
};

// Exponents are taken as x log2 e - m log2 e with the second product rounded, one instruction a logit; from 2e38 on (a mask of the type's lowest value, over a whole
// share) these products leave fp32 and the difference comes first.
__device__ __forceinline__ bool lp_far(float m) { return !(fabsf(m) < 2e38f); }
// exponent of 2 between two maxima, at most 0; 2^-1000 is 0, and so is its product with the exponent
__device__ __forceinline__ float lp_gap(float m, float to) {
  const float d = lp_far(m) || lp_far(to) ? __fmul_rn(m - to, kLog2e) : __fsub_rn(__fmul_rn(m, kLog2e), __fmul_rn(to, kLog2e));
  return lp_max_nan(d, -1000.0f);
}
struct LpSums {
  float m, s, t;   // maximum; sums, over the logits, of 2^exponent and of the exponent times it
  __device__ __forceinline__ void raise(float to) {   // to > m
    if (m > -CUDART_INF_F) {
      const float d = lp_gap(m, to), f = lp_exp2(d);
      t = f * fmaf(d, s, t);
      s *= f;
    }
    m = to;
  }
};
// the same joined, in 64 bits
struct LpJoined {
  double s, t;
  float m;
  int rank;
};
__device__ __forceinline__ void lp_rebase(double& s, double& t, float m, float to) {   // both are maxima, m <= to
  if (m == to || !(m > -CUDART_INF_F)) return;   // (a share of -infinity has sums of 0, or NaN)
  const float d = lp_gap(m, to);
  const double f = (double)lp_exp2(d);
  t = f * (t + (double)d * s);
  s *= f;
}
__device__ __forceinline__ void lp_join(LpJoined& c, LpJoined o) {
  const float m = fmaxf(c.m, o.m);
  lp_rebase(c.s, c.t, c.m, m);
  lp_rebase(o.s, o.t, o.m, m);
  c = LpJoined{c.s + o.s, c.t + o.t, m, c.rank + o.rank};
}

__device__ __forceinline__ double lp_shfl_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <typename T>
__global__ void __launch_bounds__(kLpThreads) log_probs_kernel(LogProbArgs a) {
  __shared__ LpJoined s_join[kLpWarps];
  __shared__ LpJoined s_part[kLpCluster];            // (first CTA) of every CTA of the row
  __shared__ uint32_t s_bound[kLpWarps];
  __shared__ uint64_t s_words[kLpRoom];
  __shared__ uint64_t s_best[kLpCluster * kLpTop];   // (first CTA) of every CTA of the row, 0: none
  __shared__ uint32_t s_hist[256];
  __shared__ uint64_t s_prefix;
  __shared__ int s_count, s_need;

  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const int parts = a.parts, part = (int)(blockIdx.x % parts);
  const int64_t r = (int64_t)(blockIdx.x / parts);
  if (parts > 1) {   // the first CTA runs; waited for in front of the pushes
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  }
  const LpRow<T> row(reinterpret_cast<const T*>(a.x) + r * a.x_row, a.V);
  constexpr int N = LpVec<T>::N;
  const int all = row.pieces(), v0 = (int)((int64_t)all * part / parts), v1 = (int)((int64_t)all * (part + 1) / parts);
  const int token = a.tokens[r];

  LpSums mine{-CUDART_INF_F, 0.0f, 0.0f};
  int rank = 0;
  LpVec<T> x[kLpUnroll];
  auto fetch = [&](int v) {
#pragma unroll
    for (int u = 0; u < kLpUnroll; ++u)
      if (v + u * kLpThreads < v1) x[u] = row.load(v + u * kLpThreads);
  };
  fetch(v0 + tid);
  // what the token's rank is counted against: x >= before in front of it, x >= behind behind it (a NaN: never)
  const bool given = token >= 0 && token < a.V;
  const float xt = given ? to_f<T>(row.x[token]) + 0.0f : CUDART_NAN_F;
  const float behind = xt < CUDART_INF_F ? nextafterf(xt, CUDART_INF_F) : CUDART_NAN_F;

  for (int v = v0 + tid; v < v1; v += kLpUnroll * kLpThreads) {
    if (v != v0 + tid) fetch(v);
    float top = -CUDART_INF_F;
#pragma unroll
    for (int u = 0; u < kLpUnroll; ++u)
      if (v + u * kLpThreads < v1) {
#pragma unroll
        for (int e = 0; e < N; ++e) top = fmaxf(top, x[u].get(e));
      }
    if (top > mine.m) mine.raise(top);
    float gs = 0.0f, gt = 0.0f;
    auto add = [&](auto exponent) {
#pragma unroll
      for (int u = 0; u < kLpUnroll; ++u) {
        if (v + u * kLpThreads >= v1) break;
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float d = lp_max_nan(exponent(x[u].get(e)), -1000.0f), p = lp_exp2(d);
          gs += p;
          gt = fmaf(d, p, gt);
        }
      }
    };
    const float m = mine.m > -CUDART_INF_F ? mine.m : 0.0f, ref = __fmul_rn(m, kLog2e);   // nothing but -infinity (and NaN) yet: sums of 0 (of NaN)
    if (!lp_far(m)) add([&](float y) { return fmaf(y, kLog2e, -ref); });
    else add([&](float y) { return (y - m) * kLog2e; });
    mine.s += gs;
    mine.t += gt;
#pragma unroll
    for (int u = 0; u < kLpUnroll; ++u) {
      const int at = v + u * kLpThreads;
      if (at >= v1) break;
      const int j0 = row.first(at);
      if (row.whole(at) && (j0 > token || j0 + N <= token)) {
        const float against = j0 > token ? behind : xt;
#pragma unroll
        for (int e = 0; e < N; ++e) rank += x[u].get(e) >= against;
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const int j = j0 + e;
          const float y = x[u].get(e);
          rank += j >= 0 && j < a.V && (y > xt || (y == xt && j < token));
        }
      }
    }
  }

  // ---------------- the CTA's sums, against its maximum
  const uint32_t mine_o = lp_order(mine.m), warp_o = __reduce_max_sync(0xffffffffu, mine_o);
  {
    const float m = lp_value(warp_o);
    double s = mine.s, t = mine.t;
    lp_rebase(s, t, mine.m, m);
    s = lp_shfl_sum(s);
    t = lp_shfl_sum(t);
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
      if (bound <= lp_order(-CUDART_INF_F)) bound = 0u;   // threads without a number have this maximum too: every word counts
    }
    // every element of the thread's share
    auto look = [&](bool any, auto f) {
      if (!any) return;
      for (int v = v0 + tid; v < v1; v += kLpUnroll * kLpThreads) {
        LpVec<T> y[kLpUnroll];
#pragma unroll
        for (int u = 0; u < kLpUnroll; ++u)
          if (v + u * kLpThreads < v1) y[u] = row.load(v + u * kLpThreads);
#pragma unroll
        for (int u = 0; u < kLpUnroll; ++u) {
          const int v_at = v + u * kLpThreads;
          if (v_at >= v1) break;
          const int j0 = row.first(v_at);
#pragma unroll
          for (int e = 0; e < N; ++e)
            if (j0 + e >= 0 && j0 + e < a.V) f(lp_key(y[u].get(e), j0 + e));
        }
      }
    };
    uint64_t least = (uint64_t)bound << 32;
    auto take = [&](uint64_t k) {
      if (k < least) return;
      const int at = atomicAdd(&s_count, 1);
      if (at < kLpRoom) s_words[at] = k;
    };
    look(mine_o >= bound, take);
    __syncthreads();
    if (s_count > kLpRoom) {
      // the top-th largest key, eight bits at a time
      if (tid == 0) {
        s_prefix = 0u;
        s_need = top;
      }
      for (int shift = 56; shift >= 0; shift -= 8) {
        for (int i = tid; i < 256; i += kLpThreads) s_hist[i] = 0u;
        __syncthreads();
        const uint64_t prefix = s_prefix;
        look(true, [&](uint64_t k) {
          if (shift == 56 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&s_hist[(k >> shift) & 255], 1u);
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
      look(true, take);
      __syncthreads();
    }
    if (parts > 1) cluster_wait();
    // in order: a key's place is the number of larger ones.  To the first CTA of the row.
    const int n = min(s_count, kLpRoom);
    for (int i = tid; i < n; i += kLpThreads) {
      const uint64_t k = s_words[i];
      int at = 0;
      for (int j = 0; j < n; ++j) at += s_words[j] > k;
      if (at < top) {
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
  if (tid == 0) {
    LpJoined c = s_join[0];
    for (int i = 1; i < kLpWarps; ++i) lp_join(c, s_join[i]);
    uint32_t to = (uint32_t)__cvta_generic_to_shared(&s_part[part]);
    if (parts > 1) asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(to) : "r"(to));
    asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(to), "d"(c.s) : "memory");
    asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(to + 8), "d"(c.t) : "memory");
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 16), "f"(c.m) : "memory");
    asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(to + 20), "r"(c.rank) : "memory");
  }
  if (parts > 1) cluster_sync();
  else __syncthreads();
  if (part != 0) return;

  // ---------------- the row
  if (w == 0 || tid < parts * top) {
    LpJoined c = s_part[0];
    for (int i = 1; i < parts; ++i) lp_join(c, s_part[i]);
    const bool none = !(c.m > -CUDART_INF_F);   // nothing but -infinity and NaN
    if (!none && !lp_far(c.m)) {
      // The maximum's own exponent is what rounding left of it, and its power of two is off by 2 ulp of 1: as much as all other words have where it is nearly certain
      const float own = fmaf(c.m, kLog2e, -__fmul_rn(c.m, kLog2e));
      c.s += exp2((double)own) - (double)lp_exp2(own);
    }
    const double ln2 = 0.693147180559945309417, log_s = none ? CUDART_NAN : log(c.s), ref = (double)__fmul_rn(c.m, kLog2e);
    // rounding may leave a little over 0 of a certain token
    auto value = [&](float v) {
      const double l = (lp_far(c.m) ? (double)v - (double)c.m : ((double)v * (double)kLog2e - ref) * ln2) - log_s;
      return (float)(l > 0.0 ? 0.0 : l);
    };
    if (tid == 0) {
      a.lp[r] = given ? value(xt) : token < 0 ? 0.0f : CUDART_NAN_F;
      a.rank[r] = given ? c.rank : -1;
      const double h = log_s - c.t / c.s * ln2;
      a.entropy[r] = (float)(h < 0.0 ? 0.0 : h);
    }
    if (tid < parts * top) {
      const int p = tid / top;
      const uint64_t k = s_best[p * kLpTop + tid - p * top];
      int at = 0;
      for (int q = 0; q < parts; ++q)
        for (int j = 0; j < top; ++j) at += s_best[q * kLpTop + j] > k;
      if (k != 0u && at < top) {
        a.best[r * top + at] = (int)~(uint32_t)k;
        a.best_lp[r * top + at] = value(lp_value((uint32_t)(k >> 32)));
      }
    }
  }
}

template <typename T>
static int log_probs_launch(LogProbArgs a, int64_t rows, int sms, cudaStream_t s) {
  // CTAs of a row: as many as keep all rows resident at once (two per SM), each with a round of its threads' loads at least
  const int pieces = (a.V + LpVec<T>::N - 1) / LpVec<T>::N;
  a.parts = 1;
  while (a.parts < kLpCluster && rows * a.parts * 2 <= 2 * sms && pieces / (a.parts * 2) >= kLpThreads) a.parts *= 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(rows * a.parts));
  cfg.blockDim = dim3(kLpThreads);
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = a.parts;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  TSB_CUDA(cudaLaunchKernelEx(&cfg, log_probs_kernel<T>, a));
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
