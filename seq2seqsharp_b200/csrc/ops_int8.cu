// Rows of 8-bit integers with a scale per row, as the 8-bit linears (gemm_int8.cu) take them: out of the norm in front of a block (with the
// residual's addition), and out of an activation (gated or not, or none at all).
//
//   norm: h = t(x + residual), v = h gamma, scale = max|v| / (127 sqrt(mean(h^2) + eps));   rows: v = act(a) gate, scale = max|v| / 127
//   both: q = rint(127 v / max|v|)
// The root of the norm is the same for a whole row and divides out of q, so that the sum of squares and the maximum are taken in one pass, with one
// barrier, and the bytes do not depend on the order of the sum.  h is rounded to the model type t first: it is the stream that the next layers see.
// v, sums and maxima are fp32; 127 v / max|v| has one rounding in v, one in 127 / max|v| and one in the product's sum with 1.5 2^23, whose low byte
// is the rounded integer (half to even).  A row whose values or squares leave fp32 (infinities, NaN) gets the scale NaN and bytes of 0.
//
// Every tensor is read once (rows beyond 32768 elements twice): a row lies in registers, 8 to 32 elements a thread.  With 32 (rows beyond 16384; the ring's norms without a residual) what does not
// fit into 64 registers goes to the stack, 46 to 316 bytes a thread: 2000 rows of 20000, gated silu, 83 us where the bytes take 31.  Accesses of 16 bytes where all rows start on such a boundary,
// of two elements or of one otherwise (16000 rows of 1001 bf16 with a residual 49 us, bytes 17).
// What bounds it: bytes where nothing but products is taken of an element (8192 rows of 8192 bf16, gated relu, 51 us, bytes 51), with silu its two instructions on the XU pipe (59; 55 % of
// that pipe, 65 % of the issue slots), with gelu erff (98); few rows the launch (8 of 11008 3.1 us).
#include <type_traits>

#include "stream_common.cuh"

namespace tsb {

struct Int8Rows {
  int8_t* q;           // rows of stride q_row
  float* scale;        // [rows]
  void* h;             // norm with a residual: the sum, rows of stride h_row; may be x or residual
  const void* a;       // norm: x
  const void* b;       // norm: residual; rows: gate; may be null
  const void* gamma;   // norm
  int64_t q_row, h_row, a_row, b_row;
  int64_t rows;
  int d;
  float eps;
  int act;
};

template <typename T, int N> struct __align__(N * sizeof(T)) Int8Piece { T e[N]; };

// silu, sigmoid: the power of two (off by 2 ulp, its exponent by one of itself) and the reciprocal (1 ulp) by the approximate instructions: a few 2^-22 of what they return, where
// a step of q is 2^-7 of the row's largest value
__device__ __forceinline__ float int8_sigmoid(float v) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(v * -1.44269504088896341f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return r;
}
template <int ACT>
__device__ __forceinline__ float int8_act(float v) {
  if constexpr (ACT == TSB200_ACT_SILU) return v * int8_sigmoid(v);
  else if constexpr (ACT == TSB200_ACT_SIGMOID) return int8_sigmoid(v);
  else return ep_act(v, ACT);
}

// four of them as bytes: |v inv| <= 127 (1 + 2^-22), so that the sum's low byte is the rounded integer
__device__ __forceinline__ uint32_t int8_low(float v, float inv) { return __float_as_uint(fmaf(v, inv, 12582912.0f)); }
__device__ __forceinline__ uint32_t int8_pack(const float* v, float inv) {
  const uint32_t lo = __byte_perm(int8_low(v[0], inv), int8_low(v[1], inv), 0x0040), hi = __byte_perm(int8_low(v[2], inv), int8_low(v[3], inv), 0x0040);
  return __byte_perm(lo, hi, 0x5410);
}

// larger of what is there and two values, without their signs; a NaN stays one
__device__ __forceinline__ float int8_top(float top, float a, float b) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(top), "f"(a), "f"(b));
  return r;
}
template <int N>
__device__ __forceinline__ float int8_top(float top, const float* v) {
#pragma unroll
  for (int e = 0; e + 1 < N; e += 2) top = int8_top(top, v[e], v[e + 1]);
  return N % 2 ? int8_top(top, v[N - 1], v[N - 1]) : top;
}
// sum of squares (of a norm) and maximum (as bits: those of a NaN are larger than all) over the threads of a row: a warp, or the CTA
// (turn: 0 and 1 in alternation where a CTA has several rows, so that one barrier a row is enough)
template <bool WARP, int NORM>
__device__ __forceinline__ uint32_t int8_reduce(float& sum, float largest, int turn = 0) {
  uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(largest) & 0x7fffffffu);
  if constexpr (NORM) sum = warp_sum(sum);
  if constexpr (!WARP) {
    __shared__ float s_sum[2][32];
    __shared__ uint32_t s_top[2][32];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, warps = blockDim.x >> 5;
    if (lane == 0) {
      if (NORM) s_sum[turn][w] = sum;
      s_top[turn][w] = top;
    }
    __syncthreads();
    if constexpr (NORM) sum = warp_sum(lane < warps ? s_sum[turn][lane] : 0.0f);
    top = __reduce_max_sync(0xffffffffu, lane < warps ? s_top[turn][lane] : 0u);
  }
  return top;
}

// What a row's statistics make of it: the factor of v, and the scale (written by one thread).  `up`: a power of two that v is multiplied by first, so that 127 / max|v|
// stays below infinity where the row is nearly zero.
template <int NORM>
__device__ __forceinline__ float int8_finish(const Int8Rows& p, int64_t r, float sum, uint32_t top, bool first, float& up) {
  const float mx = __uint_as_float(top);
  const bool fine = top < 0x7f800000u && (!NORM || sum < INFINITY);   // (a NaN is not below)
  up = mx < 1e-27f ? 0x1p60f : 1.0f;
  if (first) {
    float s = mx;
    if constexpr (NORM) s *= 1.0f / sqrtf(sum / (float)p.d + p.eps);
    p.scale[r] = fine ? (mx > 0.0f ? s / 127.0f : 0.0f) : NAN;   // (eps may be 0)
  }
  return fine && mx > 0.0f ? 127.0f / (mx * up) : 0.0f;
}

// Norms with an eps below 2^-100 (NORM 2; 1: the others).  A result is of ordinary size then however small its row is, but squares vanish below 1e-23 and have few digits above, and
// products with the gain below 1e-38.  Such rows are taken again, in 64 bits, by the threads that wrote them: the scale where the mean of the squares is below 2^-100, the bytes too where
// max|v| is, so that bytes do not depend on the order of a sum.  With a larger eps squares that vanish are nothing beside it, and what a product's last step of 2^-149 makes of the result is
// below 2^-99.  Kernels of their own: in the ones for every eps this cost 81 -> 87 us (16384 rows of 4096 bf16) and 32 -> 41 (16000 of 1001) in registers and issue slots.
constexpr float kInt8Small = 0x1p-100f;
template <typename T, bool WARP>
__device__ __noinline__ void int8_small_row(const T* h, const T* gamma, int8_t* q, float* scale, int d, float eps, bool bytes) {
  if constexpr (WARP) __syncwarp();
  else __syncthreads();   // the row's sums and first bytes are written
  const int i0 = threadIdx.x, step = WARP ? 32 : (int)blockDim.x;
  double sum = 0.0, top = 0.0;
  for (int i = i0; i < d; i += step) {
    const double x = (double)to_f<T>(h[i]);
    sum = fma(x, x, sum);
    top = fmax(top, fabs(x * (double)to_f<T>(gamma[i])));   // (exact)
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
  }
  if constexpr (!WARP) {
    __shared__ double s_sum[32], s_top[32];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, warps = blockDim.x >> 5;
    if (lane == 0) {
      s_sum[w] = sum;
      s_top[w] = top;
    }
    __syncthreads();
    sum = top = 0.0;
    for (int i = 0; i < warps; ++i) {
      sum += s_sum[i];
      top = fmax(top, s_top[i]);
    }
    __syncthreads();   // the CTA's next row may come here
  }
  if (threadIdx.x == 0) *scale = top > 0.0 ? (float)(top / (127.0 * sqrt(sum / d + (double)eps))) : 0.0f;
  if (!bytes) return;
  const double inv = top > 0.0 ? 127.0 / top : 0.0;
  for (int i = i0; i < d; i += step) q[i] = (int8_t)__double2int_rn((double)to_f<T>(h[i]) * (double)to_f<T>(gamma[i]) * inv);
}
// 0: the row is fine, 1: its scale, 2: its bytes too (all threads of a row have the same sum and maximum)
__device__ __forceinline__ int int8_small(const Int8Rows& p, float sum, uint32_t top) { return __uint_as_float(top) < kInt8Small ? 2 : sum < kInt8Small * (float)p.d ? 1 : 0; }
template <typename T, bool WARP>
__device__ __forceinline__ void int8_small_row(const Int8Rows& p, int64_t r, int what) {
  int8_small_row<T, WARP>(reinterpret_cast<const T*>(p.b ? p.h : p.a) + r * (p.b ? p.h_row : p.a_row), reinterpret_cast<const T*>(p.gamma), p.q + r * p.q_row, p.scale + r, p.d, p.eps,
                          what == 2);
}

template <typename T, int VEC, int NC, int NORM, bool WARP>
__global__ void __launch_bounds__(1024) int8_rows_kernel(Int8Rows p) {
  const int64_t r = WARP ? (int64_t)blockIdx.x * blockDim.y + threadIdx.y : (int64_t)blockIdx.x;
  if (r >= p.rows) return;   // (whole warps)
  typedef Int8Piece<T, VEC> Piece;
  const T* a = reinterpret_cast<const T*>(p.a) + r * p.a_row;
  const T* b = reinterpret_cast<const T*>(p.b) + r * p.b_row;
  const bool two = p.b != nullptr;
  const int step = (int)blockDim.x * VEC, i0 = (int)threadIdx.x * VEC;
  Piece pa[NC], pb[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int i = i0 + c * step;
    if (i < p.d) {
      pa[c] = *reinterpret_cast<const Piece*>(a + i);
      if (two) pb[c] = *reinterpret_cast<const Piece*>(b + i);
    }
  }
  float v[NC][VEC];
  float sum = 0.0f;
  float largest = 0.0f;
  if constexpr (NORM) {
    T* h = reinterpret_cast<T*>(p.h) + r * p.h_row;
    const T* gamma = reinterpret_cast<const T*>(p.gamma);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int i = i0 + c * step;
      if (i >= p.d) continue;
      const Piece g = *reinterpret_cast<const Piece*>(gamma + i);
      if (two) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) pa[c].e[e] = from_f<T>(to_f<T>(pa[c].e[e]) + to_f<T>(pb[c].e[e]));
        *reinterpret_cast<Piece*>(h + i) = pa[c];
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float x = to_f<T>(pa[c].e[e]);
        sum = fmaf(x, x, sum);
        v[c][e] = x * to_f<T>(g.e[e]);
      }
    }
  } else {
    auto apply = [&](auto act) {
#pragma unroll
      for (int c = 0; c < NC; ++c)
        if (i0 + c * step < p.d) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            v[c][e] = int8_act<decltype(act)::value>(to_f<T>(pa[c].e[e]));
            if (two) v[c][e] *= to_f<T>(pb[c].e[e]);
          }
        }
    };
    switch (p.act) {
      case TSB200_ACT_RELU: apply(std::integral_constant<int, TSB200_ACT_RELU>()); break;
      case TSB200_ACT_SILU: apply(std::integral_constant<int, TSB200_ACT_SILU>()); break;
      case TSB200_ACT_LEAKYRELU: apply(std::integral_constant<int, TSB200_ACT_LEAKYRELU>()); break;
      case TSB200_ACT_GELU: apply(std::integral_constant<int, TSB200_ACT_GELU>()); break;
      case TSB200_ACT_SIGMOID: apply(std::integral_constant<int, TSB200_ACT_SIGMOID>()); break;
      default: apply(std::integral_constant<int, TSB200_ACT_NONE>()); break;
    }
  }
#pragma unroll
  for (int c = 0; c < NC; ++c)
    if (i0 + c * step < p.d) largest = int8_top<VEC>(largest, v[c]);
  const uint32_t top = int8_reduce<WARP, NORM>(sum, largest);
  float up;
  const float inv = int8_finish<NORM>(p, r, sum, top, threadIdx.x == 0, up);
  int8_t* q = p.q + r * p.q_row;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int i = i0 + c * step;
    if (i >= p.d) continue;
    if (up != 1.0f || inv == 0.0f) {   // nearly or all zeros, or not finite (a factor of 0 alone would leave NaN)
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[c][e] = inv == 0.0f ? 0.0f : v[c][e] * up;
    }
    if constexpr (VEC == 8) *reinterpret_cast<uint2*>(q + i) = make_uint2(int8_pack(v[c], inv), int8_pack(v[c] + 4, inv));
    else if constexpr (VEC == 4) *reinterpret_cast<uint32_t*>(q + i) = int8_pack(v[c], inv);
    else if constexpr (VEC == 2) *reinterpret_cast<uint16_t*>(q + i) = (uint16_t)__byte_perm(int8_low(v[c][0], inv), int8_low(v[c][1], inv), 0x0040);
    else q[i] = (int8_t)int8_low(v[c][0], inv);
  }
  if constexpr (NORM == 2) {
    if (const int what = int8_small(p, sum, top)) int8_small_row<T, WARP>(p, r, what);
  }
}

// Rows of more than 32768 elements: read twice, the second time out of L2 (an element by the thread that wrote its sum)
template <typename T, int NORM>
__global__ void __launch_bounds__(1024) int8_long_rows_kernel(Int8Rows p) {
  const int64_t r = blockIdx.x;
  const T* a = reinterpret_cast<const T*>(p.a) + r * p.a_row;
  const T* b = reinterpret_cast<const T*>(p.b) + r * p.b_row;
  T* h = reinterpret_cast<T*>(p.h) + r * p.h_row;
  const bool two = p.b != nullptr;
  float sum = 0.0f;
  float largest = 0.0f;
  auto value = [&](int i) {
    float v = ep_act(to_f<T>(a[i]), p.act);
    return two ? v * to_f<T>(b[i]) : v;
  };
  for (int i = threadIdx.x; i < p.d; i += 1024) {
    float v;
    if constexpr (NORM) {
      T s = a[i];
      if (two) {
        s = from_f<T>(to_f<T>(s) + to_f<T>(b[i]));
        h[i] = s;
      }
      const float x = to_f<T>(s);
      sum = fmaf(x, x, sum);
      v = x * to_f<T>(reinterpret_cast<const T*>(p.gamma)[i]);
    } else {
      v = value(i);
    }
    largest = int8_top(largest, v, v);
  }
  const uint32_t top = int8_reduce<false, NORM>(sum, largest);
  float up;
  const float inv = int8_finish<NORM>(p, r, sum, top, threadIdx.x == 0, up);
  for (int i = threadIdx.x; i < p.d; i += 1024) {
    float v;
    if constexpr (NORM) v = to_f<T>(two ? h[i] : a[i]) * to_f<T>(reinterpret_cast<const T*>(p.gamma)[i]);
    else v = value(i);
    p.q[r * p.q_row + i] = inv == 0.0f ? (int8_t)0 : (int8_t)int8_low(v * up, inv);
  }
  if constexpr (NORM == 2) {
    if (const int what = int8_small(p, sum, top)) int8_small_row<T, false>(p, r, what);
  }
}

// Many rows that start on 16 bytes: CTAs walk over rows, whose inputs a ring of bulk copies brings into shared memory several rows ahead.  All threads have read a row when its
// sums are joined, so that the barrier which does that also gives the row's place to the next copy.
struct Int8Ring {
  int stages, bytes;      // of a row and input
  unsigned wait_limit;
  int* error;
};
template <typename T, int NC, int NORM>
__global__ void __launch_bounds__(512, NC == 1 ? 3 : 2) int8_ring_kernel(Int8Rows p, Int8Ring ring) {
  constexpr int VEC = 16 / (int)sizeof(T);
  typedef Int8Piece<T, VEC> Piece;
  extern __shared__ __align__(128) unsigned char rows_smem[];
  __shared__ __align__(8) uint64_t bars[8];
  __shared__ int s_late[2];   // a thread has given up waiting for a row; in alternation, so that no thread's next row is taken for this one
  const bool two = p.b != nullptr;
  const int per = ring.bytes * (two ? 2 : 1), step = (int)blockDim.x * VEC, i0 = (int)threadIdx.x * VEC;
  auto copy = [&](int64_t r, int s) {   // by one thread
    mbar_expect_tx(bars + s, (unsigned)per);
    bulk_g2s(rows_smem + s * per, reinterpret_cast<const T*>(p.a) + r * p.a_row, (unsigned)ring.bytes, bars + s);
    if (two) bulk_g2s(rows_smem + s * per + ring.bytes, reinterpret_cast<const T*>(p.b) + r * p.b_row, (unsigned)ring.bytes, bars + s);
  };
  int asked = 0;   // copies (of thread 0)
  if (threadIdx.x == 0) {
    for (int s = 0; s < ring.stages; ++s) mbar_init(bars + s, 1);
    s_late[0] = s_late[1] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    for (; asked < ring.stages && blockIdx.x + (int64_t)asked * gridDim.x < p.rows; ++asked) copy(blockIdx.x + (int64_t)asked * gridDim.x, asked);
  }
  Piece g[NORM ? NC : 1];
  if constexpr (NORM) {
#pragma unroll
    for (int c = 0; c < NC; ++c)
      if (i0 + c * step < p.d) g[c] = *reinterpret_cast<const Piece*>(reinterpret_cast<const T*>(p.gamma) + i0 + c * step);
  }
  __syncthreads();
  int s = 0, turn = 0;
  unsigned phase = 0;
  bool small = false;   // rows of the CTA have to be taken again
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x, turn ^= 1) {
    if (!mbar_wait(bars + s, phase, ring.wait_limit)) s_late[turn] = 1;   // what is read then means nothing
    const T* a = reinterpret_cast<const T*>(rows_smem + s * per) + i0;
    const T* b = reinterpret_cast<const T*>(rows_smem + s * per + ring.bytes) + i0;
    float v[NC][VEC];
    float sum = 0.0f;
    float largest = 0.0f;
    if constexpr (NORM) {
      T* h = reinterpret_cast<T*>(p.h) + r * p.h_row + i0;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        if (i0 + c * step >= p.d) continue;
        Piece x = *reinterpret_cast<const Piece*>(a + c * step);
        if (two) {
          const Piece y = *reinterpret_cast<const Piece*>(b + c * step);
#pragma unroll
          for (int e = 0; e < VEC; ++e) x.e[e] = from_f<T>(to_f<T>(x.e[e]) + to_f<T>(y.e[e]));
          *reinterpret_cast<Piece*>(h + c * step) = x;
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float f = to_f<T>(x.e[e]);
          sum = fmaf(f, f, sum);
          v[c][e] = f * to_f<T>(g[c].e[e]);
        }
      }
    } else {
      auto apply = [&](auto act) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          if (i0 + c * step >= p.d) continue;
          const Piece x = *reinterpret_cast<const Piece*>(a + c * step);
#pragma unroll
          for (int e = 0; e < VEC; ++e) v[c][e] = int8_act<decltype(act)::value>(to_f<T>(x.e[e]));
          if (two) {
            const Piece y = *reinterpret_cast<const Piece*>(b + c * step);
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[c][e] *= to_f<T>(y.e[e]);
          }
        }
      };
      switch (p.act) {
        case TSB200_ACT_RELU: apply(std::integral_constant<int, TSB200_ACT_RELU>()); break;
        case TSB200_ACT_SILU: apply(std::integral_constant<int, TSB200_ACT_SILU>()); break;
        case TSB200_ACT_LEAKYRELU: apply(std::integral_constant<int, TSB200_ACT_LEAKYRELU>()); break;
        case TSB200_ACT_GELU: apply(std::integral_constant<int, TSB200_ACT_GELU>()); break;
        case TSB200_ACT_SIGMOID: apply(std::integral_constant<int, TSB200_ACT_SIGMOID>()); break;
        default: apply(std::integral_constant<int, TSB200_ACT_NONE>()); break;
      }
    }
#pragma unroll
    for (int c = 0; c < NC; ++c)
      if (i0 + c * step < p.d) largest = int8_top<VEC>(largest, v[c]);
    const uint32_t top = int8_reduce<false, NORM>(sum, largest, turn);
    if (*(volatile int*)&s_late[turn]) {
      // all leave; copies in flight land before the CTA gives its shared memory back (a place whose copy is not there takes no other)
      if (threadIdx.x == 0) {
        if (ring.error) *ring.error = 1;
        for (int k = max(0, asked - ring.stages); k < asked; ++k) mbar_wait(bars + k % ring.stages, (unsigned)((k / ring.stages) & 1));
      }
      return;
    }
    if (threadIdx.x == 0 && r + (int64_t)ring.stages * gridDim.x < p.rows) {
      copy(r + (int64_t)ring.stages * gridDim.x, s);
      ++asked;
    }
    if (++s == ring.stages) s = 0, phase ^= 1;
    float up;
    const float inv = int8_finish<NORM>(p, r, sum, top, threadIdx.x == 0, up);
    const bool plain = up == 1.0f && inv > 0.0f;
    int8_t* q = p.q + r * p.q_row + i0;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if (i0 + c * step >= p.d) continue;
      if (!plain) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[c][e] = inv > 0.0f ? v[c][e] * up : 0.0f;
      }
      if constexpr (VEC == 8) *reinterpret_cast<uint2*>(q + c * step) = make_uint2(int8_pack(v[c], inv), int8_pack(v[c] + 4, inv));
      else *reinterpret_cast<uint32_t*>(q + c * step) = int8_pack(v[c], inv);
    }
    if constexpr (NORM == 2) {
      if (const int what = int8_small(p, sum, top)) {
        small = true;
        if (threadIdx.x == 0) p.scale[r] = (float)-what;   // for the end: taken again here, the row cost the others registers
      }
    }
  }
  if (small) {
    __syncthreads();
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
      const float mark = *(volatile float*)(p.scale + r);
      if (mark < 0.0f) int8_small_row<T, false>(p, r, (int)-mark);
    }
  }
}

template <typename T, int VEC, int NC, int NORM>
static int int8_launch(const Int8Rows& p, cudaStream_t s) {
  const int threads = ((p.d + VEC * NC - 1) / (VEC * NC) + 31) / 32 * 32;
  if constexpr (VEC * NC == 8) {
    if (threads == 32) {   // a warp per row, eight rows to a CTA
      int8_rows_kernel<T, VEC, NC, NORM, true><<<(unsigned)((p.rows + 7) / 8), dim3(32, 8), 0, s>>>(p);
      return 1;
    }
  }
  int8_rows_kernel<T, VEC, NC, NORM, false><<<(unsigned)p.rows, threads, 0, s>>>(p);
  return 1;
}

// ctas: per SM; two rows of each are on their way or being worked on
template <typename T, int NC, int NORM>
static int int8_ring(int device, DeviceState* st, const Int8Rows& p, int threads, int ctas, cudaStream_t s) {
  static bool done[kMaxDevices] = {};
  if (!done[device]) {
    TSB_CUDA(cudaFuncSetAttribute(int8_ring_kernel<T, NC, NORM>, cudaFuncAttributeMaxDynamicSharedMemorySize, 128 * 1024));   // (2 rows of 2 x 16384 16-bit elements)
    done[device] = true;
  }
  Int8Ring ring;
  ring.stages = 2;
  ring.bytes = p.d * (int)sizeof(T);
  ring.wait_limit = tc_wait_limit();
  ring.error = tc_error_word(device);
  st->waits = true;
  const int64_t grid = (int64_t)ctas * st->sm_count;
  int8_ring_kernel<T, NC, NORM><<<(unsigned)(grid < p.rows ? grid : p.rows), threads, 2 * ring.bytes * (p.b ? 2 : 1), s>>>(p, ring);
  return 1;
}

template <typename T, int NORM>
static int int8_rows_t(int device, DeviceState* st, const Int8Rows& p, cudaStream_t s) {
  constexpr int kWide = 16 / (int)sizeof(T);
  if (p.d > 32768) {
    int8_long_rows_kernel<T, NORM><<<(unsigned)p.rows, 1024, 0, s>>>(p);
    return 1;
  }
  auto fits = [&](int vec) {
    const uintptr_t al = (uintptr_t)p.a | (uintptr_t)p.b | (uintptr_t)p.h | (uintptr_t)p.gamma;
    const int64_t rows = p.a_row | p.b_row | p.h_row;
    return p.d % vec == 0 && al % (vec * sizeof(T)) == 0 && (p.rows == 1 || rows % vec == 0) && (uintptr_t)p.q % vec == 0 && (p.rows == 1 || p.q_row % vec == 0);
  };
  // elements a thread: 8 where there are few rows (the loads of a row at once), 16 or 32 where a CTA has no more threads
  const int e = p.d <= 8 * 1024 ? 8 : (p.d <= 16 * 1024 ? 16 : 32);
  if constexpr (sizeof(T) == 2) {
    // The ring, where it was the faster one (us, ring | a CTA per row): long rows on two CTAs of 512 threads per SM (8192 of 8192, gated silu 59 | 69, gated relu 51 | 69, gated gelu 98 | 115, 4096
    // of 11008, gated silu 42 | 80, norm of 8192 of 8192 83 | 87); shorter ones with a thread for eight elements (norm of 16384 of 4096 82 | 84; but gated silu of 8192 of 4096 36 | 34), or for 32
    // where there is one input only (norm of 16384 of 4096 52 | 64, plain rows of 8192 of 4096 18 | 28; but norm of 16384 of 2048 38 | 33).  Not: fp32 (8192 of 4096 74 | 66), two inputs of up
    // to 2048 (16384 of 2048 44 | 44), few rows.
    const bool many = p.rows > 4 * (int64_t)st->sm_count && fits(kWide) && p.d <= 16384;
    if (many && p.d > 4096) {
      return p.d <= 8192 ? int8_ring<T, 2, NORM>(device, st, p, 512, 2, s) : int8_ring<T, 4, NORM>(device, st, p, 512, p.d <= 12288 ? 2 : 1, s);
    }
    if (many && !p.b && p.d >= 1024) {
      const int threads = ((p.d + 31) / 32 + 31) / 32 * 32;
      return int8_ring<T, 4, NORM>(device, st, p, threads, 8, s);
    }
    if (many && p.d > 2048) {
      const int threads = ((p.d + 7) / 8 + 31) / 32 * 32;
      return int8_ring<T, 1, NORM>(device, st, p, threads, 1536 / threads, s);
    }
  }
  if (fits(kWide)) return e == 8 ? int8_launch<T, kWide, 8 / kWide, NORM>(p, s) : (e == 16 ? int8_launch<T, kWide, 16 / kWide, NORM>(p, s) : int8_launch<T, kWide, 32 / kWide, NORM>(p, s));
  if constexpr (sizeof(T) == 2) {
    if (fits(2)) return e == 8 ? int8_launch<T, 2, 4, NORM>(p, s) : (e == 16 ? int8_launch<T, 2, 8, NORM>(p, s) : int8_launch<T, 2, 16, NORM>(p, s));
  }
  return e == 8 ? int8_launch<T, 1, 8, NORM>(p, s) : (e == 16 ? int8_launch<T, 1, 16, NORM>(p, s) : int8_launch<T, 1, 32, NORM>(p, s));
}

template <int NORM>
static int int8_rows(int device, int dtype, Int8Rows& p, void* stream) {
  const char* op = NORM ? "rmsnorm_int8" : "rows_int8";
  KeepDevice keep;
  DeviceState* st;
  TSB_TRY(use_device(device, &st));
  cudaStream_t s = pick_stream(st, stream);
  if (dtype == TSB200_F32) TSB_TRY((int8_rows_t<float, NORM>(device, st, p, s)));
  else if (dtype == TSB200_F16) TSB_TRY((int8_rows_t<__half, NORM>(device, st, p, s)));
  else TSB_TRY((int8_rows_t<__nv_bfloat16, NORM>(device, st, p, s)));
  count_launch(device);
  return check_launch(op);
}

// what both entry points refuse; rows of no elements have no scale
static int int8_check(const char* op, int dtype, const void* q, const void* scale, const void* a, int64_t rows, int d) {
  TSB_CHECK(dtype == TSB200_F32 || is_16bit(dtype), "%s: unsupported dtype %d", op, dtype);
  TSB_CHECK(rows >= 0 && rows < ((int64_t)1 << 31), "%s: %lld rows", op, (long long)rows);
  TSB_CHECK(d > 0 && d <= (1 << 30), "%s: rows of %d elements", op, d);
  TSB_CHECK(rows == 0 || (q && scale && a), "%s: null pointer", op);
  const size_t es = dtype_size(dtype);
  TSB_CHECK((uintptr_t)scale % 4 == 0 && (uintptr_t)a % es == 0, "%s: pointers lie between elements", op);
  return 1;
}

}  // namespace tsb

using namespace tsb;

extern "C" {

int TSB200_RMSNormInt8(int device, int dtype, void* q, int64_t q_row, float* scale, void* h, int64_t h_row, const void* x, int64_t x_row, const void* residual, int64_t residual_row,
                       const void* gamma, float eps, int64_t rows, int d, void* stream) {
  TSB_TRY(int8_check("rmsnorm_int8", dtype, q, scale, x, rows, d));
  TSB_CHECK(eps >= 0.0f && eps < INFINITY, "rmsnorm_int8: eps %g", (double)eps);
  TSB_CHECK((residual == nullptr) == (h == nullptr), "rmsnorm_int8: residual and the place of the sum go together");
  TSB_CHECK(((uintptr_t)residual | (uintptr_t)h | (uintptr_t)gamma) % dtype_size(dtype) == 0, "rmsnorm_int8: pointers lie between elements");
  if (rows == 0) return 1;
  TSB_CHECK(gamma, "rmsnorm_int8: null pointer");
  TSB_CHECK(rows == 1 || (q_row >= d && (!h || h_row >= d)), "rmsnorm_int8: rows of the outputs overlap");
  Int8Rows p{};
  p.q = reinterpret_cast<int8_t*>(q); p.q_row = q_row; p.scale = scale;
  p.h = h; p.h_row = h ? h_row : 0;
  p.a = x; p.a_row = x_row;
  p.b = residual; p.b_row = residual ? residual_row : 0;
  p.gamma = gamma; p.eps = eps; p.rows = rows; p.d = d;
  return eps < kInt8Small ? int8_rows<2>(device, dtype, p, stream) : int8_rows<1>(device, dtype, p, stream);
}

int TSB200_RowsInt8(int device, int dtype, void* q, int64_t q_row, float* scale, const void* src, int64_t src_row, const void* gate, int64_t gate_row, int act, int64_t rows, int d,
                    void* stream) {
  TSB_TRY(int8_check("rows_int8", dtype, q, scale, src, rows, d));
  TSB_CHECK((uintptr_t)gate % dtype_size(dtype) == 0, "rows_int8: pointers lie between elements");
  if (act == TSB200_ACT_SWIGLU) act = TSB200_ACT_SILU;
  if (act == TSB200_ACT_GLU_NOACT) act = TSB200_ACT_NONE;
  TSB_CHECK(act >= TSB200_ACT_NONE && act <= TSB200_ACT_SIGMOID, "rows_int8: unsupported activation %d", act);
  if (rows == 0) return 1;
  TSB_CHECK(rows == 1 || q_row >= d, "rows_int8: rows of the output overlap");
  Int8Rows p{};
  p.q = reinterpret_cast<int8_t*>(q); p.q_row = q_row; p.scale = scale;
  p.a = src; p.a_row = src_row;
  p.b = gate; p.b_row = gate ? gate_row : 0;
  p.act = act; p.rows = rows; p.d = d;
  return int8_rows<0>(device, dtype, p, stream);
}

}  // extern "C"
