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
// A row is held in registers, 8 to 32 elements a thread: every tensor is read once.  Accesses of 16 bytes where all rows start on such a boundary, of two
// elements or of one otherwise.
#include <type_traits>

#include "kernels.cuh"

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

// silu, sigmoid: exp and the quotient by the approximate instructions, off by a few 2^-22 of what they return; a step of q is 2^-7 of the row's largest value
__device__ __forceinline__ float int8_sigmoid(float v) { return __fdividef(1.0f, 1.0f + __expf(-v)); }
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

// sum of squares and maximum (as the bits of a number without its sign: a NaN is larger than all) over the threads of a row: a warp, or the CTA
template <bool WARP>
__device__ __forceinline__ void int8_reduce(float& sum, uint32_t& top) {
  sum = warp_sum(sum);
  top = __reduce_max_sync(0xffffffffu, top);
  if constexpr (!WARP) {
    __shared__ float s_sum[32];
    __shared__ uint32_t s_top[32];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, warps = blockDim.x >> 5;
    if (lane == 0) {
      s_sum[w] = sum;
      s_top[w] = top;
    }
    __syncthreads();
    sum = warp_sum(lane < warps ? s_sum[lane] : 0.0f);
    top = __reduce_max_sync(0xffffffffu, lane < warps ? s_top[lane] : 0u);
  }
}

// What a row's statistics make of it: the factor of v, and the scale (written by one thread).  `up`: a power of two that v is multiplied by first, so that 127 / max|v|
// stays below infinity where the row is nearly zero.
template <bool NORM>
__device__ __forceinline__ float int8_finish(const Int8Rows& p, int64_t r, float sum, uint32_t top, bool first, float& up) {
  const float mx = __uint_as_float(top);
  const bool fine = top < 0x7f800000u && (!NORM || sum < INFINITY);   // (a NaN is not below)
  up = mx < 1e-27f ? 0x1p60f : 1.0f;
  if (first) {
    float s = mx;
    if constexpr (NORM) s *= 1.0f / sqrtf(sum / (float)p.d + p.eps);
    p.scale[r] = fine ? s / 127.0f : NAN;
  }
  return fine && mx > 0.0f ? 127.0f / (mx * up) : 0.0f;
}

template <typename T, int VEC, int NC, bool NORM, bool WARP>
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
  uint32_t top = 0u;
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
    if (i0 + c * step < p.d) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) top = max(top, __float_as_uint(v[c][e]) & 0x7fffffffu);
    }
  int8_reduce<WARP>(sum, top);
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
}

// Rows of more than 32768 elements: read twice, the second time out of L2 (an element by the thread that wrote its sum)
template <typename T, bool NORM>
__global__ void __launch_bounds__(1024) int8_long_rows_kernel(Int8Rows p) {
  const int64_t r = blockIdx.x;
  const T* a = reinterpret_cast<const T*>(p.a) + r * p.a_row;
  const T* b = reinterpret_cast<const T*>(p.b) + r * p.b_row;
  T* h = reinterpret_cast<T*>(p.h) + r * p.h_row;
  const bool two = p.b != nullptr;
  float sum = 0.0f;
  uint32_t top = 0u;
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
    top = max(top, __float_as_uint(v) & 0x7fffffffu);
  }
  int8_reduce<false>(sum, top);
  float up;
  const float inv = int8_finish<NORM>(p, r, sum, top, threadIdx.x == 0, up);
  for (int i = threadIdx.x; i < p.d; i += 1024) {
    float v;
    if constexpr (NORM) v = to_f<T>(two ? h[i] : a[i]) * to_f<T>(reinterpret_cast<const T*>(p.gamma)[i]);
    else v = value(i);
    p.q[r * p.q_row + i] = inv == 0.0f ? (int8_t)0 : (int8_t)int8_low(v * up, inv);
  }
}

template <typename T, int VEC, int NC, bool NORM>
static int int8_launch(const Int8Rows& p, cudaStream_t s) {
  const int threads = ((p.d + VEC * NC - 1) / (VEC * NC) + 31) / 32 * 32;
  if (threads == 32) {
    // a warp per row, eight rows to a CTA
    const int64_t grid = (p.rows + 7) / 8;
    int8_rows_kernel<T, VEC, NC, NORM, true><<<(unsigned)grid, dim3(32, 8), 0, s>>>(p);
  } else {
    int8_rows_kernel<T, VEC, NC, NORM, false><<<(unsigned)p.rows, threads, 0, s>>>(p);
  }
  return 1;
}

template <typename T, bool NORM>
static int int8_rows_t(DeviceState* st, const Int8Rows& p, cudaStream_t s) {
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
  if (fits(kWide)) return e == 8 ? int8_launch<T, kWide, 8 / kWide, NORM>(p, s) : (e == 16 ? int8_launch<T, kWide, 16 / kWide, NORM>(p, s) : int8_launch<T, kWide, 32 / kWide, NORM>(p, s));
  if constexpr (sizeof(T) == 2) {
    if (fits(2)) return e == 8 ? int8_launch<T, 2, 4, NORM>(p, s) : (e == 16 ? int8_launch<T, 2, 8, NORM>(p, s) : int8_launch<T, 2, 16, NORM>(p, s));
  }
  return e == 8 ? int8_launch<T, 1, 8, NORM>(p, s) : (e == 16 ? int8_launch<T, 1, 16, NORM>(p, s) : int8_launch<T, 1, 32, NORM>(p, s));
}

template <bool NORM>
static int int8_rows(int device, int dtype, Int8Rows& p, void* stream) {
  const char* op = NORM ? "rmsnorm_int8" : "rows_int8";
  KeepDevice keep;
  DeviceState* st;
  TSB_TRY(use_device(device, &st));
  cudaStream_t s = pick_stream(st, stream);
  if (dtype == TSB200_F32) TSB_TRY((int8_rows_t<float, NORM>(st, p, s)));
  else if (dtype == TSB200_F16) TSB_TRY((int8_rows_t<__half, NORM>(st, p, s)));
  else TSB_TRY((int8_rows_t<__nv_bfloat16, NORM>(st, p, s)));
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
  return int8_rows<true>(device, dtype, p, stream);
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
  return int8_rows<false>(device, dtype, p, stream);
}

}  // extern "C"
