// Product of rows and weights in 8-bit integers with a scale for each row and each output channel:
//   y[m, n] = t(float(sum_k q[m, k] w[n, k]) (sq[m] sw[n]) + bias[n])
// The sum is exact: products of bytes are at most 2^14, K is below 2^17, the accumulator has 32 bits.  It is rounded to fp32 once, multiplied by the
// product of the scales and added to the bias in one rounding each, then rounded to the type of y.  So a result does not depend on how K is split.
//
// Both operands are rows of K bytes side by side, as checkpoints and ops_int8.cu hold them: K-major operands of tcgen05.mma kind::i8 (32 k to an instruction), that TMA
// lays down in boxes of 128 bytes x rows with the 128-byte swizzle.  K and rows beyond the tensors are zero-filled.  Three kernels:
//  * up to 64 rows: the weights are the 128-row operand, the rows its N dimension; K ranges on the CTAs of a cluster (i8_cluster_kernel);
//  * more rows: pairs of CTAs on tiles of 256 rows x 256 or 128 channels (i8_pair_kernel);
//  * rows that do not start on 16 bytes, which TMA cannot read: tiles of 64 x 64 on the integer pipe (i8_plain_kernel).
// Every mbarrier wait is bounded; on timeout an error word is raised, copies and products in flight end, TMEM is freed and the kernel returns.
#include "tc_common.cuh"

namespace tsb {

struct I8Args {
  const int8_t* q;
  const int8_t* w;
  int64_t q_row, w_row;
  const float* sq;
  const float* sw;
  const void* bias;     // of y's type; may be null
  void* y;
  int64_t y_row;
  int M, N, K;
  int ks, stages;       // i8_cluster_kernel
  int four;             // whether four neighbouring channels lie on a boundary of theirs in y, sw and bias (i8_cluster_kernel)
  int units;            // whether rows of y start on 16 bytes (i8_pair_kernel)
  unsigned wait_limit;
  int* error;
};

template <typename T> struct __align__(4 * sizeof(T)) I8Four { T e[4]; };
__device__ __forceinline__ float i8_value(int acc, float sq, float sw, float bias) { return fmaf((float)acc, sq * sw, bias); }

// scale and bias of channels c .. c + 3 (0 behind the last one)
template <typename T>
__device__ __forceinline__ void i8_channels(const I8Args& a, int c, float* sw, float* bias) {
  const T* b = reinterpret_cast<const T*>(a.bias);
  if (a.four && c < a.N) {
    const float4 s = *reinterpret_cast<const float4*>(a.sw + c);
    sw[0] = s.x; sw[1] = s.y; sw[2] = s.z; sw[3] = s.w;
    I8Four<T> t;
    if (b) t = *reinterpret_cast<const I8Four<T>*>(b + c);
#pragma unroll
    for (int e = 0; e < 4; ++e) bias[e] = b ? to_f<T>(t.e[e]) : 0.0f;
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    sw[e] = c + e < a.N ? a.sw[c + e] : 0.0f;
    bias[e] = b && c + e < a.N ? to_f<T>(b[c + e]) : 0.0f;
  }
}
template <typename T>
__device__ __forceinline__ void i8_put4(T* y, float y0, float y1, float y2, float y3) {
  if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(y) = make_float4(y0, y1, y2, y3);
  else *reinterpret_cast<uint2*>(y) = make_uint2(Pair16<T>::put(y0, y1), Pair16<T>::put(y2, y3));
}
template <typename T>
__device__ __forceinline__ void i8_store4(const I8Args& a, int row, int c, const int* v, float sq, const float* sw, const float* bias) {
  T* y = reinterpret_cast<T*>(a.y) + (int64_t)row * a.y_row + c;
  if (a.four) {
    if (c >= a.N) return;
    i8_put4<T>(y, i8_value(v[0], sq, sw[0], bias[0]), i8_value(v[1], sq, sw[1], bias[1]), i8_value(v[2], sq, sw[2], bias[2]), i8_value(v[3], sq, sw[3], bias[3]));
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (c + e < a.N) y[e] = from_f<T>(i8_value(v[e], sq, sw[e], bias[e]));
}

// 32 accumulators of a lane: asked for, and there (the registers mean nothing in between)
#define TSB_V32(v)                                                                                                                                                        \
  "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]),          \
      "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]), "+r"(v[24]),         \
      "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31])
__device__ __forceinline__ void i8_tmem_ask(uint32_t taddr, uint32_t* r) {
  __syncwarp();
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void i8_tmem_have(uint32_t* r) {
  __syncwarp();
  asm volatile("tcgen05.wait::ld.sync.aligned;" : TSB_V32(r)::"memory");
}

// instruction descriptor: signed bytes, 32-bit sums, both operands K-major
constexpr uint32_t i8_idesc(int m, int n) { return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24); }

// ---- up to 64 rows ------------------------------------------------------------------------------------------------------
// A CTA owns 128 channels over a range of K; the 1 .. 8 CTAs of a cluster share the channels and push their sums, four rows at a time, into the shared
// memory of the CTA that finishes them (1 / ks of the channels each); the stores report to its mbarrier.
// warp 0: copies; warp 1: TMEM and products; warps 2-5: accumulators out of TMEM; all warps: sums and outputs.
// What bounds it: the bytes of the weights (one row of 4096 -> 22016 16.7 us, 5.4 TB/s) and, in the small ones, start, first copies, exchange and end of the launch (one row of 4096 -> 4096
// 5.3 us, of 768 -> 768 3.9; 64 rows of 11008 -> 4096 13.6).  The first round of copies is under way before TMEM is allotted and the warps have met (17.5 -> 16.8 us for the first of these).
constexpr int kI8Threads = 256;
constexpr int kI8W = 128 * 128;   // weight bytes of a stage

template <int NR>
__device__ __forceinline__ void i8_tmem_ld(uint32_t taddr, uint32_t* r) {
  if constexpr (NR == 16) {
    __syncwarp();
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
          "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                   "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])::"memory");
  } else {
    tmem_ld32(taddr, r);
  }
}

template <typename T, int NR>
__global__ void __launch_bounds__(kI8Threads) i8_cluster_kernel(const __grid_constant__ CUtensorMap mapW, const __grid_constant__ CUtensorMap mapQ, I8Args a) {
  constexpr int kQ = NR * 128, kStage = kI8W + kQ;
  constexpr uint32_t kCols = NR < 32 ? 32 : NR;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const int S = a.stages, ks = a.ks, M = a.M;
  // sums: [source rank][row quad][channel of a group][group][4 rows]; of one CTA alone over the ring, which the products have read by then
  int* red = reinterpret_cast<int*>(smem + (ks > 1 ? S * kStage : 0));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S * kStage + (ks > 1 ? NR * 512 : 0));
  const uint32_t full = s_u32(bars), empty = full + 16 * 8, acc = empty + 16 * 8, sums = acc + 8;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 34);
  __shared__ int s_err, s_asked;   // s_asked: steps whose copies are under way or done (warp 0)
  __shared__ float s_sq[NR];

  const int tid = threadIdx.x, lane = tid & 31, w = warp_index();
  const int rank = (int)(blockIdx.x % ks), col0 = (int)(blockIdx.x / ks) * 128;
  const int steps = (a.K + 127) >> 7, k0 = (int)((int64_t)steps * rank / ks), n_it = (int)((int64_t)steps * (rank + 1) / ks) - k0;   // blocks of 128 k
  const int quads = (M + 3) >> 2;

  const uint32_t ring = s_u32(smem);
  auto copy = [&](int i, int s) {
    const uint32_t dst = ring + s * kStage, bar = full + s * 8;
    tc_mbar_expect_el(bar, kStage);
    tma_load_2d_el(dst, &mapW, (k0 + i) * 128, col0, bar);
    tma_load_2d_el(dst + kI8W, &mapQ, (k0 + i) * 128, 0, bar);
  };
  const int n_pre = min(S, n_it);
  if (w == 0) {
    if (lane == 0) {
      asm volatile("prefetch.tensormap [%0];" ::"l"(&mapW) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(&mapQ) : "memory");
      for (int i = 0; i < S; ++i) {
        tc_mbar_init(bars + i, 1);
        tc_mbar_init(bars + 16 + i, 1);
      }
      tc_mbar_init(bars + 32, 1);
      tc_mbar_init(bars + 33, 1);
      s_err = 0;
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      if (ks > 1) tc_mbar_expect_tx(bars + 33, quads * 2048);   // 128 / ks channels from each of ks CTAs
    }
    __syncwarp();
    for (int i = 0; i < n_pre; ++i) copy(i, i);   // on their way while the others get TMEM
  }
  if (w == 1) {
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s_u32(tmem_slot)), "r"(kCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (w >= 2 && tid - 64 < M) s_sq[tid - 64] = a.sq[tid - 64];   // (M <= 64)
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  if (ks > 1) {   // this CTA's barriers exist; waited for in front of the pushes
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  }
  const uint32_t tmem = *tmem_slot;
  volatile int* err = &s_err;

  // this CTA finishes 128 / ks of the channels, in groups of four, of every row: a thread's channels are the same in all of its rows
  const int gsh = 5 - (31 - __clz(ks)), G = 1 << gsh;          // groups here
  const int g = (tid >> 2) & (G - 1);
  const int c = col0 + ((rank << gsh) + g) * 4, row0 = (tid >> (gsh + 2)) * 4 + (tid & 3), step = (kI8Threads >> (gsh + 2)) * 4;

  if (w == 0) {
    // ---------------- copies behind the first round
    int s = 0, i = n_pre;
    unsigned phase = 0;
    for (; i < n_it; ++i) {
      if (!tc_wait_or(empty + s * 8, phase, err, a.wait_limit)) break;
      copy(i, s);
      if (++s == S) s = 0, phase ^= 1;
    }
    if (lane == 0) s_asked = i;
    named_arrive<1, 192>();
  } else if (w == 1) {
    // ---------------- products: rows of 128 B, atoms of 8 rows 1024 B apart; 32 k = 32 B along the row
    constexpr uint32_t idesc = i8_idesc(128, NR);
    const uint32_t hi = desc_hi(1024), a0 = desc_lo(ring, 16), b0 = desc_lo(ring + kI8W, 16);
    int s = 0;
    unsigned phase = 0;
    for (int i = 0; i < n_it; ++i) {
      if (!tc_wait_or(full + s * 8, phase, err, a.wait_limit)) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t ad = a0 + s * (kStage >> 4), bd = b0 + s * (kStage >> 4);
      umma_i8_el(tmem, ad, hi, bd, hi, idesc, i > 0);
      umma_i8_el(tmem, ad + 2, hi, bd + 2, hi, idesc, 1);
      umma_i8_el(tmem, ad + 4, hi, bd + 4, hi, idesc, 1);
      umma_i8_el(tmem, ad + 6, hi, bd + 6, hi, idesc, 1);
      umma_commit_el(empty + s * 8);
      if (++s == S) s = 0, phase ^= 1;
    }
    umma_commit_el(acc);
  }
  __syncwarp();
  float sw[4], bias[4];
  i8_channels<T>(a, c, sw, bias);
  if (ks > 1) cluster_wait();   // the other CTAs' barriers exist

  if (w >= 2 && w < 6) {
    // ---------------- sums out of TMEM: warp w reads lanes 32 (w % 4) .. = channels of the group
    tc_wait_or(acc, 0, err, a.wait_limit);
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const int col = (w & 3) * 32 + lane, owner = col >> (gsh + 2), e = col & 3, here = ((col >> 2) + 2 * e) & (G - 1);
    const uint32_t local = s_u32(red) + ((uint32_t)rank * quads * (G * 4) + e * G + here) * 16, hop = G * 64;
    uint32_t remote = local, bar = sums;
    if (ks > 1) {
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(owner));
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(bar) : "r"(sums), "r"(owner));
    }
#pragma unroll 1
    for (int h = 0; h < (NR + 31) / 32; ++h) {
      if (h * 32 >= M) break;
      uint32_t v[NR < 32 ? NR : 32];
      i8_tmem_ld<NR>(tmem + ((uint32_t)((w & 3) * 32) << 16) + h * 32, v);
#pragma unroll
      for (int r = 0; r < (NR < 32 ? NR : 32); r += 4) {
        const int qd = (h * 32 + r) >> 2;
        if (qd < quads) {
          if (ks > 1)
            asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(remote + qd * hop), "r"(v[r]), "r"(v[r + 1]),
                         "r"(v[r + 2]), "r"(v[r + 3]), "r"(bar)
                         : "memory");
          else
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(local + qd * hop), "r"(v[r]), "r"(v[r + 1]), "r"(v[r + 2]), "r"(v[r + 3]) : "memory");
        }
      }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    named_arrive<1, 192>();   // TMEM has been read
  }
  if (ks > 1) {
    // arrived when everything is pushed (a CTA that gave up has pushed too); waited for before the CTA leaves, so that nobody pushes to one that has
    cluster_arrive_relaxed();
    tc_wait_or(sums, 0, err, a.wait_limit);
  } else {
    __syncthreads();
  }

  // ---------------- outputs: a group's channel e lies 2 e groups further on, so that neither the pushes nor these reads meet in a bank
  const int* from = red + ((size_t)(row0 >> 2) * (G * 4)) * 4 + (row0 & 3);
  const int at0 = g * 4, at1 = (G + ((g + 2) & (G - 1))) * 4, at2 = (2 * G + ((g + 4) & (G - 1))) * 4, at3 = (3 * G + ((g + 6) & (G - 1))) * 4;
  const int hop = quads * (G * 16), skip = (step >> 2) * (G * 16);
  if (c < a.N) {
#pragma unroll 1
    for (int row = row0; row < M; row += step, from += skip) {
      const int* f = from;
      int v[4] = {f[at0], f[at1], f[at2], f[at3]};
      for (int r = 1; r < ks; ++r) {
        f += hop;
        v[0] += f[at0]; v[1] += f[at1]; v[2] += f[at2]; v[3] += f[at3];
      }
      i8_store4<T>(a, row, c, v, s_sq[row], sw, bias);
    }
  }
  __syncwarp();
  if (ks > 1) {
    if (*err) tc_wait_short(sums, 0);   // what is on its way here lands first
    cluster_wait();
  }
  if (w == 1) {
    named_sync<1, 192>();
    if (*err) {   // warp 0, 1 or one of those that read TMEM has given up: copies and products in flight end first (otherwise the products have waited for every
      tc_land(full, S, s_asked);   // copy, and TMEM was read behind the last product)
      tc_wait_short(acc, 0);
    }
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols) : "memory");
  }
  if (*err && lane == 0 && a.error) *a.error = 1;   // the warp that gave up, at least, sees it
}

// ---- more rows -----------------------------------------------------------------------------------------------------------
// A cluster of two CTAs works on tiles of 256 rows x BN channels (cta_group::2): each CTA brings 128 rows and HALF of the channels into its shared
// memory, the leader issues the products of both, each CTA's TMEM receives its own 128 rows.  Persistent; the accumulator is double buffered, so that a tile's
// outputs leave while the products of the next are running and the copies run ahead across tiles.
// Warp 0: copies; warp 1: TMEM and products; warps 2..9: outputs (two per quarter of the TMEM lanes, each half of a tile's channels).
// What bounds it: the tensor pipe and from a few waves on the power limit (8192 x 4096 -> 22016 443 to 470 us, up to 3330 TOP/s; 4096 x 4096 -> 32000 3150); with few k the outputs (8192 x 512 -> 4096
// 26 us, where the products take 9).  An output warp finishes a row of sums in its lane, in straight code: with edges and biases decided per chunk it fetched more instructions than it
// executed (51 us for the last of these), and sums that cross shared memory as integers, to be finished by columns, took 34.  Scales and biases of a tile's channels lie in the warp's shared
// memory, read for the next tile while this one leaves; boxes of 32 x 32 outputs go out by TMA, two in turn.
constexpr int kI8PThreads = 320, kI8PWarps = 8;
constexpr int kI8A = 128 * 128;
template <typename T, int BN>
struct I8Pair {
  static constexpr int kB = BN / 2 * 128;               // weight bytes of a stage and CTA
  static constexpr int kStages = BN == 256 ? (sizeof(T) == 4 ? 4 : 5) : (sizeof(T) == 4 ? 6 : 7);
  static constexpr int kStage = kI8A + kB;
  static constexpr int kBox = 32 * 32 * (int)sizeof(T); // outputs of a warp on their way from rows of TMEM to y: two of these in turn,
  static constexpr int kOut = 2 * kBox + 1024;          // and scales and biases of the warp's channels
  static constexpr int kSmem = kStages * kStage + 1024 + 256 + kI8PWarps * kOut;
  static constexpr int kCols = BN / 2;                  // channels of an output warp
};
__device__ __forceinline__ void i8_store_box(const CUtensorMap* map, uint32_t from, int c0, int c1) {   // by one lane
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map), "r"(from), "r"(c0), "r"(c1) : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}

template <typename T, int BN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kI8PThreads, 1)
    i8_pair_kernel(const __grid_constant__ CUtensorMap mapQ, const __grid_constant__ CUtensorMap mapW, const __grid_constant__ CUtensorMap mapY, I8Args a, int m_tiles, int n_tiles) {
  typedef I8Pair<T, BN> P;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const uint32_t sA = s_u32(smem), sB = sA + P::kStages * kI8A;
  unsigned char* outs = smem + P::kStages * P::kStage;
  uint64_t* bars = reinterpret_cast<uint64_t*>(outs + kI8PWarps * P::kOut);
  // full: the leader's counts the copies of both CTAs; acc_empty: the leader's, both CTAs' output warps arrive
  const uint32_t full = s_u32(bars), empty = full + P::kStages * 8, acc_full = empty + P::kStages * 8, acc_empty = acc_full + 16, drain = acc_empty + 16;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * P::kStages + 5);
  __shared__ int s_err;

  const int tid = threadIdx.x, lane = tid & 31, w = warp_index();
  const int rank = (int)(blockIdx.x & 1), pair = (int)(blockIdx.x >> 1), n_pairs = (int)(gridDim.x >> 1);
  const int k_total = (a.K + 127) >> 7, n_total = m_tiles * n_tiles;
  constexpr uint32_t kTmem = 2 * BN;
  __shared__ int2 s_peer;   // from the other CTA: whether it has given up, and the stages it has asked for
  int asked = 0;            // (warp 0)

  if (tid == 0) {
    for (int i = 0; i < 2 * P::kStages + 2; ++i) tc_mbar_init(bars + i, 1);
    for (int i = 0; i < 2; ++i) tc_mbar_init(bars + 2 * P::kStages + 2 + i, 2 * kI8PWarps);
    tc_mbar_init(bars + 2 * P::kStages + 4, 1);
    s_err = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (w == 1) {
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s_u32(tmem_slot)), "r"(kTmem) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  cluster_sync();   // both CTAs' barriers exist
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = *tmem_slot;
  volatile int* err = &s_err;

  if (w == 0) {
    // ---------------- copies of this CTA
    const uint32_t full0 = tc_leader_addr(full);
    int s = 0;
    unsigned phase = 1;   // parity of the ring's previous round
    bool ok = true;
    for (int t = pair; t < n_total && ok; t += n_pairs) {
      const TcTile tl = tc_tile_of(t, m_tiles, n_tiles, 8);
      const int row = (tl.m_tile * 2 + rank) * 128, col = tl.n_tile * BN + rank * (BN / 2);
      for (int it = 0; it < k_total; ++it) {
        if (asked >= P::kStages && !(ok = tc_wait_or(empty + s * 8, phase, err, a.wait_limit))) break;
        if (rank == 0) tc_mbar_expect_el(full + s * 8, 2 * P::kStage);
        tc_pair_load_2d(sA + s * kI8A, &mapQ, it * 128, row, full0 + s * 8);
        tc_pair_load_2d(sB + s * P::kB, &mapW, it * 128, col, full0 + s * 8);
        ++asked;
        if (++s == P::kStages) s = 0, phase ^= 1;
      }
    }
  } else if (w == 1 && rank == 0) {
    // ---------------- products: rows of 128 B, atoms of 8 rows 1024 B apart; 32 k = 32 B along the row
    constexpr uint32_t idesc = i8_idesc(256, BN);
    const uint32_t hi = desc_hi(1024), a0 = desc_lo(sA, 16), b0 = desc_lo(sB, 16);
    int s = 0, n_done = 0;
    unsigned phase = 0;
    bool ok = true;
    for (int t = pair; t < n_total && ok; t += n_pairs, ++n_done) {
      const int buf = n_done & 1;
      if (n_done >= 2 && !(ok = tc_wait_or(acc_empty + buf * 8, (unsigned)(((n_done >> 1) - 1) & 1), err, a.wait_limit))) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t acc = tmem_base + buf * BN;
      for (int it = 0; it < k_total; ++it) {
        if (!(ok = tc_wait_or(full + s * 8, phase, err, a.wait_limit))) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t ad = a0 + s * (kI8A >> 4), bd = b0 + s * (P::kB >> 4);
        umma_i8_pair_el(acc, ad, hi, bd, hi, idesc, it > 0);
        umma_i8_pair_el(acc, ad + 2, hi, bd + 2, hi, idesc, 1);
        umma_i8_pair_el(acc, ad + 4, hi, bd + 4, hi, idesc, 1);
        umma_i8_pair_el(acc, ad + 6, hi, bd + 6, hi, idesc, 1);
        umma_commit_pair_el(empty + s * 8);
        if (++s == P::kStages) s = 0, phase ^= 1;
      }
      if (ok) umma_commit_pair_el(acc_full + buf * 8);
    }
    umma_commit_pair_el(drain);
    tc_wait_short(drain, 0);
  } else if (w >= 2) {
    // ---------------- outputs: TMEM lanes 32 (w % 4) .. = rows of this CTA's half, channels kCols ((w - 2) / 4) ..
    const int q = w & 3, half = (w - 2) >> 2;
    unsigned char* mine = outs + (w - 2) * P::kOut;
    float* s_w = reinterpret_cast<float*>(mine + 2 * P::kBox);   // scales of the tile's channels, biases behind them
    constexpr int kPer = P::kCols / 32;
    constexpr int kUnits = 2 * (int)sizeof(T);   // 16-byte units of a line of 32 outputs; which of them a lane begins with is the swizzle of the tensor map
    const int swz = sizeof(T) == 4 ? lane & 7 : (lane >> 1) & 3;
    // of the next tile: what it has of scales and biases is on its way while one leaves
    int row0 = 0, n0 = 0, n_live = 0;
    float sq = 0.0f, nw[kPer], nb[kPer];
    auto ahead = [&](int t) {
      const TcTile tl = tc_tile_of(t, m_tiles, n_tiles, 8);
      row0 = (tl.m_tile * 2 + rank) * 128 + q * 32;
      n0 = tl.n_tile * BN + half * P::kCols;
      n_live = min(32, a.M - row0);
      sq = lane < n_live ? a.sq[row0 + lane] : 0.0f;
#pragma unroll
      for (int k = 0; k < kPer; ++k) {
        const int col = n0 + k * 32 + lane;
        const bool there = n_live > 0 && col < a.N;
        nw[k] = there ? a.sw[col] : 0.0f;
        nb[k] = there && a.bias ? to_f<T>(reinterpret_cast<const T*>(a.bias)[col]) : 0.0f;
      }
    };
    if (pair < n_total) ahead(pair);
    int n_done = 0, n_boxes = 0;
    for (int t = pair; t < n_total; t += n_pairs, ++n_done) {
      const int buf = n_done & 1, row = row0, col0 = n0, live = n_live;
      const float scale = sq;
      if (!tc_wait_or(acc_full + buf * 8, (unsigned)((n_done >> 1) & 1), err, a.wait_limit)) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t acc = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(buf * BN + half * P::kCols);
      const int cols = live > 0 ? min(P::kCols, a.N - col0) : 0;
      uint32_t v[32];
      if (cols > 0) i8_tmem_ask(acc, v);
#pragma unroll
      for (int k = 0; k < kPer; ++k) {
        s_w[k * 32 + lane] = nw[k];
        s_w[P::kCols + k * 32 + lane] = nb[k];
      }
      if (t + n_pairs < n_total) ahead(t + n_pairs);
      // the accumulator is free once this warp's last 32 sums of it are in registers (nothing that it wrote has to be seen by anyone)
      auto done = [&]() {
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(tc_leader_addr(acc_empty + buf * 8)) : "memory");
      };
      if (cols <= 0) {
        done();
        continue;
      }
      i8_tmem_have(v);
      // a lane's row: 32 channels finished, in the type of y, and laid down as the tensor map wants them
#pragma unroll 1
      for (int c = 0; c < cols; c += 32, ++n_boxes) {
        const bool more = c + 32 < cols;
        if (!more) done();
        unsigned char* box = mine + (n_boxes & 1) * P::kBox;
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");   // the box before the last one has left
        __syncwarp();
        unsigned char* line = box + lane * (32 * (int)sizeof(T));
#pragma unroll
        for (int j = 0; j < kUnits; ++j) {
          constexpr int kE = 16 / (int)sizeof(T);
          float y[kE];
#pragma unroll
          for (int e = 0; e < kE; e += 4) {
            const float4 sw = *reinterpret_cast<const float4*>(s_w + c + j * kE + e), b = *reinterpret_cast<const float4*>(s_w + P::kCols + c + j * kE + e);
            const uint32_t* x = v + j * kE + e;
            y[e] = i8_value((int)x[0], scale, sw.x, b.x);
            y[e + 1] = i8_value((int)x[1], scale, sw.y, b.y);
            y[e + 2] = i8_value((int)x[2], scale, sw.z, b.z);
            y[e + 3] = i8_value((int)x[3], scale, sw.w, b.w);
          }
          uint4 o;
          if constexpr (sizeof(T) == 4) o = make_uint4(__float_as_uint(y[0]), __float_as_uint(y[1]), __float_as_uint(y[2]), __float_as_uint(y[3]));
          else o = make_uint4(Pair16<T>::put(y[0], y[1]), Pair16<T>::put(y[2], y[3]), Pair16<T>::put(y[4], y[5]), Pair16<T>::put(y[6], y[7]));
          *reinterpret_cast<uint4*>(line + ((j ^ swz) << 4)) = o;
        }
        if (more) i8_tmem_ask(acc + c + 32, v);   // on their way while these leave
        if (a.units) {
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) i8_store_box(&mapY, s_u32(box), col0 + c, row);   // rows and channels that are not there are left out
        } else {
          // a lane per channel: rows of y start anywhere
          __syncwarp();
          const int col = col0 + c + lane, rows = col < a.N ? live : 0;
          T* at = reinterpret_cast<T*>(a.y) + (int64_t)row * a.y_row + col;
#pragma unroll 8
          for (int rr = 0; rr < 32; ++rr, at += a.y_row) {
            constexpr int kE = 16 / (int)sizeof(T);
            const int unit = (lane / kE) ^ (sizeof(T) == 4 ? rr & 7 : (rr >> 1) & 3);
            if (rr < rows) *at = reinterpret_cast<const T*>(box + rr * (32 * (int)sizeof(T)) + (unit << 4))[lane % kE];
          }
        }
        if (more) i8_tmem_have(v);
      }
      __syncwarp();   // scales and biases have been read
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");   // shared memory is not given back before it has been read
    __syncwarp();
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (tid == 0) {
    uint32_t to;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(s_u32(&s_peer)), "r"(rank ^ 1));
    asm volatile("st.shared::cluster.v2.s32 [%0], {%1, %2};" ::"r"(to), "r"(s_err), "r"(asked) : "memory");
  }
  cluster_sync();   // nobody reports to a CTA that has left
  if (s_err | s_peer.x) {
    // Copies in flight land in both CTAs.  One CTA may have asked for up to kStages stages more than the other, whose part the leader's barrier
    // then waits for in vain, or does not know of: the difference is put right, in the phases that are open, before they are waited for.
    if (w == 0 && rank == 0) {
      for (int j = min(asked, s_peer.y); j < max(asked, s_peer.y); ++j) {
        const uint32_t bar = full + (j % P::kStages) * 8;
        if (asked > s_peer.y) tc_mbar_complete_el(bar, P::kStage);
        else tc_mbar_expect_el(bar, P::kStage);
      }
      tc_land(full, P::kStages, max(asked, s_peer.y));
    }
    cluster_sync();
  }
  if (w == 1) {
    if (rank == 1) tc_wait_short(drain, 0);   // the leader has seen its own arrive
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmem) : "memory");
  }
  if (tid == 0 && s_err && a.error) *a.error = 1;
}

// ---- rows that start anywhere --------------------------------------------------------------------------------------------
// 64 x 64 outputs of a CTA, 64 k at a time through shared memory, four bytes to a dp4a.  Bound by the loads, a byte each; it is there for views that TMA cannot read
// (256 x 4001 -> 4096: 320 us, of rows at multiples of 16 bytes 15; one row 295 and 6.5).
template <typename T>
__global__ void __launch_bounds__(256) i8_plain_kernel(I8Args a, int n_tiles) {
  __shared__ int sq[64][17], sw[64][17];   // words of four k; an odd stride: no two rows of a column in one bank
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int m0 = (int)(blockIdx.x / n_tiles) * 64, n0 = (int)(blockIdx.x % n_tiles) * 64;
  int acc[4][4] = {};
  for (int k0 = 0; k0 < a.K; k0 += 64) {
    for (int i = tid; i < 64 * 64; i += 256) {
      const int row = i >> 6, k = k0 + (i & 63);
      reinterpret_cast<int8_t*>(&sq[row][0])[i & 63] = m0 + row < a.M && k < a.K ? a.q[(int64_t)(m0 + row) * a.q_row + k] : (int8_t)0;
      reinterpret_cast<int8_t*>(&sw[row][0])[i & 63] = n0 + row < a.N && k < a.K ? a.w[(int64_t)(n0 + row) * a.w_row + k] : (int8_t)0;
    }
    __syncthreads();
#pragma unroll 4
    for (int k = 0; k < 16; ++k) {
      int x[4], y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[j] = sq[ty + 16 * j][k];
        y[j] = sw[tx + 16 * j][k];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(x[i], y[j], acc[i][j]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
      if (m < a.M && n < a.N)
        reinterpret_cast<T*>(a.y)[(int64_t)m * a.y_row + n] = from_f<T>(i8_value(acc[i][j], a.sq[m], a.sw[n], a.bias ? to_f<T>(reinterpret_cast<const T*>(a.bias)[n]) : 0.0f));
    }
}

// ---- host side -----------------------------------------------------------------------------------------------------------
static int i8_map(CUtensorMap* map, EncodeTiledFn enc, const int8_t* at, int64_t row, int rows, int K, int box_rows) {
  const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)(rows > 1 ? row : (K + 15) / 16 * 16)};   // of a single row means nothing
  const cuuint32_t box[2] = {128, (cuuint32_t)box_rows};
  const cuuint32_t el[2] = {1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t*>(at), dims, strides, box, el, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TSB_CHECK(r == CUDA_SUCCESS, "linear_int8: cuTensorMapEncodeTiled failed with %d", (int)r);
  return 1;
}
// outputs, in boxes of 32 x 32
template <typename T>
static int i8_map_out(CUtensorMap* map, EncodeTiledFn enc, const I8Args& a) {
  const cuuint64_t dims[2] = {(cuuint64_t)a.N, (cuuint64_t)a.M};
  const cuuint64_t strides[1] = {(cuuint64_t)a.y_row * sizeof(T)};
  const cuuint32_t box[2] = {32, 32};
  const cuuint32_t el[2] = {1, 1};
  const CUtensorMapDataType type = sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16;   // moved as they are
  const CUresult r = enc(map, type, 2, a.y, dims, strides, box, el, CU_TENSOR_MAP_INTERLEAVE_NONE, sizeof(T) == 4 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                         CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TSB_CHECK(r == CUDA_SUCCESS, "linear_int8: cuTensorMapEncodeTiled failed with %d for the outputs", (int)r);
  return 1;
}

template <typename T, int NR>
static int i8_cluster(DeviceState* st, int device, EncodeTiledFn enc, I8Args a, cudaStream_t s) {
  constexpr int kStage = kI8W + NR * 128;
  const int groups = (a.N + 127) / 128, steps = (a.K + 127) / 128;
  // K ranges: as long as every CTA has an SM of its own and four blocks of 128 k; with ten blocks also two CTAs to an SM.  us with 1, 2, 4, 8 ranges: one row of 4096 -> 4096
  // 6.6, 5.8, 5.3, 6.1; of 2048 -> 2048 5.0, 5.0, 4.2, 4.7; of 768 -> 768 3.9, 4.2; 64 rows of 4096 -> 4096 8.4, 8.5, 7.4, 8.9; of 11008 -> 4096 27, 19, 14.0, 13.5
  a.ks = 1;
  while (a.ks < 8 && (((int64_t)groups * a.ks * 2 <= st->sm_count && steps / (a.ks * 2) >= 4) || ((int64_t)groups * a.ks * 2 <= 2 * st->sm_count && steps / (a.ks * 2) >= 10))) a.ks *= 2;
  // rings for two CTAs per SM (one with the whole of it: a cluster of eight no longer fits a GPC twice, and 16 of them make two waves)
  const int sums = a.ks > 1 ? NR * 512 : 0;
  a.stages = (112 * 1024 - 1024 - 512 - sums) / kStage;
  if (a.stages > 16) a.stages = 16;
  const int smem = a.stages * kStage + sums + 512 + 1024;
  static bool done[kMaxDevices] = {};
  if (!done[device]) {
    TSB_CUDA(cudaFuncSetAttribute(i8_cluster_kernel<T, NR>, cudaFuncAttributeMaxDynamicSharedMemorySize, 112 * 1024));
    done[device] = true;
  }
  CUtensorMap mapW, mapQ;
  TSB_TRY(i8_map(&mapW, enc, a.w, a.w_row, a.N, a.K, 128));
  TSB_TRY(i8_map(&mapQ, enc, a.q, a.q_row, a.M, a.K, NR));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(groups * a.ks);
  cfg.blockDim = dim3(kI8Threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = a.ks;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  TSB_CUDA(cudaLaunchKernelEx(&cfg, i8_cluster_kernel<T, NR>, mapW, mapQ, a));
  return 1;
}

template <typename T, int BN>
static int i8_pair(DeviceState* st, int device, EncodeTiledFn enc, const I8Args& a, cudaStream_t s) {
  static bool done[kMaxDevices] = {};
  if (!done[device]) {
    TSB_CUDA(cudaFuncSetAttribute(i8_pair_kernel<T, BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, I8Pair<T, BN>::kSmem));
    done[device] = true;
  }
  CUtensorMap mapW, mapQ, mapY{};
  if (a.units) TSB_TRY(i8_map_out<T>(&mapY, enc, a));
  TSB_TRY(i8_map(&mapW, enc, a.w, a.w_row, a.N, a.K, BN / 2));
  TSB_TRY(i8_map(&mapQ, enc, a.q, a.q_row, a.M, a.K, 128));
  const int pairs = st->sm_count / 2, m_tiles = (a.M + 255) / 256, n_tiles = (a.N + BN - 1) / BN;
  const int64_t tiles = (int64_t)m_tiles * n_tiles;
  i8_pair_kernel<T, BN><<<2 * (int)(tiles < pairs ? tiles : pairs), kI8PThreads, I8Pair<T, BN>::kSmem, s>>>(mapQ, mapW, mapY, a, m_tiles, n_tiles);
  return 1;
}

template <typename T>
static int i8_linear(DeviceState* st, int device, I8Args a, cudaStream_t s) {
  a.four = a.N % 4 == 0 && (uintptr_t)a.y % (4 * sizeof(T)) == 0 && (a.M == 1 || a.y_row % 4 == 0) && (uintptr_t)a.sw % 16 == 0 && (uintptr_t)a.bias % (4 * sizeof(T)) == 0;
  a.units = (uintptr_t)a.y % 16 == 0 && a.y_row * sizeof(T) % 16 == 0;
  const bool boxes = ((uintptr_t)a.q | (uintptr_t)a.w) % 16 == 0 && (a.M == 1 || (a.q_row % 16 == 0 && a.q_row >= a.K)) &&
                     (a.N == 1 || (a.w_row % 16 == 0 && a.w_row >= a.K));
  EncodeTiledFn enc = boxes ? get_encode() : nullptr;
  if (!enc) {
    const int64_t n_tiles = (a.N + 63) / 64, tiles = n_tiles * ((a.M + 63) / 64);
    TSB_CHECK(tiles < ((int64_t)1 << 31), "linear_int8: too many tiles");
    i8_plain_kernel<T><<<(unsigned)tiles, 256, 0, s>>>(a, (int)n_tiles);
    return 1;
  }
  st->waits = true;
  a.wait_limit = tc_wait_limit();
  a.error = tc_error_word(device);
  if (a.M <= 16) return i8_cluster<T, 16>(st, device, enc, a, s);
  if (a.M <= 32) return i8_cluster<T, 32>(st, device, enc, a, s);
  if (a.M <= 64) return i8_cluster<T, 64>(st, device, enc, a, s);
  // us: whole waves of pairs times steps of 128 k (0.33 for a tile of 256 channels, 0.19 for one of 128) and the last tile's outputs; launch and start, some 4, are the same for both.  Measured (us,
  // 256 | 128): 100 x 4096 -> 4096 14.9 | 9.9, 256 x 11008 -> 4096 31 | 21, 1024 x 4096 -> 22016 63 | 74, 2048 x 4096 -> 32000 166 | 216, 4096 x 4096 -> 4096 66 | 50.  Of 120 products of 65 to 8192
  // rows the slower one is taken, by more than 5 %, for four: 512 x 4096 -> 32000 52 | 55, 4096 x 1000 -> 2047 17.9 | 19.2, 4096 x 2048 -> 8192 59 | 55, 8192 x 512 -> 4096 26 | 28.
  const int pairs = st->sm_count / 2, m_tiles = (a.M + 255) / 256, k_total = (a.K + 127) / 128;
  const int64_t t256 = (int64_t)m_tiles * ((a.N + 255) / 256), t128 = (int64_t)m_tiles * ((a.N + 127) / 128);
  TSB_CHECK(t128 < (1 << 30), "linear_int8: too many tiles");
  const double c256 = (double)((t256 + pairs - 1) / pairs) * k_total * 0.33 + 3.3, c128 = (double)((t128 + pairs - 1) / pairs) * k_total * 0.19 + 1.6;
  return c256 <= c128 ? i8_pair<T, 256>(st, device, enc, a, s) : i8_pair<T, 128>(st, device, enc, a, s);
}

}  // namespace tsb

using namespace tsb;

extern "C" {

int TSB200_LinearInt8(int device, int dtype, void* y, int64_t y_row, const void* q, int64_t q_row, const float* q_scale, const void* w, int64_t w_row, const float* w_scale,
                      const void* bias, int64_t rows, int K, int N, void* stream) {
  TSB_CHECK(dtype == TSB200_F32 || is_16bit(dtype), "linear_int8: unsupported dtype %d", dtype);
  TSB_CHECK(rows >= 0 && rows < ((int64_t)1 << 31) - 256, "linear_int8: %lld rows", (long long)rows);
  TSB_CHECK(K > 0 && K < (1 << 17), "linear_int8: rows of %d bytes; sums of 2^17 and more may leave 32 bits", K);
  TSB_CHECK(N > 0 && N <= (1 << 30), "linear_int8: %d channels", N);
  TSB_CHECK(rows == 0 || (y && q && q_scale && w && w_scale), "linear_int8: null pointer");
  const size_t es = dtype_size(dtype);
  TSB_CHECK(((uintptr_t)y | (uintptr_t)bias) % es == 0 && ((uintptr_t)q_scale | (uintptr_t)w_scale) % 4 == 0, "linear_int8: pointers lie between elements");
  TSB_CHECK(rows <= 1 || y_row >= N, "linear_int8: rows of the output overlap");
  TSB_CHECK((rows <= 1 || q_row >= 0) && (N == 1 || w_row >= 0), "linear_int8: negative strides");
  if (rows == 0) return 1;
  KeepDevice keep;
  DeviceState* st;
  TSB_TRY(use_device(device, &st));
  cudaStream_t s = pick_stream(st, stream);
  I8Args a{};
  a.q = reinterpret_cast<const int8_t*>(q); a.q_row = q_row; a.sq = q_scale;
  a.w = reinterpret_cast<const int8_t*>(w); a.w_row = w_row; a.sw = w_scale;
  a.bias = bias; a.y = y; a.y_row = y_row;
  a.M = (int)rows; a.N = N; a.K = K;
  if (dtype == TSB200_F32) TSB_TRY(i8_linear<float>(st, device, a, s));
  else if (dtype == TSB200_F16) TSB_TRY(i8_linear<__half>(st, device, a, s));
  else TSB_TRY(i8_linear<__nv_bfloat16>(st, device, a, s));
  count_launch(device);
  return check_launch("linear_int8");
}

}  // extern "C"
