// Attention of few rows per sequence over a paged cache (16-bit types, head sizes 64 and 128): single tokens, drafts, short chunks.  paged.cuh says what is computed.
//
// Two CTAs per SM take their runs of units; an item is 16 or 32 (query, head) pairs of a KV head, a unit 64 of its keys.  A warp copies: keys and values come by
// TMA tensor copies, a box per page (128-byte swizzle; an entry that names no page is a coordinate outside of the map and arrives as zeros), three or six
// tiles ahead of their use.  Four warps multiply (mma.sync: the rows of a tensor-core tile of tcgen05 would be 7/8 empty): WR of them share the
// rows, the others the keys of a tile, whose states (maximum, sum, output) meet in shared memory at an item's end.  No warp waits for another within an item.
// Weights are rounded to the cache's 16-bit type, because A and B of a product have one type, and the sums add them as rounded; all else is fp32 up to the output.
// What bounds it: bytes; 192 KB of an SM are on their way.  64 single tokens over 165600 keys in all, 32 / 8 heads of 128: 119 us, 5.7 TB/s; with heads of 64 a unit has half
// the bytes and the same chain (16 x 5 rows over up to 16384: 4.9 TB/s); few short sequences are bound by
// the chain lengths - page entries - copies - records (8 tokens over 9600 keys 18 us, one over 530 10).
#include <cfloat>

#include "paged.cuh"
#include "tc_common.cuh"

namespace tsb {

constexpr int kPmWarps = 4, kPmThreads = (kPmWarps + 1) * 32, kPmKeys = 64, kPmBox = kPmKeys * 128, kPmCtas = 2;
constexpr int pm_stages(int BX) { return 6 / BX; }
// copies | rows 0-7 (then 8-15) of three warps, and all warps' maxima and sums
constexpr int pm_merge_floats(int BX) { return 3 * 8 * BX * 64 + kPmWarps * 16 * 2; }
constexpr int pm_smem(int BX) { return 2 * pm_stages(BX) * BX * kPmBox + pm_merge_floats(BX) * 4 + 1024; }
static_assert(kPmCtas * (pm_smem(2) + 1024 + 1024) <= 228 * 1024 && kPmCtas * (pm_smem(1) + 1024 + 1024) <= 228 * 1024, "two CTAs on an SM");

__device__ __forceinline__ void pm_ldmatrix(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void pm_ldmatrix_trans(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ float pm_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// BX: 64-column boxes of a row; WR: warps that share the rows (16 each)
template <typename H, int BX, int WR>
__global__ void __launch_bounds__(kPmThreads, kPmCtas) paged_mma_kernel(const __grid_constant__ CUtensorMap mapK, const __grid_constant__ CUtensorMap mapV,
                                                                        const __grid_constant__ PagedArgs a) {
  constexpr int HD = BX * 64, NS = pm_stages(BX), RT = 16 * WR, KG = kPmWarps / WR, KS = HD / 16, NB = HD / 8;
  static_assert(KG > 1, "the warps of other keys meet in shared memory");
  constexpr int SK = kPmKeys / KG, SN = SK / 8;   // keys of a tile that a warp weighs
  extern __shared__ __align__(1024) unsigned char pm_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)pm_raw + 1023) & ~(uintptr_t)1023);
  const uint32_t ring = s_u32(smem);
  float* merge = reinterpret_cast<float*>(smem + 2 * NS * BX * kPmBox);
  float* ml = merge + 3 * 8 * HD;   // [warp][16][2]
  __shared__ uint64_t full[NS], empty[NS];
  __shared__ unsigned gone_of[NS];  // bit i: keys 8 i .. of the tile have no page
  __shared__ PagedPlanShared plan;
  __shared__ int s_err;
  const int tid = threadIdx.x, lane = tid & 31, w = warp_index();
  if (tid == kPmWarps * 32) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&mapK) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&mapV) : "memory");
  }
  pdl_trigger();
  long long all;
  int runs;
  if (!paged_locate<kPmThreads, RT, kPmKeys>(a, blockIdx.x, gridDim.x, plan, all, runs)) return;
  if (tid == 0) {
    for (int i = 0; i < NS; ++i) {
      tc_mbar_init(&full[i], 1);
      tc_mbar_init(&empty[i], kPmWarps);
    }
    s_err = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  volatile int* err = &s_err;
  PagedRun run;
  run.begin(a, plan, RT);
  uint32_t c = 0;                   // tiles so far
  bool ok = true;

  if (w == kPmWarps) {
    // ---------------- copies
    const int page_mask = (1 << a.page_shift) - 1, blocks = min(kPmKeys, 1 << a.page_shift) / 8;   // eights of keys in a box
    for (; ok && run.next(a, plan, RT, kPmKeys); run.step(a)) {
      const int cap = min(run.seq.len, a.max_blocks << a.page_shift);
      const int* table = a.table + run.b * a.table_stride;
      auto entry_of = [&](int tile) {
        const int key = tile * kPmKeys + (lane & 7) * 8;
        const int page = key < cap ? table[key >> a.page_shift] : -1;
        return page >= 0 && page < a.num_pages ? page : -1;
      };
      int next = entry_of(run.k0), ahead = entry_of(run.k0 + 1);
      for (int kt = run.k0; kt < run.k1; ++kt, ++c) {
        const int entry = next;
        next = ahead;
        ahead = entry_of(kt + 2);
        const uint32_t st = c % NS, bar = s_u32(&full[st]), at = ring + st * 2 * BX * kPmBox;
        if (c >= NS && !(ok = tc_wait_or(s_u32(&empty[st]), (c / NS - 1) & 1, err, a.wait_limit))) break;
        const unsigned gone = __ballot_sync(0xffffffffu, entry < 0) & 0xffu;
        if (lane == 0) {
          gone_of[st] = gone;
          tc_mbar_expect_tx(&full[st], 2 * BX * kPmBox);
        }
        __syncwarp();
        const int page = __shfl_sync(0xffffffffu, entry, lane * blocks & 7);
        if (lane * blocks < 8) {
          const int z = page >= 0 ? page : a.num_pages, y = kt * kPmKeys & page_mask;
#pragma unroll
          for (int i = 0; i < BX; ++i) {
            tma_load_4d(at + i * kPmBox + lane * blocks * 1024, &mapK, 64 * i, y, run.h, z, bar);
            tma_load_4d(at + (BX + i) * kPmBox + lane * blocks * 1024, &mapV, 64 * i, y, run.h, z, bar);
          }
        }
      }
    }
    tc_land(s_u32(full), NS, (int)c);   // whichever wait has run out, nothing is written to this shared memory any more
  } else {
    // ---------------- products
    // (a warp that has given up walks on without waiting: the others meet it at the barriers)
    const int rg = w % WR, kg = w / WR, g8 = lane >> 2, t4 = lane & 3;
    for (; run.next(a, plan, RT, kPmKeys); run.step(a)) {
      const PagedSeq& s = run.seq;
      const int pairs = s.n * a.G, cap = min(s.len, a.max_blocks << a.page_shift);
      // this lane's two rows
      const int pA = run.t * RT + rg * 16 + g8, pB = pA + 8, iA = a.by_G(pA), iB = a.by_G(pB);
      const bool liveA = pA < pairs, liveB = pB < pairs;
      const int hA = run.h * a.G + pA - iA * a.G, hB = run.h * a.G + pB - iB * a.G;
      const int posA = s.len - s.n + iA, posB = s.len - s.n + iB;
      const int hiA = liveA ? min(posA + 1, cap) : 0, hiB = liveB ? min(posB + 1, cap) : 0;
      const int loA = a.window > 0 ? posA - a.window + 1 : 0, loB = a.window > 0 ? posB - a.window + 1 : 0;
      // of the warp's rows: keys that all of them see
      const int first = run.t * RT + rg * 16, last = min(first + 15, pairs - 1);
      const int see_to = min(s.len - s.n + a.by_G(first) + 1, cap), see_from = a.window > 0 ? s.len - s.n + a.by_G(max(last, 0)) - a.window + 1 : 0;
      uint32_t qa[KS][4];
      {
        const H* qA = reinterpret_cast<const H*>(a.q) + (liveA ? (int64_t)(s.row0 + iA) * a.q_row + hA * a.q_head : 0) + 2 * t4;
        const H* qB = reinterpret_cast<const H*>(a.q) + (liveB ? (int64_t)(s.row0 + iB) * a.q_row + hB * a.q_head : 0) + 2 * t4;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          qa[k][0] = liveA ? *reinterpret_cast<const uint32_t*>(qA + k * 16) : 0u;
          qa[k][1] = liveB ? *reinterpret_cast<const uint32_t*>(qB + k * 16) : 0u;
          qa[k][2] = liveA ? *reinterpret_cast<const uint32_t*>(qA + k * 16 + 8) : 0u;
          qa[k][3] = liveB ? *reinterpret_cast<const uint32_t*>(qB + k * 16 + 8) : 0u;
        }
      }
      float mA = -INFINITY, mB = -INFINITY, lA = 0.0f, lB = 0.0f, o[NB][4];
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] = 0.0f;
      for (int kt = run.k0; kt < run.k1; ++kt, ++c) {
        const uint32_t st = c % NS;
        ok = ok && tc_wait_or(s_u32(&full[st]), (c / NS) & 1, err, a.wait_limit);
        if (!ok) continue;
        const unsigned gone = gone_of[st];
        const uint32_t kb = ring + st * 2 * BX * kPmBox, vb = kb + BX * kPmBox;
        // values that no row sees, in front of every window or behind the sequence's end: a weight of 0 times what lies there would be NaN where that is, or an infinity
        const auto clear = [&](int from, int to) {   // of this warp's keys
          for (int r = max(from, kg * SK) + (lane >> 3); r < min(to, (kg + 1) * SK); r += 4)
#pragma unroll
            for (int i = 0; i < BX; ++i) *reinterpret_cast<uint4*>(smem + (st * 2 + 1) * BX * kPmBox + i * kPmBox + r * 128 + (lane & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // before the next copy to this place
          __syncwarp();
        };
        if (cap - kt * kPmKeys < kPmKeys) clear(cap - kt * kPmKeys, kPmKeys);
        const int t0 = kg * SK, key0 = kt * kPmKeys + t0;
        float sc[SN][4];
#pragma unroll
        for (int n = 0; n < SN; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[n][e] = 0.0f;
#pragma unroll
        for (int k = 0; k < KS / 2; ++k)
#pragma unroll
          for (int n = 0; n < SN; ++n) {
            uint32_t b[4];
            const int ch = k * 4 + (lane >> 3), r = t0 + n * 8 + (lane & 7);
            pm_ldmatrix(kb + (ch >> 3) * kPmBox + r * 128 + (((ch & 7) ^ (r & 7)) << 4), b);
            mma_16816<H>(sc[n], qa[2 * k][0], qa[2 * k][1], qa[2 * k][2], qa[2 * k][3], b[0], b[1]);
            mma_16816<H>(sc[n], qa[2 * k + 1][0], qa[2 * k + 1][1], qa[2 * k + 1][2], qa[2 * k + 1][3], b[2], b[3]);
          }
        if (gone != 0 || key0 + SK > see_to || key0 < see_from) {
          if (key0 < see_from) clear(0, paged_front(a, s, run.t * RT) - kt * kPmKeys);
#pragma unroll
          for (int n = 0; n < SN; ++n) {
            const bool none = gone >> ((t0 >> 3) + n) & 1;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int j = key0 + n * 8 + 2 * t4 + e;
              if (!(j < hiA && j >= loA && !none)) sc[n][e] = -INFINITY;
              if (!(j < hiB && j >= loB && !none)) sc[n][2 + e] = -INFINITY;
            }
          }
        }
        float xA = fmaxf(sc[0][0], sc[0][1]), xB = fmaxf(sc[0][2], sc[0][3]);
#pragma unroll
        for (int n = 1; n < SN; ++n) {
          xA = fmaxf(xA, fmaxf(sc[n][0], sc[n][1]));
          xB = fmaxf(xB, fmaxf(sc[n][2], sc[n][3]));
        }
        xA = fmaxf(xA, __shfl_xor_sync(0xffffffffu, xA, 1));
        xB = fmaxf(xB, __shfl_xor_sync(0xffffffffu, xB, 1));
        xA = fmaxf(xA, __shfl_xor_sync(0xffffffffu, xA, 2));
        xB = fmaxf(xB, __shfl_xor_sync(0xffffffffu, xB, 2));
        if (__any_sync(0xffffffffu, xA > mA || xB > mB)) {
          // maxima of scores as they are, and from there exp2(c (score - maximum)); no key seen yet: every weight is exp2(-inf)
          const float uA = fmaxf(mA, xA), uB = fmaxf(mB, xB);
          const float fA = uA == -INFINITY ? 1.0f : pm_ex2((mA - uA) * a.c), fB = uB == -INFINITY ? 1.0f : pm_ex2((mB - uB) * a.c);
          mA = uA;
          mB = uB;
          lA *= fA;
          lB *= fB;
#pragma unroll
          for (int n = 0; n < NB; ++n) {
            o[n][0] *= fA;
            o[n][1] *= fA;
            o[n][2] *= fB;
            o[n][3] *= fB;
          }
        }
        const float nA = mA == -INFINITY ? 0.0f : -mA * a.c, nB = mB == -INFINITY ? 0.0f : -mB * a.c;
        uint32_t p[SN][2];
#pragma unroll
        for (int n = 0; n < SN; ++n) {
          p[n][0] = Pair16<H>::put(pm_ex2(fmaf(sc[n][0], a.c, nA)), pm_ex2(fmaf(sc[n][1], a.c, nA)));
          p[n][1] = Pair16<H>::put(pm_ex2(fmaf(sc[n][2], a.c, nB)), pm_ex2(fmaf(sc[n][3], a.c, nB)));
          // the weights as they are rounded for the product: what rounding does to the numerator it does to the denominator
          const float2 a2 = Pair16<H>::get(p[n][0]), b2 = Pair16<H>::get(p[n][1]);
          lA += a2.x + a2.y;
          lB += b2.x + b2.y;
        }
#pragma unroll
        for (int i = 0; i < SN / 2; ++i) {
          const int vr = t0 + i * 16 + (lane & 7) + ((lane >> 3) & 1) * 8;
#pragma unroll
          for (int n = 0; n < NB / 2; ++n) {
            uint32_t b[4];
            const int ch = n * 2 + (lane >> 4);
            pm_ldmatrix_trans(vb + (ch >> 3) * kPmBox + vr * 128 + (((ch & 7) ^ (vr & 7)) << 4), b);
            mma_16816<H>(o[2 * n], p[2 * i][0], p[2 * i][1], p[2 * i + 1][0], p[2 * i + 1][1], b[0], b[1]);
            mma_16816<H>(o[2 * n + 1], p[2 * i][0], p[2 * i][1], p[2 * i + 1][0], p[2 * i + 1][1], b[2], b[3]);
          }
        }
        __syncwarp();
        if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(s_u32(&empty[st])) : "memory");
      }
      if (mA != -INFINITY) mA *= a.c;   // in units of exp2 from here on
      if (mB != -INFINITY) mB *= a.c;
      lA += __shfl_xor_sync(0xffffffffu, lA, 1);
      lB += __shfl_xor_sync(0xffffffffu, lB, 1);
      lA += __shfl_xor_sync(0xffffffffu, lA, 2);
      lB += __shfl_xor_sync(0xffffffffu, lB, 2);
      {
        // the warps of other keys: factors of every warp's rows first, then rows 0-7 and 8-15 through the same place
        if (t4 == 0) {
          float2* m2 = reinterpret_cast<float2*>(ml) + w * 16 + g8;
          m2[0] = make_float2(mA, lA);
          m2[8] = make_float2(mB, lB);
        }
        named_sync<1, kPmWarps * 32>();
        float fA = 1.0f, fB = 1.0f;
        {
          const float2* m2 = reinterpret_cast<const float2*>(ml) + rg * 16 + g8;
          float uA = -INFINITY, uB = -INFINITY;
#pragma unroll
          for (int k = 0; k < KG; ++k) {
            uA = fmaxf(uA, m2[k * WR * 16].x);
            uB = fmaxf(uB, m2[k * WR * 16 + 8].x);
          }
          const float nA = fmaxf(uA, -FLT_MAX), nB = fmaxf(uB, -FLT_MAX);
          lA = lB = 0.0f;
#pragma unroll
          for (int k = 0; k < KG; ++k) {
            const float2 x = m2[k * WR * 16], y = m2[k * WR * 16 + 8];
            lA += x.y * pm_ex2(x.x - nA);
            lB += y.y * pm_ex2(y.x - nB);
          }
          fA = pm_ex2(mA - nA);
          fB = pm_ex2(mB - nB);
          mA = uA;
          mB = uB;
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          if (half == 1 && run.t * RT + 8 >= pairs) break;   // no row group has a row there
          if (half == 1) named_sync<1, kPmWarps * 32>();
          const float f = half ? fB : fA;
          float* to = merge + (((kg - 1) * WR + rg) * 8 + g8) * HD + 2 * t4;
#pragma unroll
          for (int n = 0; n < NB; ++n) {
            o[n][2 * half] *= f;
            o[n][2 * half + 1] *= f;
            // columns in eights that a row turns by its number: eight rows meet no bank twice
            if (kg > 0) *reinterpret_cast<float2*>(to + ((n ^ g8) & 7) * 8 + (n & ~7) * 8) = make_float2(o[n][2 * half], o[n][2 * half + 1]);
          }
          named_sync<1, kPmWarps * 32>();
          if (kg == 0)
#pragma unroll
            for (int k = 1; k < KG; ++k) {
              const float* from = merge + (((k - 1) * WR + rg) * 8 + g8) * HD + 2 * t4;
#pragma unroll
              for (int n = 0; n < NB; ++n) {
                const float2 x = *reinterpret_cast<const float2*>(from + ((n ^ g8) & 7) * 8 + (n & ~7) * 8);
                o[n][2 * half] += x.x;
                o[n][2 * half + 1] += x.y;
              }
            }
        }
      }
      if (kg == 0) {
        const bool whole = run.first && run.last;
        if (whole) {
          const float vA = lA == 0.0f ? 0.0f : 1.0f / lA, vB = lB == 0.0f ? 0.0f : 1.0f / lB;
          H* outA = reinterpret_cast<H*>(a.out) + (int64_t)(s.row0 + iA) * a.o_row + (int64_t)hA * a.o_head + 2 * t4;
          H* outB = reinterpret_cast<H*>(a.out) + (int64_t)(s.row0 + iB) * a.o_row + (int64_t)hB * a.o_head + 2 * t4;
#pragma unroll
          for (int n = 0; n < NB; ++n) {
            if (liveA) *reinterpret_cast<uint32_t*>(outA + n * 8) = Pair16<H>::put(o[n][0] * vA, o[n][1] * vA);
            if (liveB) *reinterpret_cast<uint32_t*>(outB + n * 8) = Pair16<H>::put(o[n][2] * vB, o[n][3] * vB);
          }
        } else {
          float* rec = a.part + (2 * (int64_t)blockIdx.x + (run.first ? 1 : 0)) * paged_record_floats(RT, HD);
          const int rA = rg * 16 + g8, rB = rA + 8;
          if (t4 == 0) {
            if (liveA) *reinterpret_cast<float2*>(rec + 2 * rA) = make_float2(mA, lA);
            if (liveB) *reinterpret_cast<float2*>(rec + 2 * rB) = make_float2(mB, lB);
          }
          float *toA = rec + 2 * RT + rA * HD + 2 * t4, *toB = rec + 2 * RT + rB * HD + 2 * t4;
#pragma unroll
          for (int n = 0; n < NB; ++n) {
            if (liveA) *reinterpret_cast<float2*>(toA + n * 8) = make_float2(o[n][0], o[n][1]);
            if (liveB) *reinterpret_cast<float2*>(toB + n * 8) = make_float2(o[n][2], o[n][3]);
          }
        }
      }
      named_sync<1, kPmWarps * 32>();   // the next item writes to the same places
    }
  }
  __syncthreads();
  if (tid == 0 && s_err && a.error) *a.error = 1;
}

template <typename H, int BX, int WR>
static int pm_launch(int device, DeviceState* st, const PagedArgs& a, cudaStream_t s) {
  static bool done[kMaxDevices] = {};
  if (!done[device]) {
    TSB_CUDA(cudaFuncSetAttribute(paged_mma_kernel<H, BX, WR>, cudaFuncAttributeMaxDynamicSharedMemorySize, pm_smem(BX)));
    done[device] = true;
  }
  CUtensorMap mk, mv;
  constexpr int dtype = Pair16<H>::kBf16 ? TSB200_BF16 : TSB200_F16;
  TSB_TRY(paged_map(&mk, dtype, a.K, a, kPmKeys));
  TSB_TRY(paged_map(&mv, dtype, a.V, a, kPmKeys));
  paged_mma_kernel<H, BX, WR><<<kPmCtas * st->sm_count, kPmThreads, pm_smem(BX), s>>>(mk, mv, a);
  count_launch(device);
  return check_launch("paged_mma");
}

int launch_paged_mma(int device, DeviceState* st, int dtype, PagedArgs a, int RT, cudaStream_t s) {
  a.wait_limit = tc_wait_limit();
  a.error = tc_error_word(device);
  a.min_units = 1;   // one token of 530: 9.6 us, with two 10.0
  a.snap = 0;
  a.start = 1;
  st->waits = true;
#define TSB_PM(H, BX)                                                        \
  do {                                                                       \
    if (RT == 16) TSB_TRY((pm_launch<H, BX, 1>(device, st, a, s)));          \
    else TSB_TRY((pm_launch<H, BX, 2>(device, st, a, s)));                   \
  } while (0)
  if (dtype == TSB200_F16) {
    if (a.hd == 64) TSB_PM(__half, 1);
    else TSB_PM(__half, 2);
  } else {
    if (a.hd == 64) TSB_PM(__nv_bfloat16, 1);
    else TSB_PM(__nv_bfloat16, 2);
  }
#undef TSB_PM
  return launch_paged_combine(device, dtype, a, RT, kPmCtas * st->sm_count, s);
}

}  // namespace tsb
