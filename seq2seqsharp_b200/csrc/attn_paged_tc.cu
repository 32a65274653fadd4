// Attention of chunks over a paged cache on the 5th-generation tensor cores (16-bit types, head sizes 64 and 128): paged.cuh says what is computed.
//
// One CTA per SM takes its run of units.  An item is 256 (query, head) pairs of a KV head as two tiles of 128 rows; a unit is 128 of its keys.  Roles: warps 0-3 and
// 4-7 do the softmax of one tile each (a thread owns a row), warp 9 issues the products, warps 8, 10 and 11 bring rows in.  TMEM: S0 | S1 | O0 | O1; P goes over S as 16-bit
// operand; the products of one tile run behind the exponentials of the other (PV0(j) QK0(j+1) PV1(j) QK1(j+1)), and those of the next item's first keys
// behind the output of this one's last.
//
// Rows come by cp.async, 16 bytes a lane, into the 128-byte swizzle that the products read: eight keys lie in one page whatever its size, so a warp looks up one
// entry per eight rows; places behind the sequence's end or without a page become zeros (a weight of 0 times what the cache holds there would be
// NaN where that is), any strides do, and a page may end anywhere in a tile.  The copies are generic-proxy writes: they report to the stage's mbarrier when they
// have landed, and the issuing thread orders them before its products with a proxy fence.
#include "attn_tmem.cuh"
#include "paged.cuh"

namespace tsb {

constexpr int kPtThreads = 384, kPtRows = 128, kPtKeys = 128, kPtTile = 2 * kPtRows, kPtBox = kPtKeys * 128, kPtCopiers = 96;
// registers per thread: 384 x 168 at launch
constexpr int kPtSoftmaxRegs = 208, kPtOtherRegs = 88;
static_assert(256 * kPtSoftmaxRegs + 128 * kPtOtherRegs <= kPtThreads * 168, "the warpgroups' registers come out of the launch's");

constexpr int pt_smem(int BX, int NS) { return (2 + 2 * NS) * BX * kPtBox + 1024 + 256; }

__device__ __forceinline__ void pt_cp16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
// one arrival of this thread when its copies so far have landed
__device__ __forceinline__ void pt_arrive_copies(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(s_u32(bar)) : "memory");
}

// key tiles of the run that the two row tiles of an item need
struct PtCounts {
  int n[2], most;
};
__device__ __forceinline__ PtCounts pt_counts(const PagedArgs& a, const PagedRun& r) {
  PtCounts c;
  const int pairs = r.seq.n * a.G, cap = a.max_blocks << a.page_shift;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int p0 = r.t * kPtTile + t * kPtRows, p1 = min(pairs, p0 + kPtRows) - 1;
    const int hi = min(r.seq.len - r.seq.n + p1 / a.G + 1, cap);
    c.n[t] = p0 < pairs ? max(0, min((hi + kPtKeys - 1) / kPtKeys, r.k1) - r.k0) : 0;
  }
  c.most = max(c.n[0], c.n[1]);
  return c;
}

// BX: 64-column boxes of a row (head size 64 BX); NS: key and value tiles in flight
template <typename H, int BX, int NS>
__global__ void __launch_bounds__(kPtThreads, 1) paged_tc_kernel(const __grid_constant__ PagedArgs a) {
  constexpr int HD = BX * 64, CPR = HD / 8;   // 16-byte pieces of a row
  extern __shared__ __align__(1024) unsigned char pt_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)pt_raw + 1023) & ~(uintptr_t)1023);
  const uint32_t sQ = s_u32(smem), sK = sQ + 2 * BX * kPtBox, sV = sK + NS * BX * kPtBox;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + (2 + 2 * NS) * BX * kPtBox);
  uint64_t *k_full = bars, *k_empty = k_full + NS, *v_full = k_empty + NS, *v_empty = v_full + NS;
  uint64_t *q_full = v_empty + NS, *q_empty = q_full + 1, *s_full = q_empty + 1, *p_full = s_full + 2, *o_full = p_full + 2, *o_empty = o_full + 2, *drain = o_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  __shared__ PagedPlanShared plan;
  __shared__ int s_err;

  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  long long all;
  int runs;
  if (!paged_locate<kPtThreads, kPtTile, kPtKeys>(a, blockIdx.x, gridDim.x, plan, all, runs)) return;

  if (tid == 0) {
    for (int i = 0; i < NS; ++i) {
      tc_mbar_init(&k_full[i], kPtCopiers);
      tc_mbar_init(&k_empty[i], 1);
      tc_mbar_init(&v_full[i], kPtCopiers);
      tc_mbar_init(&v_empty[i], 1);
    }
    tc_mbar_init(q_full, kPtCopiers);
    tc_mbar_init(q_empty, 1);
    for (int i = 0; i < 2; ++i) {
      tc_mbar_init(&s_full[i], 1);
      tc_mbar_init(&p_full[i], kPtRows);
      tc_mbar_init(&o_full[i], 1);
      tc_mbar_init(&o_empty[i], kPtRows);
    }
    tc_mbar_init(drain, 1);
    s_err = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (w == 9) {
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s_u32(tmem_slot)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *tmem_slot;
  pdl_trigger();
  volatile int* err = &s_err;
  PagedRun run;
  run.begin(a, plan, kPtTile);

  if (w >= 8) {
    pa_fewer_registers<kPtOtherRegs>();
    if (w != 9) {
      // ---------------- copies
      const int cw = w == 8 ? 0 : w - 9;                      // 0 .. 2
      const int lr = lane / CPR, lc = lane % CPR;             // this lane's row of a pass and piece
      constexpr int RP = 32 / CPR;                            // rows of a pass
      const int page_mask = (1 << a.page_shift) - 1;
      const uint32_t lane_box = (uint32_t)(lc >> 3) * kPtBox;
      uint32_t kc = 0, qc = 0;
      bool ok = true;
      for (; ok && run.next(a, plan, kPtTile, kPtKeys); run.step(a)) {
        const PtCounts n = pt_counts(a, run);
        if (n.most == 0) continue;
        const PagedSeq& s = run.seq;
        const int cap = min(s.len, a.max_blocks << a.page_shift);
        const int* table = a.table + run.b * a.table_stride;
        const int64_t head = run.h * a.c_head + lc * 8;
        // one tile of keys (or values): lane i < 16 knows the page of keys 8 i ..
        auto load = [&](const void* src, uint32_t dst, int tile, int entry) {
#pragma unroll 2
          for (int blk = cw; blk < kPtKeys / 8; blk += 3) {
            const int page = __shfl_sync(0xffffffffu, entry, blk);
            const int key = tile * kPtKeys + blk * 8 + lr;
            const H* p = reinterpret_cast<const H*>(src) + (page >= 0 ? page * a.c_page + head + (key & page_mask) * a.c_tok : 0);
            const uint32_t d = dst + lane_box + blk * 1024;
#pragma unroll
            for (int i = 0; i < 8 / RP; ++i) {
              const int r = lr + i * RP;
              pt_cp16(d + r * 128 + (((lc & 7) ^ r) << 4), page >= 0 && key + i * RP < cap ? p + (int64_t)(i * RP) * a.c_tok : reinterpret_cast<const H*>(src), page >= 0 && key + i * RP < cap);
            }
          }
        };
        auto entry_of = [&](int tile) {
          const int key = tile * kPtKeys + (lane & 15) * 8;
          const int page = key < cap ? table[key >> a.page_shift] : -1;
          return page >= 0 && page < a.num_pages ? page : -1;
        };
        auto load_k = [&](int j, int entry) {
          const uint32_t c = kc + j, st = c % NS;
          if (c >= NS && !tc_wait_or(s_u32(&k_empty[st]), (c / NS - 1) & 1, err, a.wait_limit)) return false;
          load(a.K, sK + st * BX * kPtBox, run.k0 + j, entry);
          pt_arrive_copies(&k_full[st]);
          return true;
        };
        int entry = entry_of(run.k0), ahead = entry;
        ok = load_k(0, entry);
        if (ok && qc > 0) ok = tc_wait_or(s_u32(q_empty), (qc - 1) & 1, err, a.wait_limit);
        if (!ok) break;
        ++qc;
        const int p0 = run.t * kPtTile, pairs = s.n * a.G;
        for (int r0 = cw * RP; r0 < (n.n[1] > 0 ? kPtTile : kPtRows); r0 += 3 * RP) {
          const int r = r0 + lr, p = p0 + r;
          const bool there = p < pairs;
          const H* src = reinterpret_cast<const H*>(a.q);
          if (there) src += (int64_t)(s.row0 + p / a.G) * a.q_row + (int64_t)(run.h * a.G + p % a.G) * a.q_head + lc * 8;
          if (r < kPtTile) pt_cp16(sQ + (r >> 7) * BX * kPtBox + lane_box + (r & 127) * 128 + (((lc & 7) ^ (r & 7)) << 4), src, there);
        }
        pt_arrive_copies(q_full);
        for (int j = 0; j < n.most; ++j) {
          if (j + 1 < n.most) {
            ahead = entry_of(run.k0 + j + 1);
            if (!(ok = load_k(j + 1, ahead))) break;
          }
          const uint32_t c = kc + j, st = c % NS;
          if (c >= NS && !(ok = tc_wait_or(s_u32(&v_empty[st]), (c / NS - 1) & 1, err, a.wait_limit))) break;
          load(a.V, sV + st * BX * kPtBox, run.k0 + j, entry);
          pt_arrive_copies(&v_full[st]);
          entry = ahead;
        }
        kc += n.most;
      }
      asm volatile("cp.async.wait_all;" ::: "memory");   // nothing is written to this shared memory any more, whichever wait has run out
    } else if (lane == 0) {
      // ---------------- products.  Instruction descriptors: fp32 accumulator, A K-major, 128 rows; K: N = 128 K-major; V: N = HD MN-major
      const uint32_t fmt = (1u << 4) | (Pair16<H>::kUmmaFormat << 7) | (Pair16<H>::kUmmaFormat << 10) | ((uint32_t)(kPtRows >> 4) << 24);
      const uint32_t id_qk = fmt | ((uint32_t)(kPtKeys >> 3) << 17), id_pv = fmt | (1u << 16) | ((uint32_t)(HD >> 3) << 17);
      uint32_t kc = 0, qc = 0, pc[2] = {0, 0}, oc[2] = {0, 0};
      bool ok = true;
      auto qk = [&](int t, uint32_t st) {
        const uint32_t q = sQ + t * BX * kPtBox, k = sK + st * BX * kPtBox;
#pragma unroll
        for (int i = 0; i < BX * 4; ++i) {
          const uint32_t off = (i >> 2) * kPtBox + (i & 3) * 32;
          umma_f16(tmem + t * kPtKeys, make_desc(q + off, 16, 1024), make_desc(k + off, 16, 1024), id_qk, i > 0 ? 1u : 0u);
        }
        umma_commit(&s_full[t]);
      };
      auto landed = [&](uint64_t* bar, uint32_t parity) {
        const bool in = pa_wait(bar, parity, err, a.wait_limit);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        return in;
      };
      for (; ok && run.next(a, plan, kPtTile, kPtKeys); run.step(a)) {
        const PtCounts n = pt_counts(a, run);
        if (n.most == 0) continue;
        ok = landed(q_full, qc & 1) && landed(&k_full[kc % NS], (kc / NS) & 1);
        ++qc;
        if (!ok) break;
#pragma unroll
        for (int t = 0; t < 2; ++t)
          if (n.n[t] > 0) qk(t, kc % NS);
        umma_commit(&k_empty[kc % NS]);
        if (n.most == 1) umma_commit(q_empty);
        for (int j = 0; j < n.most && ok; ++j) {
          const bool more = j + 1 < n.most;
          const uint32_t c = kc + j, st = c % NS, next = (c + 1) % NS;
          ok = landed(&v_full[st], (c / NS) & 1);
          if (ok && more) ok = landed(&k_full[next], ((c + 1) / NS) & 1);
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (!ok || j >= n.n[t]) continue;
            ok = pa_wait(&p_full[t], pc[t]++ & 1, err, a.wait_limit);
            if (ok && j == 0 && oc[t]++ > 0) ok = pa_wait(&o_empty[t], oc[t] & 1, err, a.wait_limit);   // the output of the item before has been read
            if (!ok) continue;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            // V stage = [box][128 keys][128 B]: 8-key groups 1024 B apart (SBO), boxes kPtBox apart (LBO); 16 keys = 2048 B
            const uint32_t v = sV + st * BX * kPtBox;
#pragma unroll
            for (int i = 0; i < kPtKeys / 16; ++i)
              pa_umma_ts(tmem + 2 * kPtKeys + t * HD, tmem + t * kPtKeys + i * 8, make_desc(v + i * 2048, kPtBox, 1024), id_pv, (j > 0 || i > 0) ? 1u : 0u);
            if (j + 1 < n.n[t]) qk(t, next);
            else umma_commit(&o_full[t]);
          }
          umma_commit(&v_empty[st]);
          if (more) umma_commit(&k_empty[next]);
          if (j + 2 == n.most) umma_commit(q_empty);
        }
        kc += n.most;
      }
    }
  } else {
    // ---------------- softmax: thread = row of tile t
    pa_more_registers<kPtSoftmaxRegs>();
    const int t = w >> 2, row = tid & 127, page_shift = a.page_shift;
    const uint32_t lanes = (uint32_t)((w & 3) * 32) << 16;
    const uint32_t tS = tmem + lanes + t * kPtKeys, tO = tmem + lanes + 2 * kPtKeys + t * HD;
    const float c = a.c;
    uint32_t sc = 0, oc = 0;
    bool ok = true;
    for (; ok && run.next(a, plan, kPtTile, kPtKeys); run.step(a)) {
      const PagedSeq& s = run.seq;
      const int p0 = run.t * kPtTile + t * kPtRows, pairs = s.n * a.G, p = p0 + row;
      if (p0 >= pairs) continue;
      const PtCounts counts = pt_counts(a, run);
      const int n = t ? counts.n[1] : counts.n[0];
      const int cap = min(s.len, a.max_blocks << page_shift), base = s.len - s.n;
      const bool live = p < pairs;
      const int pos = base + p / a.G, head = run.h * a.G + p % a.G;
      // keys [lo, lim) are visible (a row without a query: zeros, never stored); of the warp: the smallest lim, the largest lo
      const int lim = live ? min(pos + 1, cap) : 0x7fffffff, lo = live && a.window > 0 ? pos - a.window + 1 : 0;
      const int wp = p0 + (row & ~31);
      const int warp_lim = min(base + wp / a.G + 1, cap);
      const int warp_lo = a.window > 0 ? base + min(wp + 31, pairs - 1) / a.G - a.window + 1 : 0;
      const int* table = a.table + run.b * a.table_stride;
      auto hidden = [&](int tile) {   // bit i: keys 8 i .. of the tile have no page
        const int key = tile * kPtKeys + (lane & 15) * 8;
        const int page = key < cap ? table[key >> page_shift] : 0;
        return page < 0 || page >= a.num_pages;
      };
      bool none = n > 0 && hidden(run.k0);
      float m = -INFINITY, l = 0.0f;
      for (int j = 0; j < n; ++j) {
        const unsigned gone = __ballot_sync(0xffffffffu, none) & 0xffffu;
        if (j + 1 < n) none = hidden(run.k0 + j + 1);
        ok = __all_sync(0xffffffffu, pa_wait(&s_full[t], sc & 1, err, a.wait_limit));
        if (!ok) break;
        ++sc;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        uint32_t x[4][32];
#pragma unroll
        for (int q = 0; q < 4; ++q) pa_ld32(tS + q * 32, x[q]);
#pragma unroll
        for (int q = 0; q < 4; ++q) pa_ld_wait(x[q]);
        const int k0 = (run.k0 + j) * kPtKeys;
        if (k0 + kPtKeys > warp_lim || k0 < warp_lo) {
          const int from = lo - k0, to = lim - k0;
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (q * 32 + i >= to || q * 32 + i < from) x[q][i] = 0xff800000u;
        }
        if (gone) {
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (gone >> (q * 4 + i / 8) & 1) x[q][i] = 0xff800000u;
        }
        float mx[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) mx[q] = __uint_as_float(x[q][0]);
#pragma unroll
        for (int i = 1; i < 32; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q) mx[q] = fmaxf(mx[q], __uint_as_float(x[q][i]));
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        if (j == 0) {
          m = top;
        } else if (__any_sync(0xffffffffu, top > m)) {
          const float up = fmaxf(m, top);
          const float f = up == -INFINITY ? 1.0f : pa_ex2((m - up) * c);
          m = up;
          l *= f;
#pragma unroll 1
          for (int q = 0; q < HD / 32; ++q) {
            uint32_t o[32];
            pa_ld32(tO + q * 32, o);
            pa_ld_wait(o);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
            pa_st32(tO + q * 32, o);
          }
        }
        const float mc = m == -INFINITY ? 0.0f : -m * c;   // no key seen yet: every weight is exp2(-inf)
        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t y[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const uint32_t* e = &x[2 * h + (i >> 4)][2 * (i & 15)];
            float2 v = pa_fma2(__uint_as_float(e[0]), __uint_as_float(e[1]), c, mc);
            v.x = pa_ex2(v.x);
            v.y = pa_ex2(v.y);
            y[i] = Pair16<H>::put(v.x, v.y);
            pa_add_pair<H>(sum[i & 3], y[i]);   // the weights as they are rounded for the product: what rounding does to the numerator it does to the denominator
          }
          pa_st32(tS + h * 32, y);
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        pa_st_wait();
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        pa_arrive(&p_full[t]);
      }
      if (!ok) break;
      if (n > 0) {
        ok = __all_sync(0xffffffffu, pa_wait(&o_full[t], oc & 1, err, a.wait_limit));
        if (!ok) break;
        ++oc;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      }
      const bool whole = run.first && run.last;
      float* rec = a.part + (2 * (int64_t)blockIdx.x + (run.first ? 1 : 0)) * paged_record_floats(kPtTile, HD);
      const int r = t * kPtRows + row;
      if (!whole && live) *reinterpret_cast<float2*>(rec + 2 * r) = make_float2(m == -INFINITY ? m : m * c, l);   // the combine's maxima are in units of exp2
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      H* out = reinterpret_cast<H*>(a.out) + (int64_t)(s.row0 + p / a.G) * a.o_row + (int64_t)head * a.o_head;
#pragma unroll 1
      for (int q = 0; q < HD / 32; ++q) {
        uint32_t o[32];
        if (n > 0) {
          pa_ld32(tO + q * 32, o);
          pa_ld_wait(o);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0u;
        }
        if (!live) continue;
        if (whole) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = Pair16<H>::put(__uint_as_float(o[8 * i + 2 * e]) * inv, __uint_as_float(o[8 * i + 2 * e + 1]) * inv);
            reinterpret_cast<uint4*>(out + q * 32)[i] = make_uint4(y[0], y[1], y[2], y[3]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            reinterpret_cast<uint4*>(rec + 2 * kPtTile + (int64_t)r * HD + q * 32)[i] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
        }
      }
      if (n > 0) {
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        pa_arrive(&o_empty[t]);
      }
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (w == 9) {
    if (lane == 0) {   // products in flight end before TMEM is given back, whichever wait has run out
      umma_commit(drain);
      tc_mbar_wait(drain, 0);
    }
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
  if (tid == 0 && s_err && a.error) *a.error = 1;
}

template <typename H, int BX, int NS>
static int pt_launch(int device, DeviceState* st, const PagedArgs& a, cudaStream_t s) {
  constexpr int smem = pt_smem(BX, NS);
  static_assert(smem <= 227 * 1024, "shared memory of a CTA");
  static bool done[kMaxDevices] = {};
  if (!done[device]) {
    TSB_CUDA(cudaFuncSetAttribute(paged_tc_kernel<H, BX, NS>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    done[device] = true;
  }
  paged_tc_kernel<H, BX, NS><<<st->sm_count, kPtThreads, smem, s>>>(a);
  count_launch(device);
  return check_launch("paged_tc");
}

int launch_paged_tc(int device, DeviceState* st, int dtype, PagedArgs a, cudaStream_t s) {
  a.wait_limit = tc_wait_limit();
  a.error = tc_error_word(device);
  a.min_units = 4;
  st->waits = true;
  if (dtype == TSB200_F16) {
    if (a.hd == 64) TSB_TRY((pt_launch<__half, 1, 4>(device, st, a, s)));
    else TSB_TRY((pt_launch<__half, 2, 2>(device, st, a, s)));
  } else {
    if (a.hd == 64) TSB_TRY((pt_launch<__nv_bfloat16, 1, 4>(device, st, a, s)));
    else TSB_TRY((pt_launch<__nv_bfloat16, 2, 2>(device, st, a, s)));
  }
  return launch_paged_combine(device, dtype, a, kPtTile, kPtKeys, st->sm_count, s);
}

}  // namespace tsb
