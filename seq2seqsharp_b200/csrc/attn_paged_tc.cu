// Attention of chunks over a paged cache on the 5th-generation tensor cores (16-bit types, head sizes 64 and 128): paged.cuh says what is computed.
//
// One CTA per SM takes its run of units.  An item is 256 (query, head) pairs of a KV head as two tiles of 128 rows; a unit is 128 of its keys.  Roles: warps 0-3 and
// 4-7 do the softmax of one tile each (a thread owns a row), warp 9 issues the products, warp 8 brings rows in (10 and 11 help with queries).  TMEM: S0 | S1 |
// O0 | O1; P goes over S as 16-bit operand; the products of one tile run behind the exponentials of the other (PV0(j) QK0(j+1) PV1(j) QK1(j+1)), and those of the
// next item's first keys behind the output of this one's last.
//
// Keys and values come by TMA tensor copies, a box per page (128-byte swizzle, any strides that are multiples of 16 bytes); an entry that names no page is a coordinate
// outside of the map, which arrives as zeros, and the values behind a sequence's end and in front of every window are overwritten with zeros before their product.  Queries come by TMA where
// whole ones fill a tile (1, 2, 4 .. heads to a KV head), else by cp.async into the same swizzle: generic-proxy writes, which the issuing warp orders before
// its products with a proxy fence.
//
// Weights are rounded to the cache's 16-bit type, because A and B of a product have one type; each is off by half a step at most, as the output is.  The sums add them as
// rounded (1.3 to 2 % of the time: 1561 -> 1581 us for the chunks below): with sums of the unrounded ones, two at a time, weights that all round down left a
// mean of equal values 2^-8 (fp16: 2^-11) below them.
//
// What bounds it: the chain of a unit (scores, maximum, exponentials, sums, weights back to TMEM), which two tiles hide from the tensor core only in part.  Two chunks
// of up to 2048 over up to 32768, 32 / 8 heads of 128: 1.56 ms, 1105 TFLOP/s of the 1644 that a library product reaches; prompts of 16384 of heads of 128
// 1.90 ms, of 64 1.58.  What was measured on the way (ms, same chunks): cp.async for keys and values 2.39; one lane for the products and outputs rescaled at every
// new maximum 1.81; boxes prefetched to L2 1.74; scores of 64 keys at a time 1.78.
#include "attn_tmem.cuh"
#include "paged.cuh"

namespace tsb {

constexpr int kPtThreads = 384, kPtRows = 128, kPtKeys = 128, kPtTile = 2 * kPtRows, kPtBox = kPtKeys * 128, kPtCopiers = 96;
// registers per thread: 384 x 168 at launch
constexpr int kPtSoftmaxRegs = 208, kPtOtherRegs = 88;
static_assert(256 * kPtSoftmaxRegs + 128 * kPtOtherRegs <= kPtThreads * 168, "the warpgroups' registers come out of the launch's");

constexpr int kPtStage = 32 * 64;   // bytes of a softmax warp to turn rows of outputs into lines
constexpr int pt_smem(int BX, int NS) { return (2 + 2 * NS) * BX * kPtBox + 8 * kPtStage + 1024; }

// one arrival of this thread when its copies so far have landed
__device__ __forceinline__ void pt_arrive_copies(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(s_u32(bar)) : "memory");
}

// A row's output is rescaled when its maximum is this much (in powers of two) above the one in use (a published method for attention on matrix units): one of a
// warp's 32 rows has a new maximum in nearly every tile of the first hundred.  Weights are then up to 2^8, in range of both types; the largest is rounded like the others, no longer 1
constexpr float kPtLag = 8.0f;

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
    const int hi = min(r.seq.len - r.seq.n + a.by_G(p1) + 1, cap);
    c.n[t] = p0 < pairs ? max(0, min((hi + kPtKeys - 1) / kPtKeys, r.k1) - r.k0) : 0;
  }
  c.most = max(c.n[0], c.n[1]);
  return c;
}

// BX: 64-column boxes of a row (head size 64 BX); NS: key and value tiles in flight
template <typename H, int BX, int NS>
__global__ void __launch_bounds__(kPtThreads, 1) paged_tc_kernel(const __grid_constant__ CUtensorMap mapK, const __grid_constant__ CUtensorMap mapV,
                                                                 const __grid_constant__ CUtensorMap mapQ, const __grid_constant__ PagedArgs a, int q_boxes) {
  constexpr int HD = BX * 64, CPR = HD / 8;   // CPR: 16-byte pieces of a row
  extern __shared__ __align__(1024) unsigned char pt_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)pt_raw + 1023) & ~(uintptr_t)1023);
  const uint32_t sQ = s_u32(smem), sK = sQ + 2 * BX * kPtBox, sV = sK + NS * BX * kPtBox;
  unsigned char* stage = smem + (2 + 2 * NS) * BX * kPtBox;
  __shared__ uint64_t k_full[NS], k_empty[NS], v_full[NS], v_empty[NS], q_full[1], q_empty[1], s_full[2], p_full[4], o_full[2], o_empty[2], drain[1];
  __shared__ uint32_t tmem_slot[1];
  __shared__ PagedPlanShared plan;
  __shared__ PagedRun wrun[12];   // of every warp: where it is (registers are the softmax's)
  __shared__ unsigned gone_of[8]; // bit i: keys 8 i .. of the key tile have no page
  __shared__ int s_err;

  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  if (tid == 8 * 32) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&mapK) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&mapQ) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&mapV) : "memory");
  }
  long long all;
  int runs;
  if (!paged_locate<kPtThreads, kPtTile, kPtKeys>(a, blockIdx.x, gridDim.x, plan, all, runs)) return;

  if (tid == 0) {
    for (int i = 0; i < NS; ++i) {
      tc_mbar_init(&k_full[i], 1);
      tc_mbar_init(&k_empty[i], 1);
      tc_mbar_init(&v_full[i], 1);
      tc_mbar_init(&v_empty[i], 1);
    }
    tc_mbar_init(q_full, q_boxes ? 1 : kPtCopiers);
    tc_mbar_init(q_empty, 1);
    for (int i = 0; i < 2; ++i) {
      tc_mbar_init(&s_full[i], 1);
      tc_mbar_init(&p_full[2 * i], kPtRows);       // of the tile's first 64 keys, and of its others
      tc_mbar_init(&p_full[2 * i + 1], kPtRows);
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
  PagedRun& run = wrun[w];
  bool begun = false;
  auto next_item = [&]() {   // by a whole warp
    bool more = false;
    __syncwarp();
    if (lane == 0) {
      PagedRun r = run;
      if (begun) r.step(a);
      else r.begin(a, plan, kPtTile);
      more = r.next(a, plan, kPtTile, kPtKeys);
      run = r;
    }
    begun = true;
    more = __shfl_sync(0xffffffffu, more, 0);
    __syncwarp();
    return more;
  };

  if (w >= 8) {
    pa_fewer_registers<kPtOtherRegs>();
    if (w != 9) {
      // ---------------- copies: warp 8 keys, values and, where whole queries fill a tile, the queries; else all three share the queries' rows
      const int cw = w == 8 ? 0 : w - 9;
      const int page_mask = (1 << a.page_shift) - 1, box_blocks = min(kPtKeys, 1 << a.page_shift) / 8;   // eights of keys in a box of the maps
      uint32_t kc = 0, qc = 0;
      int ks = 0, vs = 0;                                     // tiles asked for so far
      bool ok = cw == 0 || !q_boxes;
      while (ok && next_item()) {
        const PtCounts n = pt_counts(a, run);
        if (n.most == 0) continue;
        const PagedSeq s = run.seq;
        const int cap = min(s.len, a.max_blocks << a.page_shift), k0 = run.k0, h = run.h;
        const int* table = a.table + run.b * a.table_stride;
        auto entry_of = [&](int tile) {   // lane i < 16: the page of keys 8 i ..
          const int key = tile * kPtKeys + (lane & 15) * 8;
          const int page = key < cap ? table[key >> a.page_shift] : -1;
          return page >= 0 && page < a.num_pages ? page : -1;
        };
        // a tile of keys or values by boxes of a page; a page that there is not lies outside of the map and arrives as zeros
        auto load = [&](const CUtensorMap* map, uint32_t dst, uint64_t* full, int tile, int entry) {
          if (lane == 0) tc_mbar_expect_tx(full, BX * kPtBox);
          __syncwarp();
          const int page = __shfl_sync(0xffffffffu, entry, lane * box_blocks & 15);
          if (lane * box_blocks < 16)
#pragma unroll
            for (int i = 0; i < BX; ++i)
              tma_load_4d(dst + i * kPtBox + lane * box_blocks * 1024, map, 64 * i, tile * kPtKeys & page_mask, h, page >= 0 ? page : a.num_pages, s_u32(full));
        };
        auto load_k = [&](int j, int entry) {
          const uint32_t c = kc + j, st = c % NS;
          if (c >= NS && !tc_wait_or(s_u32(&k_empty[st]), (c / NS - 1) & 1, err, a.wait_limit)) return false;
          // read behind the tile's scores; a tile NS + 1 in front has been weighed when this one's copies begin
          const unsigned gone = __ballot_sync(0xffffffffu, entry < 0) & 0xffffu;
          if (lane == 0) gone_of[c & 7] = gone;
          load(&mapK, sK + st * BX * kPtBox, &k_full[st], k0 + j, entry);
          ks = c + 1;
          return true;
        };
        // entries are looked up two tiles ahead
        int entry = 0, next = 0;
        if (cw == 0) {
          entry = entry_of(k0);
          next = entry_of(k0 + 1);
          ok = load_k(0, entry);
        }
        if (ok && qc > 0) ok = tc_wait_or(s_u32(q_empty), (qc - 1) & 1, err, a.wait_limit);
        if (!ok) break;
        ++qc;
        const int p0 = run.t * kPtTile, pairs = s.n * a.G;
        if (q_boxes) {
          // boxes of G heads (rows behind the sequence's are another's, and are not stored)
          const int tiles = n.n[1] > 0 ? 2 : 1;
          if (lane == 0) tc_mbar_expect_tx(q_full, tiles * BX * kPtBox);
          __syncwarp();
          if (lane < tiles * BX) tma_load_3d(sQ + lane * kPtBox, &mapQ, lane % BX * 64, h * a.G, s.row0 + a.by_G(p0 + lane / BX * kPtRows), s_u32(q_full));
        } else {
          const int lr = lane / CPR, lc = lane % CPR;   // this lane's row of a pass and piece
          constexpr int RP = 32 / CPR;                  // rows of a pass
          for (int r0 = cw * RP; r0 < (n.n[1] > 0 ? kPtTile : kPtRows); r0 += 3 * RP) {
            const int r = r0 + lr, p = p0 + r, query = a.by_G(p);
            const bool there = p < pairs;
            const H* src = reinterpret_cast<const H*>(a.q);
            if (there) src += (int64_t)(s.row0 + query) * a.q_row + (int64_t)(h * a.G + p - query * a.G) * a.q_head + lc * 8;
            if (r < kPtTile) paged_cp16(sQ + (r >> 7) * BX * kPtBox + (lc >> 3) * kPtBox + (r & 127) * 128 + (((lc & 7) ^ (r & 7)) << 4), src, there);
          }
          pt_arrive_copies(q_full);
        }
        if (cw != 0) continue;
        for (int j = 0; j < n.most; ++j) {
          const int ahead = entry_of(k0 + j + 2);
          if (j + 1 < n.most && !(ok = load_k(j + 1, next))) break;
          const uint32_t c = kc + j, st = c % NS;
          if (c >= NS && !(ok = tc_wait_or(s_u32(&v_empty[st]), (c / NS - 1) & 1, err, a.wait_limit))) break;
          load(&mapV, sV + st * BX * kPtBox, &v_full[st], k0 + j, entry);
          vs = c + 1;
          entry = next;
          next = ahead;
        }
        kc += n.most;
      }
      // nothing is written to this shared memory any more, whichever wait has run out (tc_land)
      asm volatile("cp.async.wait_all;" ::: "memory");
      if (cw == 0) {
        tc_land(s_u32(k_full), NS, ks);
        tc_land(s_u32(v_full), NS, vs);
        if (q_boxes && qc > 0) tc_wait_short(s_u32(q_full), (qc - 1) & 1);
      }
    } else {
      // ---------------- products, issued by an elected lane of a converged warp: 32 to a unit leave no time for the descriptors of a diverged one.
      // Instruction descriptors: fp32 accumulator, A K-major, 128 rows; K: N = 128 K-major; V: N = HD MN-major
      const uint32_t fmt = (1u << 4) | (Pair16<H>::kUmmaFormat << 7) | (Pair16<H>::kUmmaFormat << 10) | ((uint32_t)(kPtRows >> 4) << 24);
      const uint32_t id_qk = fmt | ((uint32_t)(kPtKeys >> 3) << 17), id_pv = fmt | (1u << 16) | ((uint32_t)(HD >> 3) << 17);
      const uint32_t hi = desc_hi(1024);
      uint32_t kc = 0, qc = 0, pc[2] = {0, 0}, oc[2] = {0, 0};
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity) { return tc_wait_or(s_u32(bar), parity & 1, err, a.wait_limit); };
      auto landed = [&](uint64_t* bar, uint32_t parity) {
        const bool in = wait(bar, parity);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        return in;
      };
      auto qk = [&](int t, uint32_t st) {
        const uint32_t q = desc_lo(sQ + t * BX * kPtBox, 16), k = desc_lo(sK + st * BX * kPtBox, 16);
#pragma unroll
        for (int i = 0; i < BX * 4; ++i) {
          const uint32_t off = ((i >> 2) * kPtBox + (i & 3) * 32) >> 4;
          umma_el(tmem + t * kPtKeys, q + off, hi, k + off, hi, id_qk, i > 0 ? 1u : 0u);
        }
        umma_commit_el(s_u32(&s_full[t]));
      };
      while (ok && next_item()) {
        const PtCounts n = pt_counts(a, run);
        if (n.most == 0) continue;
        const int cap = min(run.seq.len, a.max_blocks << a.page_shift), front = paged_front(a, run.seq, run.t * kPtTile);
        ok = landed(q_full, qc) && wait(&k_full[kc % NS], kc / NS);
        ++qc;
        if (!ok) break;
#pragma unroll
        for (int t = 0; t < 2; ++t)
          if (n.n[t] > 0) qk(t, kc % NS);
        umma_commit_el(s_u32(&k_empty[kc % NS]));
        if (n.most == 1) umma_commit_el(s_u32(q_empty));
        for (int j = 0; j < n.most && ok; ++j) {
          const bool more = j + 1 < n.most;
          const uint32_t c = kc + j, st = c % NS, next = (c + 1) % NS;
          ok = wait(&v_full[st], c / NS);
          const int hidden = front - (run.k0 + j) * kPtKeys, left = cap - (run.k0 + j) * kPtKeys;   // keys of the tile in front of every window, and up to the sequence's end
          if (ok && (left < kPtKeys || hidden > 0)) {
            // values that no row sees: a weight of 0 times what lies there would be NaN where that is, or an infinity
            for (int r = hidden > 0 ? lane : max(left, 0) * 8 + lane; r < kPtKeys * 8; r += 32)
#pragma unroll
              for (int i = 0; i < BX; ++i)
                if (r < hidden * 8 || r >= left * 8) *reinterpret_cast<uint4*>(smem + (2 + NS + st) * BX * kPtBox + i * kPtBox + r * 16) = make_uint4(0u, 0u, 0u, 0u);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
          }
          if (ok && more) ok = wait(&k_full[next], (c + 1) / NS);
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (!ok || j >= n.n[t]) continue;
            // V stage = [box][128 keys][128 B]: 8-key groups 1024 B apart (SBO), boxes kPtBox apart (LBO); 16 keys = 2048 B
            const uint32_t v = desc_lo(sV + st * BX * kPtBox, kPtBox);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              ok = ok && wait(&p_full[2 * t + h], pc[t]);
              if (ok && h == 0 && j == 0 && oc[t]++ > 0) ok = wait(&o_empty[t], oc[t]);   // the output of the item before has been read
              if (!ok) break;
              asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
              for (int i = 4 * h; i < 4 * h + 4; ++i)
                pa_umma_ts_el(tmem + 2 * kPtKeys + t * HD, tmem + t * kPtKeys + i * 8, v + i * (2048 >> 4), hi, id_pv, (j > 0 || i > 0) ? 1u : 0u);
            }
            ++pc[t];
            if (!ok) continue;
            if (j + 1 < n.n[t]) qk(t, next);
            else umma_commit_el(s_u32(&o_full[t]));
          }
          umma_commit_el(s_u32(&v_empty[st]));
          if (more) umma_commit_el(s_u32(&k_empty[next]));
          if (j + 2 == n.most) umma_commit_el(s_u32(q_empty));
        }
        kc += n.most;
      }
    }
  } else {
    // ---------------- softmax: thread = row of tile t
    pa_more_registers<kPtSoftmaxRegs>();
    const int t = w >> 2, row = tid & 127;
    const uint32_t lanes = (uint32_t)((w & 3) * 32) << 16;
    const uint32_t tS = tmem + lanes + t * kPtKeys, tO = tmem + lanes + 2 * kPtKeys + t * HD;
    const float c = a.c;
    uint32_t sc = 0, oc = 0, kc = 0;
    bool ok = true;
    while (ok && next_item()) {
      const PtCounts counts = pt_counts(a, run);
      const int n = t ? counts.n[1] : counts.n[0], k0_item = run.k0;
      const uint32_t c0 = kc;
      kc += counts.most;
      // keys [lo, lim) are visible (a row without a query: zeros, never stored); of the warp: the smallest lim, the largest lo
      int lim, lo, warp_lim, warp_lo;
      {
        const int p0 = run.t * kPtTile + t * kPtRows, pairs = run.seq.n * a.G, p = p0 + row;
        if (p0 >= pairs) continue;
        const int cap = min(run.seq.len, a.max_blocks << a.page_shift), base = run.seq.len - run.seq.n, pos = base + a.by_G(p), wp = p0 + (row & ~31);
        lim = p < pairs ? min(pos + 1, cap) : 0x7fffffff;
        lo = p < pairs && a.window > 0 ? pos - a.window + 1 : 0;
        warp_lim = min(base + a.by_G(wp) + 1, cap);
        warp_lo = a.window > 0 ? base + a.by_G(min(wp + 31, pairs - 1)) - a.window + 1 : 0;
      }
      float m = -INFINITY, l = 0.0f;
      for (int j = 0; j < n; ++j) {
        ok = __all_sync(0xffffffffu, pa_wait(&s_full[t], sc & 1, err, a.wait_limit));
        if (!ok) break;
        ++sc;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        uint32_t x[4][32];
#pragma unroll
        for (int q = 0; q < 4; ++q) pa_ld32(tS + q * 32, x[q]);
#pragma unroll
        for (int q = 0; q < 4; ++q) pa_ld_wait(x[q]);
        const unsigned gone = gone_of[(c0 + j) & 7];
        const int k0 = (k0_item + j) * kPtKeys;
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
        for (int i = 1; i < 31; i += 2)
#pragma unroll
          for (int q = 0; q < 4; ++q) mx[q] = fmaxf(fmaxf(mx[q], __uint_as_float(x[q][i])), __uint_as_float(x[q][i + 1]));
#pragma unroll
        for (int q = 0; q < 4; ++q) mx[q] = fmaxf(mx[q], __uint_as_float(x[q][31]));
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        if (j == 0) {
          m = top;
        } else if (__any_sync(0xffffffffu, (top - m) * c > kPtLag || m == -INFINITY)) {
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
            pa_add_pair<H>(sum[i & 3], y[i]);   // as rounded for the product: what rounding does to the numerator it does to the denominator
          }
          pa_st32(tS + h * 32, y);
          pa_st_wait();
          asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
          pa_arrive(&p_full[2 * t + h]);
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      }
      if (!ok) break;
      if (n > 0) {
        ok = __all_sync(0xffffffffu, pa_wait(&o_full[t], oc & 1, err, a.wait_limit));
        if (!ok) break;
        ++oc;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      }
      const PagedSeq s = run.seq;
      const int p0 = run.t * kPtTile + t * kPtRows + (row & ~31), pairs = s.n * a.G, p = p0 + lane;   // of the warp, of the lane
      const bool whole = run.first && run.last;
      const int64_t rf = paged_record_floats(kPtTile, HD);
      float* rec = a.part + (2 * (int64_t)blockIdx.x + (run.first ? 1 : 0)) * rf;
      if (!whole && p < pairs) *reinterpret_cast<float2*>(rec + 2 * (t * kPtRows + row)) = make_float2(m == -INFINITY ? m : m * c, l);   // the combine's maxima are in units of exp2
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      // 64 bytes of 32 rows at a time, through shared memory: the rows of lanes lie far from each other, and a store of 32 lines takes as long as four of eight
      unsigned char* mine = stage + w * kPtStage;
      const int line = lane >> 2, ch = lane & 3;   // of eight rows, and the piece of 16 bytes
      auto turn = [&](const uint32_t* v, auto put) {
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(mine + lane * 64 + ((i ^ (lane >> 1 & 3)) << 4)) = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        __syncwarp();
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int r = k * 8 + line;
          const uint4 u = *reinterpret_cast<const uint4*>(mine + r * 64 + ((ch ^ (r >> 1 & 3)) << 4));
          if (p0 + r < pairs) put(r, u);
        }
      };
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
        if (whole) {
          uint32_t y[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) y[i] = Pair16<H>::put(__uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv);
          turn(y, [&](int r, uint4 u) {
            const int pr = p0 + r, query = a.by_G(pr);
            H* out = reinterpret_cast<H*>(a.out) + (int64_t)(s.row0 + query) * a.o_row + (int64_t)(run.h * a.G + pr - query * a.G) * a.o_head + q * 32;
            reinterpret_cast<uint4*>(out)[ch] = u;
          });
        } else {
#pragma unroll
          for (int half = 0; half < 2; ++half)
            turn(o + 16 * half, [&](int r, uint4 u) {
              reinterpret_cast<uint4*>(rec + 2 * kPtTile + (int64_t)(t * kPtRows + (row & ~31) + r) * HD + q * 32 + half * 16)[ch] = u;
            });
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
    umma_commit_el(s_u32(drain));   // products in flight end before TMEM is given back, whichever wait has run out
    tc_wait_short(s_u32(drain), 0);
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
  if (tid == 0 && s_err && a.error) *a.error = 1;
}

// a box: 64 columns of up to `keys` tokens of a page
int paged_map(CUtensorMap* map, int dtype, const void* base, const PagedArgs& a, int keys) {
  EncodeTiledFn enc = get_encode();
  TSB_CHECK(enc, "paged_attention: the driver has no cuTensorMapEncodeTiled");
  const cuuint64_t page = (cuuint64_t)1 << a.page_shift;
  const cuuint64_t dims[4] = {(cuuint64_t)a.hd, page, (cuuint64_t)a.Hkv, (cuuint64_t)a.num_pages};
  // the stride of a single head or page means nothing
  const cuuint64_t strides[3] = {(cuuint64_t)a.c_tok * 2, (cuuint64_t)(a.Hkv > 1 ? a.c_head : a.hd) * 2, (cuuint64_t)(a.num_pages > 1 ? a.c_page : a.hd) * 2};
  const cuuint32_t box[4] = {64, page < (cuuint64_t)keys ? (cuuint32_t)page : (cuuint32_t)keys, 1, 1}, el[4] = {1, 1, 1, 1};
  const CUresult r = enc(map, dtype == TSB200_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base), dims, strides, box, el,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TSB_CHECK(r == CUDA_SUCCESS, "paged_attention: cuTensorMapEncodeTiled failed with %d", (int)r);
  return 1;
}
constexpr int64_t paged_stride_most = (int64_t)1 << 39;   // elements: bytes below 2^40
static int pt_map_q(CUtensorMap* map, int dtype, const PagedArgs& a) {
  EncodeTiledFn enc = get_encode();
  const cuuint64_t dims[3] = {(cuuint64_t)a.hd, (cuuint64_t)a.H, (cuuint64_t)a.rows};
  const cuuint64_t strides[2] = {(cuuint64_t)(a.H > 1 ? a.q_head : a.hd) * 2, (cuuint64_t)a.q_row * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)a.G, (cuuint32_t)(kPtRows / a.G)}, el[3] = {1, 1, 1};
  const CUresult r = enc(map, dtype == TSB200_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(a.q), dims, strides, box, el,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TSB_CHECK(r == CUDA_SUCCESS, "paged_attention: cuTensorMapEncodeTiled failed with %d", (int)r);
  return 1;
}
// strides that a tensor map takes
bool paged_tc_strides(const PagedArgs& a) {
  const int64_t most = paged_stride_most;
  return a.num_pages > 0 && a.c_tok > 0 && a.c_tok < most && (a.Hkv == 1 || (a.c_head > 0 && a.c_head < most)) && (a.num_pages == 1 || (a.c_page > 0 && a.c_page < most));
}

template <typename H, int BX, int NS>
static int pt_launch(int device, DeviceState* st, const PagedArgs& a, cudaStream_t s) {
  constexpr int smem = pt_smem(BX, NS);
  static_assert(smem <= 225 * 1024, "shared memory of a CTA, beside 2 KB of fixed size");
  static bool done[kMaxDevices] = {};
  if (!done[device]) {
    TSB_CUDA(cudaFuncSetAttribute(paged_tc_kernel<H, BX, NS>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    done[device] = true;
  }
  CUtensorMap mk, mv, mq;
  constexpr int dtype = Pair16<H>::kBf16 ? TSB200_BF16 : TSB200_F16;
  TSB_TRY(paged_map(&mk, dtype, a.K, a, kPtKeys));
  TSB_TRY(paged_map(&mv, dtype, a.V, a, kPtKeys));
  const int q_boxes = kPtRows % a.G == 0 && a.q_row > 0 && a.q_row < paged_stride_most && (a.H == 1 || (a.q_head > 0 && a.q_head < paged_stride_most));
  if (q_boxes) TSB_TRY(pt_map_q(&mq, dtype, a));
  else mq = mk;
  paged_tc_kernel<H, BX, NS><<<st->sm_count, kPtThreads, smem, s>>>(mk, mv, mq, a, q_boxes);
  count_launch(device);
  return check_launch("paged_tc");
}

int launch_paged_tc(int device, DeviceState* st, int dtype, PagedArgs a, cudaStream_t s) {
  a.wait_limit = tc_wait_limit();
  a.error = tc_error_word(device);
  // us with ends moved by up to 1 | 4 units: 2 x 30 rows over 4096 24 | 28, 256 over 8192 53 | 57, a prompt of 1024 of heads of 64 29 | 28
  a.min_units = 4;
  a.snap = 1;
  a.start = 2;
  st->waits = true;
  if (dtype == TSB200_F16) {
    if (a.hd == 64) TSB_TRY((pt_launch<__half, 1, 4>(device, st, a, s)));
    else TSB_TRY((pt_launch<__half, 2, 2>(device, st, a, s)));
  } else {
    if (a.hd == 64) TSB_TRY((pt_launch<__nv_bfloat16, 1, 4>(device, st, a, s)));
    else TSB_TRY((pt_launch<__nv_bfloat16, 2, 2>(device, st, a, s)));
  }
  return launch_paged_combine(device, dtype, a, kPtTile, st->sm_count, s);
}

}  // namespace tsb
