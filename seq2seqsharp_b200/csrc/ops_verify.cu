// Check of drafted tokens against the target's probabilities, from given uniform numbers.
//
// Row i of a sequence holds the target's probabilities p_i after i drafted tokens; draft i was drawn from q_i (null: it was certain).  Draft i is accepted
// while u_i q_i(x_i) < p_i(x_i), which holds with probability min(1, p / q).  At the first refusal the token is drawn from max(p_i - q_i, 0), behind
// the last accepted draft from p_i: the smallest t with w_0 + .. + w_t > u (w_0 + .. + w_{V-1}).  So the tokens are distributed as the target's own.
// Products, differences and sums are 64-bit: u q is then exact, p - q off by 2^-53 of itself at most (exact unless the two are further apart than 2^29), and a sum of V
// weights by V 2^-53 of itself.  The order in which a vocabulary is added up can decide which token is drawn only where u times the whole is that near to the border of two.
//
// A cluster per sequence.  Its warps share the vocabulary in equal runs and push what theirs weigh to every CTA; after one cluster barrier all know the run that
// the draw falls into, and that warp's CTA shares it out once more.  Rows that no draw needs are not read.  What bounds it: four dependent reads of memory, the
// launch and the barriers for few sequences (one of 32000 words: 5.5 us; 44 with one CTA), and for many the latency of a warp's rounds of reads, four one after the other (64 of
// 50257 words, 25.7 MB: 11.7 us, 17.8 with one warp looking for the token and widening before the comparison; FP64 pipe 11 %, conversions 23 %, DRAM 20 % busy).
#include "kernels.cuh"

namespace tsb {

struct VerifyArgs {
  int* tokens;            // [B, K + 1]
  int* counts;            // [B]
  const float* p;         // rows of stride p_row
  const float* q;         // [B K] rows of stride q_row, may be null
  int64_t p_row, q_row;
  const int* draft;       // [B, K]
  const int* starts;      // [B + 1], or null: K + 1 rows each
  const float* u;         // [B, K + 1]: u[K] draws the last token
  int K, V, rows;
};
constexpr int kVerifyThreads = 512, kVerifyWarps = kVerifyThreads / 32, kVerifyMaxCtas = 8;

__device__ __forceinline__ void push_double(double* local, uint32_t cta, double v) {
  uint32_t ra;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"((uint32_t)__cvta_generic_to_shared(local)), "r"(cta));
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(ra), "d"(v) : "memory");
}
__device__ __forceinline__ double warp_scan(double v, int lane) {   // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  return v;
}

__global__ void __launch_bounds__(kVerifyThreads) verify_draft_kernel(const __grid_constant__ VerifyArgs a, int ctas) {
  __shared__ double parts[kVerifyWarps];
  __shared__ int over, weighs;   // first thread whose words pass the draw, last one whose words weigh anything
  __shared__ double sums[2][kVerifyMaxCtas * kVerifyWarps];   // of every warp's run: of max(p - q, 0), and of p
  const int b = (int)blockIdx.x / ctas, rank = (int)blockIdx.x % ctas, tid = threadIdx.x, lane = tid & 31, w = rank * kVerifyWarps + (tid >> 5);
  const int row0 = a.starts ? a.starts[b] : b * (a.K + 1);
  int n = a.starts ? a.starts[b + 1] - row0 : a.K + 1;
  if (row0 < 0 || n < 0 || n > a.rows - row0) n = 0;
  n = min(n, a.K + 1);
  int* out = a.tokens + (int64_t)b * (a.K + 1);
  if (n == 0) {   // of all of the cluster's CTAs
    if (rank == 0) {
      for (int i = tid; i <= a.K; i += kVerifyThreads) out[i] = -1;
      if (tid == 0) a.counts[b] = 0;
    }
    return;
  }
  cluster_arrive_relaxed();   // the other CTAs exist before anything is pushed to them
  const int* x = a.draft + (int64_t)b * a.K;
  const float* u = a.u + (int64_t)b * (a.K + 1);
  // every warp tests the drafts, a lane each
  int taken = 0;
  for (; taken < n - 1; taken += 32) {
    const int i = taken + lane;
    bool ok = false;
    if (i < n - 1) {
      const int t = x[i];
      if (t >= 0 && t < a.V) {
        const double q = a.q ? (double)a.q[((int64_t)b * a.K + i) * a.q_row + t] : 1.0;
        ok = (double)u[i] * q < (double)a.p[(int64_t)(row0 + i) * a.p_row + t];
      }
    }
    const unsigned bad = __ballot_sync(0xffffffffu, !ok);
    if (bad) {
      taken += __ffs(bad) - 1;
      break;
    }
  }
  taken = min(taken, n - 1);
  const bool refused = taken < n - 1;
  const float* p = a.p + (int64_t)(row0 + taken) * a.p_row;
  const float* q = refused && a.q ? a.q + ((int64_t)b * a.K + taken) * a.q_row : nullptr;
  const int certain = refused && !a.q ? x[taken] : -1;
  constexpr int N = 8;   // steps of 32 words on their way at a time
  float pt[N], qt[N];
  auto fetch = [&](int t0, int end) {
#pragma unroll
    for (int k = 0; k < N; ++k) pt[k] = t0 + 32 * k + lane < end ? p[t0 + 32 * k + lane] : 0.0f;
    if (q) {
#pragma unroll
      for (int k = 0; k < N; ++k) qt[k] = t0 + 32 * k + lane < end ? q[t0 + 32 * k + lane] : 0.0f;
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k) qt[k] = t0 + 32 * k + lane == certain ? 1.0f : 0.0f;
    }
  };
  // this warp's run of the vocabulary, 32 words at a time
  const int warps = ctas * kVerifyWarps, per = ((a.V + warps - 1) / warps + 31) & ~31, v0 = min((int64_t)a.V, (int64_t)w * per), v1 = min((int64_t)a.V, (int64_t)v0 + per);
  {
    double rest = 0.0, all = 0.0;
    for (int t0 = v0; t0 < v1; t0 += 32 * N) {
      fetch(t0, v1);
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const float x = fmaxf(pt[k], 0.0f);   // of NaN: 0
        all += (double)x;
        rest += x > qt[k] ? (double)x - (double)qt[k] : 0.0;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      rest += __shfl_xor_sync(0xffffffffu, rest, o);
      all += __shfl_xor_sync(0xffffffffu, all, o);
    }
    cluster_wait();
    if (lane < ctas) {
      push_double(&sums[0][w], lane, rest);
      push_double(&sums[1][w], lane, all);
    }
  }
  cluster_sync();
  // where nothing is left of p - q: p itself.  A lane has the runs of four neighbouring warps
  double run[4], before = 0.0, whole = 0.0;
  bool rest = refused;
  for (;; rest = false) {
    double mine = 0.0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      run[k] = lane * 4 + k < warps ? sums[rest ? 0 : 1][lane * 4 + k] : 0.0;
      mine += run[k];
    }
    const double to = warp_scan(mine, lane);
    before = to - mine;
    whole = __shfl_sync(0xffffffffu, to, 31);
    if (!rest || whole > 0.0) break;
  }
  if (rank == 0) {
    for (int i = tid; i <= a.K; i += kVerifyThreads)
      if (i != taken) out[i] = i < taken ? x[i] : -1;
    if (tid == 0) {
      a.counts[b] = taken + 1;
      if (!(whole > 0.0)) out[taken] = -1;
    }
  }
  if (!(whole > 0.0)) return;
  // the run that the draw falls into; where the sum rounded below u times the whole: the last one that weighs anything
  const double r = (double)u[a.K] * whole;
  int hit = 1 << 30, last = -1;
  double start = 0.0, at = before;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (run[k] > 0.0) {
      last = lane * 4 + k;
      if (hit == 1 << 30 && at + run[k] > r) hit = lane * 4 + k, start = at;
    }
    at += run[k];
  }
  const unsigned any = __ballot_sync(0xffffffffu, hit < 1 << 30);
  if (any) {
    const int src = __ffs(any) - 1;
    hit = __shfl_sync(0xffffffffu, hit, src);
    start = __shfl_sync(0xffffffffu, start, src);
  } else {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) last = max(last, __shfl_xor_sync(0xffffffffu, last, o));
    hit = last;
    start = r;   // its last word
  }
  if (hit / kVerifyWarps != rank) return;
  // its CTA shares the run out once more: so many neighbouring words to a thread
  const int h0 = (int)min((int64_t)a.V, (int64_t)hit * per), h1 = (int)min((int64_t)a.V, (int64_t)h0 + per), each = per > kVerifyThreads ? (per + kVerifyThreads - 1) / kVerifyThreads : 1;
  const int t0 = (int)min((int64_t)h1, (int64_t)h0 + (int64_t)tid * each), t1 = min(h1, t0 + each);
  auto weight = [&](int t) {
    const float pw = fmaxf(p[t], 0.0f), qw = q ? q[t] : t == certain ? 1.0f : 0.0f;
    return !rest ? (double)pw : pw > qw ? (double)pw - (double)qw : 0.0;
  };
  double mine = 0.0;
#pragma unroll 4
  for (int t = t0; t < t1; ++t) mine += weight(t);
  const double to = warp_scan(mine, lane);
  if (lane == 31) parts[tid >> 5] = to;
  if (tid == 0) over = kVerifyThreads, weighs = -1;
  __syncthreads();
  for (int i = 0; i < tid >> 5; ++i) start += parts[i];
  start += to - mine;
  if (mine > 0.0) {
    if (any && start + mine > r) atomicMin(&over, tid);
    atomicMax(&weighs, tid);
  }
  __syncthreads();
  const bool drawn = over < kVerifyThreads;
  if (tid != (drawn ? over : weighs)) return;
  int token = -1, some = -1;
  for (int t = t0; t < t1 && token < 0; ++t) {
    const double v = weight(t);
    start += v;
    if (v > 0.0) some = t;
    if (drawn && v > 0.0 && start > r) token = t;
  }
  out[taken] = token >= 0 ? token : some;
}

}  // namespace tsb

using namespace tsb;

extern "C" {

int TSB200_VerifyDraft(int device, int32_t* tokens, int32_t* counts, const float* p, int64_t p_row, const float* q, int64_t q_row, const int32_t* draft,
                       const int32_t* starts, const float* u, int B, int K, int V, int rows, void* stream) {
  TSB_CHECK(B >= 0 && K >= 0 && V >= 1 && rows >= 0, "verify_draft: %d sequences, %d drafts, %d words, %d rows", B, K, V, rows);
  TSB_CHECK(starts || (int64_t)B * (K + 1) <= rows, "verify_draft: %d rows, %d sequences of %d drafts need more", rows, B, K);
  TSB_CHECK((int64_t)B * kVerifyMaxCtas <= 0x7fffffff && V <= 0x40000000, "verify_draft: %d sequences of %d words", B, V);
  if (B == 0) return 1;
  TSB_CHECK(tokens && counts && (p || rows == 0) && (draft || K == 0) && u, "verify_draft: null pointer");
  KeepDevice keep;
  DeviceState* st;
  TSB_TRY(use_device(device, &st));
  VerifyArgs a{tokens, counts, p, q, p_row, q_row, draft, starts, u, K, V, rows};
  // as many CTAs to a sequence as are there at once (two on an SM), and at least 512 words to each
  int ctas = kVerifyMaxCtas;
  while (ctas > 1 && ((int64_t)B * ctas > 2 * st->sm_count || V < 512 * ctas)) ctas /= 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(B * ctas);
  cfg.blockDim = dim3(kVerifyThreads);
  cfg.stream = pick_stream(st, stream);
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = ctas;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  TSB_CUDA(cudaLaunchKernelEx(&cfg, verify_draft_kernel, a, ctas));
  count_launch(device);
  return check_launch("verify_draft");
}

}  // extern "C"
