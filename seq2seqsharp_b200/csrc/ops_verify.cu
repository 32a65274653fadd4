// Check of drafted tokens against the target's probabilities, from given uniform numbers.
//
// Row i of a sequence holds the target's probabilities p_i after i drafted tokens; draft i was drawn from q_i (null: it was certain).  Draft i is accepted
// while u_i q_i(x_i) < p_i(x_i), which holds with probability min(1, p / q).  At the first refusal the token is drawn from max(p_i - q_i, 0), behind
// the last accepted draft from p_i: the smallest t with w_0 + .. + w_t > u (w_0 + .. + w_{V-1}).  So the tokens are distributed as the target's own.
// Products, differences and sums are 64-bit: u q and p - q are then exact, and a sum's rounding is far below the distance of two fp32 weights, so that
// the order in which a vocabulary is added up does not decide which token is drawn.
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
constexpr int kVerifyThreads = 512;

__global__ void __launch_bounds__(kVerifyThreads) verify_draft_kernel(const __grid_constant__ VerifyArgs a) {
  __shared__ double sums[kVerifyThreads / 32];
  __shared__ int found, last;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const int row0 = a.starts ? a.starts[b] : b * (a.K + 1);
  int n = a.starts ? a.starts[b + 1] - row0 : a.K + 1;
  if (row0 < 0 || n < 0 || n > a.rows - row0) n = 0;
  n = min(n, a.K + 1);
  int* out = a.tokens + (int64_t)b * (a.K + 1);
  if (n == 0) {
    for (int i = tid; i <= a.K; i += kVerifyThreads) out[i] = -1;
    if (tid == 0) a.counts[b] = 0;
    return;
  }
  const int* x = a.draft + (int64_t)b * a.K;
  const float* u = a.u + (int64_t)b * (a.K + 1);
  // every thread tests the drafts for itself: a handful of loads
  int taken = 0;
  for (; taken < n - 1; ++taken) {
    const int t = x[taken];
    if (t < 0 || t >= a.V) break;
    const double q = a.q ? (double)a.q[((int64_t)b * a.K + taken) * a.q_row + t] : 1.0;
    if (!((double)u[taken] * q < (double)a.p[(row0 + taken) * a.p_row + t])) break;
  }
  const float* p = a.p + (row0 + taken) * a.p_row;
  const bool refused = taken < n - 1;
  const float* q = refused && a.q ? a.q + ((int64_t)b * a.K + taken) * a.q_row : nullptr;
  const int certain = refused && !a.q ? x[taken] : -1;
  // a thread's run of the vocabulary
  const int per = (a.V + kVerifyThreads - 1) / kVerifyThreads, v0 = min(a.V, tid * per), v1 = min(a.V, v0 + per);
  auto weight = [&](int t, bool rest) {
    double x = (double)p[t];
    if (rest) x -= q ? (double)q[t] : (t == certain ? 1.0 : 0.0);
    return x > 0.0 ? x : 0.0;
  };
  for (int round = refused ? 0 : 1; round < 2; ++round) {   // where nothing is left of p - q: p itself
    const bool rest = round == 0;
    double mine = 0.0;
    for (int t = v0; t < v1; ++t) mine += weight(t, rest);
    double s = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += y;
    }
    __syncthreads();
    if (lane == 31) sums[w] = s;
    if (tid == 0) {
      found = a.V;
      last = -1;
    }
    __syncthreads();
    double before = 0.0, all = 0.0;
    for (int i = 0; i < kVerifyThreads / 32; ++i) {
      if (i < w) before += sums[i];
      all += sums[i];
    }
    if (!(all > 0.0)) continue;
    const double r = (double)u[a.K] * all;
    double at = before + s - mine;
    int some = -1;
    for (int t = v0; t < v1; ++t) {
      const double x = weight(t, rest);
      at += x;
      if (x > 0.0) some = t;
      if (x > 0.0 && at > r) {
        atomicMin(&found, t);
        break;
      }
    }
    if (some >= 0) atomicMax(&last, some);
    __syncthreads();
    if (tid == 0 && found == a.V) found = last;   // a sum that rounded below u times the whole
    __syncthreads();
    break;
  }
  __syncthreads();
  for (int i = tid; i <= a.K; i += kVerifyThreads) out[i] = i < taken ? x[i] : (i == taken && found < a.V ? found : -1);
  if (tid == 0) a.counts[b] = taken + 1;
}

}  // namespace tsb

using namespace tsb;

extern "C" {

int TSB200_VerifyDraft(int device, int32_t* tokens, int32_t* counts, const float* p, int64_t p_row, const float* q, int64_t q_row, const int32_t* draft,
                       const int32_t* starts, const float* u, int B, int K, int V, int rows, void* stream) {
  TSB_CHECK(B >= 0 && K >= 0 && V >= 1 && rows >= 0, "verify_draft: %d sequences, %d drafts, %d words, %d rows", B, K, V, rows);
  TSB_CHECK(starts || (int64_t)B * (K + 1) <= rows, "verify_draft: %d rows, %d sequences of %d drafts need more", rows, B, K);
  if (B == 0) return 1;
  TSB_CHECK(tokens && counts && (p || rows == 0) && (draft || K == 0) && u, "verify_draft: null pointer");
  KeepDevice keep;
  DeviceState* st;
  TSB_TRY(use_device(device, &st));
  VerifyArgs a{tokens, counts, p, q, p_row, q_row, draft, starts, u, K, V, rows};
  verify_draft_kernel<<<B, kVerifyThreads, 0, pick_stream(st, stream)>>>(a);
  count_launch(device);
  return check_launch("verify_draft");
}

}  // extern "C"
