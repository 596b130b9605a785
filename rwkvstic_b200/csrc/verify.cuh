// Verification of drafted tokens on the device.  Per stream: drafted token d of step t is accepted where
//   u_t q_t(d) / Q_t < p_t(d) / P_t          (p: the target's weights of the step, P their sum; q, Q: the draft's)
// up to the first refusal; there one token is drawn from max(0, p/P - q/Q), or, with every drafted token accepted, from the
// target's next row.  What comes out is distributed as if every token had been drawn from the target.
//
// Sums, products and comparisons are fp64: a draw among 50277 tokens meets a border that sums of 24 bits misplace in one of
// a thousand cases.  Weights of the steps need not sum to one, so the sums of all rows that may be looked at come first,
// one warp per segment of 1024 weights (verify_sums_kernel); the second launch (verify_draw_kernel, a cluster of CTAs per
// stream) adds the segments of a row in their order, decides, forms the remaining distribution in the same segments, and walks
// to the segment, then the token, that holds the uniform number.  The segments depend on the vocabulary alone, so a stream's
// result does not depend on the other streams of the call.
// Bounds: the first launch by memory (one pass over the rows), the second by the latency of its few steps.
#pragma once

#include <cooperative_groups.h>

#include "common.cuh"

namespace b200 {

constexpr int kVerifySeg = 1024;           // weights per segment
constexpr int kVerifySumWarps = 8;
constexpr int kVerifyThreads = 512, kVerifyWarps = kVerifyThreads / 32;
constexpr int kVerifyMaxDrafts = 64;
constexpr int kVerifyMaxSegs = 512;        // vocabularies up to 524288
constexpr int kVerifyMaxCluster = 8;

struct VerifyParams {
  const float *target, *draft;             // draft null: the draft is sure of its tokens
  long long target_stream, target_row, draft_stream, draft_row;   // strides in elements
  const long long *tokens, *lengths;       // lengths null: all of the drafts
  const float* u;                          // [B][K + 1]
  double* sums;                            // [B][rows][segs]: K + 1 target rows, then K draft rows
  long long *out, *accepted;               // [B][K + 1], [B]
  int B, K, V, segs;
};

__device__ __forceinline__ int verify_length(const VerifyParams& P, int b) {
  if (!P.lengths) return P.K;
  const long long n = __ldg(P.lengths + b);
  return n < 0 ? 0 : n > P.K ? P.K : int(n);
}
// a weight counts where it is above zero (so not where it is NaN)
__device__ __forceinline__ double verify_weight(float w) { return w > 0.f ? double(w) : 0.0; }
__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__global__ void __launch_bounds__(kVerifySumWarps * 32) verify_sums_kernel(const VerifyParams P) {
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rows = P.K + 1 + (P.draft ? P.K : 0);
  const long long item = (long long)blockIdx.x * kVerifySumWarps + warp, row_id = item / P.segs;
  const int seg = int(item - row_id * P.segs), b = int(row_id / rows), r = int(row_id - (long long)b * rows);
  if (b >= P.B) return;
  const int len = verify_length(P, b);
  if (r <= P.K ? r > len : r - P.K - 1 >= len) return;             // never looked at
  const float* row = r <= P.K ? P.target + b * P.target_stream + r * P.target_row
                              : P.draft + b * P.draft_stream + (r - P.K - 1) * P.draft_row;
  const int first = seg * kVerifySeg, n = min(kVerifySeg, P.V - first);
  float w[kVerifySeg / 32];
#pragma unroll
  for (int i = 0; i < kVerifySeg / 32; ++i) w[i] = i * 32 + lane < n ? __ldg(row + first + i * 32 + lane) : 0.f;
  double s = 0.0;
#pragma unroll
  for (int i = 0; i < kVerifySeg / 32; ++i) s += verify_weight(w[i]);
  s = warp_sum_f64(s);
  if (lane == 0) P.sums[row_id * P.segs + seg] = s;
}

struct VerifyShared {
  double p_sum[kVerifyMaxDrafts + 1], q_sum[kVerifyMaxDrafts];
  double seg[kVerifyMaxSegs];              // of the distribution that is drawn from; rank 0's is used
  int ok[kVerifyMaxDrafts];
  double P, Q;
  int accepted, length, token;             // token: the refused one
  int found;
  double before, total;
};

// The sum of one row's segments, by a warp.
__device__ __forceinline__ double verify_row_sum(const double* s, int segs) {
  double v = 0.0;
  for (int i = threadIdx.x & 31; i < segs; i += 32) v += __ldcg(s + i);
  return warp_sum_f64(v);
}

__global__ void __launch_bounds__(kVerifyThreads) verify_draw_kernel(const VerifyParams P) {
  namespace cg = cooperative_groups;
  __shared__ VerifyShared S;
  const cg::cluster_group cluster = cg::this_cluster();
  const int C = int(cluster.num_blocks()), rank = int(cluster.block_rank()), b = int(blockIdx.x) / C;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, K = P.K, V = P.V, segs = P.segs;
  const int rows = K + 1 + (P.draft ? K : 0), len = verify_length(P, b);
  const float *target = P.target + b * P.target_stream, *draft = P.draft ? P.draft + b * P.draft_stream : nullptr;
  const long long* tokens = P.tokens + (long long)b * K;
  const float* u = P.u + (long long)b * (K + 1);
  griddep_wait();
  const double* sums = P.sums + (long long)b * rows * segs;
  for (int r = warp; r <= len; r += kVerifyWarps) {
    const double p = verify_row_sum(sums + (long long)r * segs, segs);
    const double q = draft && r < len ? verify_row_sum(sums + (long long)(K + 1 + r) * segs, segs) : 1.0;
    if (lane == 0) {
      S.p_sum[r] = p;
      if (r < len) {
        S.q_sum[r] = q;
        const long long d = __ldg(tokens + r);
        const bool known = d >= 0 && d < V;                        // any other token is refused
        const double pd = known ? verify_weight(__ldg(target + r * P.target_row + d)) : 0.0;
        const double qd = known && draft ? verify_weight(__ldg(draft + r * P.draft_row + d)) : 1.0;
        S.ok[r] = double(u[r]) * qd * p < pd * q;
      }
    }
  }
  __syncthreads();
  int n = 0;
  while (n < len && S.ok[n]) ++n;
  // the distribution: 0 the row itself, 1 without the refused token, 2 what the draft leaves of it
  const int kind = n == len ? 0 : draft ? 2 : 1;
  const float *pr = target + n * P.target_row, *qr = kind == 2 ? draft + n * P.draft_row : nullptr;
  const double Ps = S.p_sum[n], Qs = kind == 2 ? S.q_sum[n] : 1.0;
  const long long refused = kind ? __ldg(tokens + n) : -1;
  auto weight = [&](int i, int how) -> double {
    const double p = verify_weight(__ldg(pr + i));
    if (how == 0) return p;
    if (how == 1) return i == refused ? 0.0 : p;
    return fmax(p * Qs - verify_weight(__ldg(qr + i)) * Ps, 0.0);
  };
  VerifyShared* S0 = cluster.map_shared_rank(&S, 0);
  cluster.sync();                                                  // all CTAs run, so their shared memory exists
  int how = kind;
  for (;;) {                                                       // a second time where the first distribution is empty
    for (int s = rank * kVerifyWarps + warp; s < segs; s += C * kVerifyWarps) {
      double v = 0.0;
#pragma unroll 8
      for (int i = 0; i < kVerifySeg / 32; ++i) {
        const int at = s * kVerifySeg + i * 32 + lane;
        if (at < V) v += weight(at, how);
      }
      v = warp_sum_f64(v);
      if (lane == 0) S0->seg[s] = v;
    }
    cluster.sync();
    double any = 0.0;
    if (how) {
      for (int s = 0; s < segs; ++s) any += S0->seg[s];
      cluster.sync();                                              // read before it is written again
    }
    if (how == 0 || any > 0.0) break;
    how = 0;
  }
  if (rank != 0) return;
  if (warp == 0) {
    double total = 0.0;
    for (int s = 0; s < segs; ++s) total += S.seg[s];
    const double aim = double(u[K]) * total;
    int found = -1;
    double run = 0.0, before = 0.0;
    for (int s = 0; s < segs; ++s) {
      const double v = S.seg[s];
      if (v > 0.0) {
        found = s; before = run;
        if (run + v >= aim) break;
      }
      run += v;
    }
    long long pick = -1;
    if (found >= 0) {
      run = before;
      for (int i = 0; i < kVerifySeg / 32; ++i) {
        const int at = found * kVerifySeg + i * 32 + lane;
        const double w = at < V ? weight(at, how) : 0.0;
        double inc = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double x = __shfl_up_sync(0xffffffffu, inc, o);
          if (lane >= o) inc += x;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, w > 0.0 && run + inc >= aim), some = __ballot_sync(0xffffffffu, w > 0.0);
        if (some) pick = found * kVerifySeg + i * 32 + (hit ? __ffs(hit) - 1 : 31 - __clz(some));
        if (hit) break;
        run += __shfl_sync(0xffffffffu, inc, 31);
      }
    }
    for (int i = lane; i <= K; i += 32) P.out[(long long)b * (K + 1) + i] = i < n ? tokens[i] : i == n ? pick : -1;
    if (lane == 0) P.accepted[b] = n;
  }
}

inline int verify_segs(int V) { return (V + kVerifySeg - 1) / kVerifySeg; }

// CTAs per stream: as many as leave an SM to each, and at most one warp per segment.
inline int verify_cluster(int B, int segs, int sms) {
  int c = 1;
  while (c < kVerifyMaxCluster && (long long)B * 2 * c <= sms && segs > c * kVerifyWarps) c *= 2;
  return c;
}

}  // namespace b200
