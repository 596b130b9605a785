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
constexpr int kVerifyMaxSegs = 512;        // vocabularies up to 524288; at most 16 a lane
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
  double turn[32][33];                     // the weights of the segment that holds the number
  int ok[kVerifyMaxDrafts];
  int any;                                 // the distribution has a weight above zero
};

// The sum of one row's segments, by a warp.
__device__ __forceinline__ double verify_row_sum(const double* s, int segs) {
  double v = 0.0;
  for (int i = threadIdx.x & 31; i < segs; i += 32) v += __ldcg(s + i);
  return warp_sum_f64(v);
}

__device__ __forceinline__ double warp_inclusive_f64(double v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double x = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += x;
  }
  return v;
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
  const double* sums = P.sums + (long long)b * rows * segs;
  if (tid == 0) S.any = 0;
  // what was drafted, before the dependency: none of it comes from the first launch
  double pd = 0.0, qd = 1.0, ut = 0.0;
  if (warp < len) {
    const long long d = __ldg(tokens + warp);
    const bool known = d >= 0 && d < V;                            // any other token is refused
    ut = double(__ldg(u + warp));
    if (known) pd = verify_weight(__ldg(target + warp * P.target_row + d));
    if (known && draft) qd = verify_weight(__ldg(draft + warp * P.draft_row + d));
  }
  griddep_wait();
  for (int r = warp; r <= len; r += kVerifyWarps) {
    const double p = verify_row_sum(sums + (long long)r * segs, segs);
    const double q = draft && r < len ? verify_row_sum(sums + (long long)(K + 1 + r) * segs, segs) : 1.0;
    if (r > warp && r < len) {                                     // beyond the first: rare, many drafts
      const long long d = __ldg(tokens + r);
      const bool known = d >= 0 && d < V;
      ut = double(__ldg(u + r));
      pd = known ? verify_weight(__ldg(target + r * P.target_row + d)) : 0.0;
      qd = known && draft ? verify_weight(__ldg(draft + r * P.draft_row + d)) : 1.0;
    }
    if (lane == 0) {
      S.p_sum[r] = p;
      if (r < len) {
        S.q_sum[r] = q;
        S.ok[r] = ut * qd * p < pd * q;
      }
    }
  }
  __syncthreads();
  int n = 0;
  while (n < len && S.ok[n]) ++n;
  // the distribution: 0 the row itself, 1 without the refused token, 2 what the draft leaves of it
  int kind = n == len ? 0 : draft ? 2 : 1;
  const float *pr = target + n * P.target_row, *qr = kind == 2 ? draft + n * P.draft_row : pr;
  const double Ps = S.p_sum[n], Qs = kind == 2 ? S.q_sum[n] : 1.0;
  const long long refused = kind ? __ldg(tokens + n) : -1;
  auto weight = [&](float pf, float qf, int i) -> double {
    const double p = verify_weight(pf);
    if (kind == 0) return p;
    if (kind == 1) return i == refused ? 0.0 : p;
    return fmax(p * Qs - verify_weight(qf) * Ps, 0.0);
  };
  constexpr int kPer = kVerifySeg / 32;
  VerifyShared* S0 = cluster.map_shared_rank(&S, 0);
  cluster.sync();                                                  // all CTAs run, so their shared memory exists
  for (;;) {                                                       // a second time where the first distribution is empty
    for (int s = rank * kVerifyWarps + warp; s < segs; s += C * kVerifyWarps) {
      const int first = s * kVerifySeg, m = V - first;
      double v = 0.0;
      if (kind == 0) {                                             // the first launch has these
        v = lane == 0 ? __ldcg(sums + (long long)n * segs + s) : 0.0;
      } else {
        float p[kPer], q[kPer];
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const int at = i * 32 + lane;
          p[i] = at < m ? __ldg(pr + first + at) : 0.f;
          q[i] = kind == 2 && at < m ? __ldg(qr + first + at) : 0.f;
        }
#pragma unroll
        for (int i = 0; i < kPer; ++i) v += weight(p[i], q[i], first + i * 32 + lane);
        v = warp_sum_f64(v);
      }
      if (lane == 0) {
        S0->seg[s] = v;
        if (v > 0.0)
          for (int c = 0; c < C; ++c) cluster.map_shared_rank(&S, c)->any = 1;
      }
    }
    cluster.sync();
    if (kind == 0 || S.any) break;                                 // the same in all CTAs
    kind = 0;
    cluster.sync();
  }
  if (rank != 0 || warp != 0) return;
  // the segment that holds the number: a lane has `per` consecutive ones
  const int per = (segs + 31) / 32, s0 = min(segs, lane * per), s1 = min(segs, s0 + per);
  double mine = 0.0;
  for (int s = s0; s < s1; ++s) mine += S.seg[s];
  const double upto = warp_inclusive_f64(mine), total = __shfl_sync(0xffffffffu, upto, 31), aim = double(__ldg(u + K)) * total;
  // the first with weight whose running sum reaches the aim, else (rounding) the last with weight
  auto choose = [&](bool some, bool reached) {
    const unsigned hit = __ballot_sync(0xffffffffu, some && reached), any = __ballot_sync(0xffffffffu, some);
    return hit ? __ffs(hit) - 1 : any ? 31 - __clz(any) : -1;
  };
  const int who = choose(mine > 0.0, upto >= aim);
  long long pick = -1;
  if (who >= 0) {
    double run = __shfl_sync(0xffffffffu, upto - mine, who);
    const int w0 = who * per;
    const double seg = lane < per && w0 + lane < segs ? S.seg[w0 + lane] : 0.0;
    const double seg_upto = warp_inclusive_f64(seg) + run;
    const int at = choose(seg > 0.0, seg_upto >= aim), first = (w0 + at) * kVerifySeg, m = V - first;
    run = __shfl_sync(0xffffffffu, seg_upto - seg, at);
    float p[kPer], q[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int j = i * 32 + lane;
      p[i] = j < m ? __ldg(pr + first + j) : 0.f;
      q[i] = kind == 2 && j < m ? __ldg(qr + first + j) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) S.turn[i][lane] = weight(p[i], q[i], first + i * 32 + lane);
    __syncwarp();
    double sum = 0.0;                                              // of the lane's 32 consecutive weights
#pragma unroll
    for (int i = 0; i < kPer; ++i) sum += S.turn[lane][i];
    const double sum_upto = warp_inclusive_f64(sum) + run;
    const int group = choose(sum > 0.0, sum_upto >= aim);
    run = __shfl_sync(0xffffffffu, sum_upto - sum, group);
    const double w = S.turn[group][lane], w_upto = warp_inclusive_f64(w) + run;
    pick = first + group * 32 + choose(w > 0.0, w_upto >= aim);
  }
  for (int i = lane; i <= K; i += 32) P.out[(long long)b * (K + 1) + i] = i < n ? __ldg(tokens + i) : i == n ? pick : -1;
  if (lane == 0) P.accepted[b] = n;
}

inline int verify_segs(int V) { return (V + kVerifySeg - 1) / kVerifySeg; }

// CTAs per stream: as many as leave an SM to each, and at most one warp per segment.
inline int verify_cluster(int B, int segs, int sms) {
  int c = 1;
  while (c < kVerifyMaxCluster && (long long)B * 2 * c <= sms && segs > c * kVerifyWarps) c *= 2;
  return c;
}

}  // namespace b200
