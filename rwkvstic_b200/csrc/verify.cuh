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
// Bounds (times on the GPU alone; a call costs 2 us more, one of a single stream 7): the first launch by memory and by turning
// weights into fp64, 16 a clock and SM (256 streams, vocabulary 50277, 1150 rows looked at, 231 MB: 41 us), the second by latency (the same 256 streams, no draft distribution: 12 us, part of it
// beside the first, 19 where it formed all segments anew; 1 stream of 4 drafted tokens: 9.8 us for both).  All in one launch of
// a cluster per stream was slower where a stream is alone, 13.9 us against 9.8, since eight CTAs then sum what 50 times more
// warps do here.
#pragma once

#include <cooperative_groups.h>

#include <utility>

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
__device__ __forceinline__ double verify_weight(float w) { return double(fmaxf(w, 0.f)); }
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
  double s[4] = {0.0, 0.0, 0.0, 0.0};                            // four chains: an addition waits long for the one before
#pragma unroll
  for (int i = 0; i < kVerifySeg / 32; ++i) s[i & 3] += verify_weight(w[i]);
  const double all = warp_sum_f64((s[0] + s[1]) + (s[2] + s[3]));
  if (lane == 0) P.sums[row_id * P.segs + seg] = all;
}

struct VerifyShared {
  double p_sum[kVerifyMaxDrafts + 1], q_sum[kVerifyMaxDrafts];
  double seg[kVerifyMaxSegs];              // of the distribution that is drawn from; rank 0's is used
  double turn[32][33];                     // the weights of the segment that holds the number
  int ok[kVerifyMaxDrafts];
  int any;                                 // the distribution has a weight above zero
};

// The sums of the segments of one row, or of two (b may be null), by a warp.
__device__ __forceinline__ double2 verify_row_sums(const double* a, const double* b, int segs) {
  double2 v = make_double2(0.0, 0.0);
  for (int i = threadIdx.x & 31; i < segs; i += 32) {
    const double p = __ldcg(a + i), q = b ? __ldcg(b + i) : 0.0;
    v.x += p; v.y += q;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const double p = __shfl_xor_sync(0xffffffffu, v.x, o), q = __shfl_xor_sync(0xffffffffu, v.y, o);
    v.x += p; v.y += q;
  }
  return v;
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

// The distribution that a stream's token is drawn from.  One form per kind, without branches per weight: the 50 segments of a
// vocabulary of 50277 are some 3000 weights a warp and stream, and instructions are what this costs.
enum { VERIFY_TARGET, VERIFY_OTHERS, VERIFY_LEFT };        // the row itself; without the refused token; what the draft leaves of it
struct VerifyRow {
  const float *p, *q;
  double Ps, Qs;
  int V, refused;                                          // VERIFY_OTHERS: the refused token, or -1
};
template <int KIND>
__device__ __forceinline__ double verify_value(float p, float q, const VerifyRow& R) {
  const double pd = verify_weight(p);
  if (KIND != VERIFY_LEFT) return pd;
  // each product rounded: as one fused operation equal rows would leave the rounding errors of one of them
  const double v = __dsub_rn(__dmul_rn(pd, R.Qs), __dmul_rn(verify_weight(q), R.Ps));
  const int hi = __double2hiint(v), keep = ~(hi >> 31);    // zero where negative
  return __hiloint2double(hi & keep, __double2loint(v) & keep);
}
// put(i, value) for the 32 weights i * 32 + lane of a segment, 16 requested at a time
template <int KIND, typename Put>
__device__ __forceinline__ void verify_segment(const VerifyRow& R, int seg, Put put) {
  constexpr int kPer = kVerifySeg / 32, kHalf = kPer / 2;
  const int lane = threadIdx.x & 31, first = seg * kVerifySeg, m = R.V - first;
  const float *pr = R.p + first + lane, *qr = KIND == VERIFY_LEFT ? R.q + first + lane : nullptr;
  const int gone = KIND == VERIFY_OTHERS && (R.refused & 31) == lane ? (R.refused - first) >> 5 : -1;   // the lane's weight that does not count
#pragma unroll
  for (int h = 0; h < kPer; h += kHalf) {
    float p[kHalf], q[kHalf];
    if (m >= kVerifySeg) {
#pragma unroll
      for (int i = 0; i < kHalf; ++i) {
        p[i] = __ldg(pr + (h + i) * 32);
        q[i] = KIND == VERIFY_LEFT ? __ldg(qr + (h + i) * 32) : 0.f;
      }
    } else {
#pragma unroll
      for (int i = 0; i < kHalf; ++i) {
        const bool in = (h + i) * 32 + lane < m;
        p[i] = in ? __ldg(pr + (h + i) * 32) : 0.f;
        q[i] = KIND == VERIFY_LEFT && in ? __ldg(qr + (h + i) * 32) : 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < kHalf; ++i) put(h + i, verify_value<KIND>(KIND == VERIFY_OTHERS && h + i == gone ? 0.f : p[i], q[i], R));
  }
}
template <int KIND>
__device__ __forceinline__ double verify_segment_sum(const VerifyRow& R, int seg) {
  double c[4] = {0.0, 0.0, 0.0, 0.0};                      // four chains: an addition waits long for the one before
  verify_segment<KIND>(R, seg, [&](int i, double v) { c[i & 3] += v; });
  return warp_sum_f64((c[0] + c[1]) + (c[2] + c[3]));
}

__global__ void __launch_bounds__(kVerifyThreads, 2) verify_draw_kernel(const VerifyParams P) {
  namespace cg = cooperative_groups;
  __shared__ VerifyShared S;
  if (threadIdx.x == 0) S.any = 0;
  const cg::cluster_group cluster = cg::this_cluster();
  auto started = cluster.barrier_arrive();                         // met before the first access to another CTA's memory
  const int C = int(cluster.num_blocks()), rank = int(cluster.block_rank()), b = int(blockIdx.x) / C;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, K = P.K, V = P.V, segs = P.segs;
  const int rows = K + 1 + (P.draft ? K : 0), len = verify_length(P, b);
  const float *target = P.target + b * P.target_stream, *draft = P.draft ? P.draft + b * P.draft_stream : nullptr;
  const long long* tokens = P.tokens + (long long)b * K;
  const float* u = P.u + (long long)b * (K + 1);
  const double* sums = P.sums + (long long)b * rows * segs;
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
    const bool drafted = draft && r < len;
    const double2 both = verify_row_sums(sums + (long long)r * segs, drafted ? sums + (long long)(K + 1 + r) * segs : nullptr, segs);
    const double p = both.x, q = drafted ? both.y : 1.0;
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
  int kind = n == len ? VERIFY_TARGET : draft ? VERIFY_LEFT : VERIFY_OTHERS;
  VerifyRow R;
  R.p = target + n * P.target_row; R.q = kind == VERIFY_LEFT ? draft + n * P.draft_row : nullptr;
  R.Ps = S.p_sum[n]; R.Qs = kind == VERIFY_LEFT ? S.q_sum[n] : 1.0; R.V = V;
  const long long d = kind == VERIFY_OTHERS ? __ldg(tokens + n) : -1;
  R.refused = d >= 0 && d < V ? int(d) : -1;
  const int refused_seg = R.refused >= 0 ? R.refused / kVerifySeg : -1;
  cluster.barrier_wait(std::move(started));                        // all CTAs run, so their shared memory exists, and S.any is set
  VerifyShared* S0 = cluster.map_shared_rank(&S, 0);
  for (;;) {                                                       // a second time where the first distribution is empty
    for (int s = rank * kVerifyWarps + warp; s < segs; s += C * kVerifyWarps) {
      // the first launch has the target's own, also where a refused token is elsewhere
      const double v = kind == VERIFY_TARGET || (kind == VERIFY_OTHERS && s != refused_seg) ? __ldcg(sums + (long long)n * segs + s)
                       : kind == VERIFY_LEFT ? verify_segment_sum<VERIFY_LEFT>(R, s) : verify_segment_sum<VERIFY_OTHERS>(R, s);
      if (lane == 0) {
        S0->seg[s] = v;
        if (v > 0.0)
          for (int c = 0; c < C; ++c) cluster.map_shared_rank(&S, c)->any = 1;
      }
    }
    cluster.sync();
    if (kind == VERIFY_TARGET || S.any) break;                     // the same in all CTAs
    kind = VERIFY_TARGET;
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
    const int at = choose(seg > 0.0, seg_upto >= aim);
    run = __shfl_sync(0xffffffffu, seg_upto - seg, at);
    auto put = [&](int i, double v) { S.turn[i][lane] = v; };
    if (kind == VERIFY_TARGET) verify_segment<VERIFY_TARGET>(R, w0 + at, put);
    else if (kind == VERIFY_LEFT) verify_segment<VERIFY_LEFT>(R, w0 + at, put);
    else verify_segment<VERIFY_OTHERS>(R, w0 + at, put);
    __syncwarp();
    double c[4] = {0.0, 0.0, 0.0, 0.0};                            // of the lane's 32 consecutive weights
#pragma unroll
    for (int i = 0; i < kVerifySeg / 32; ++i) c[i & 3] += S.turn[lane][i];
    const double sum = (c[0] + c[1]) + (c[2] + c[3]);
    const double sum_upto = warp_inclusive_f64(sum) + run;
    const int group = choose(sum > 0.0, sum_upto >= aim);
    run = __shfl_sync(0xffffffffu, sum_upto - sum, group);
    const double w = S.turn[group][lane], w_upto = warp_inclusive_f64(w) + run;
    pick = (long long)(w0 + at) * kVerifySeg + group * 32 + choose(w > 0.0, w_upto >= aim);
  }
  for (int i = lane; i <= K; i += 32) P.out[(long long)b * (K + 1) + i] = i < n ? __ldg(tokens + i) : i == n ? pick : -1;
  if (lane == 0) P.accepted[b] = n;
}

inline int verify_segs(int V) { return (V + kVerifySeg - 1) / kVerifySeg; }

// CTAs per stream: as many as run at once, two per SM, and at most a warp per segment.
inline int verify_cluster(int B, int segs, int sms) {
  int c = 1;
  while (c < kVerifyMaxCluster && (long long)B * c <= sms && segs > c * kVerifyWarps) c *= 2;
  return c;
}

}  // namespace b200
