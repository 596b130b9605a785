// The state of B streams after the first n_b of a step's T tokens, all blocks in one launch: what is left of a step when some
// of its drafted tokens are refused.  A recurrent state cannot drop its newest tokens, so the step's rows are kept (`trace`)
// and the state in front of it is moved on by the accepted ones:
//   rows 0, 1   layer norms of row n - 1 of the block's inputs and of its ffn's (the token-shift carries)
//   rows 2..4   n steps of the WKV recurrence over the kept keys and values
// Memory-bound: keys and values of the accepted tokens, two rows and the state are read, the state is written (32 blocks of 4096
// channels, 64 streams, 6 tokens, 573 MB: 100 us on the GPU, 108 per call; 12 blocks of 768, one stream: 2.9 and 7.9).
#pragma once

#include "common.cuh"

namespace b200 {

constexpr int kAdvanceThreads = 256;

struct AdvanceParams {
  const float *state, *trace, *params;   // [B][L][5][C]; [L][4][B][T][C]: x, x of the ffn, k, v; [L][5][C]: ln1 w, b, ln2 w, b, decay
  const long long* counts;
  float* out;                            // may be state
  int B, L, T, C;
};

// Grid (B * L, 2 + WKV chunks): CTAs 0 and 1 of a block's state take its layer norms, the others four channels per thread.
__global__ void __launch_bounds__(kAdvanceThreads) advance_state_kernel(const AdvanceParams P) {
  __shared__ float red[2][kAdvanceThreads / 32];
  const int b = blockIdx.x / P.L, l = blockIdx.x - b * P.L, C = P.C, T = P.T, tid = threadIdx.x;
  const long long asked = __ldg(P.counts + b);
  const int n = asked < 0 ? 0 : asked > T ? T : int(asked);
  const size_t so = (size_t(b) * P.L + l) * 5 * C;
  const float* par = P.params + size_t(l) * 5 * C;
  auto rows = [&](int which) { return P.trace + ((size_t(l) * 4 + which) * P.B + b) * T * C; };
  if (blockIdx.y < 2) {
    const int which = blockIdx.y;
    if (n == 0) {
      if (P.out != P.state)
        for (int i = tid; i < C; i += kAdvanceThreads) P.out[so + size_t(which) * C + i] = P.state[so + size_t(which) * C + i];
      return;
    }
    const float4* x = reinterpret_cast<const float4*>(rows(which) + size_t(n - 1) * C);
    const float4 *w = reinterpret_cast<const float4*>(par + size_t(2 * which) * C), *bias = reinterpret_cast<const float4*>(par + size_t(2 * which + 1) * C);
    auto total = [&](float v, float* s) {
      v = warp_sum(v);
      if ((tid & 31) == 0) s[tid >> 5] = v;
      __syncthreads();
      float a = 0.f;
      for (int i = 0; i < kAdvanceThreads / 32; ++i) a += s[i];
      return a;
    };
    float s = 0.f;
    for (int i = tid; i < C / 4; i += kAdvanceThreads) { const float4 v = __ldg(x + i); s += (v.x + v.y) + (v.z + v.w); }
    const float mean = total(s, red[0]) / float(C);
    s = 0.f;
    for (int i = tid; i < C / 4; i += kAdvanceThreads) {
      const float4 v = __ldg(x + i);
      const float a = v.x - mean, c = v.y - mean, d = v.z - mean, e = v.w - mean;
      s += (a * a + c * c) + (d * d + e * e);
    }
    const float dev = sqrtf(total(s, red[1]) / float(C) + 1e-5f);
    for (int i = tid; i < C / 4; i += kAdvanceThreads) {
      const float4 v = __ldg(x + i), ww = __ldg(w + i), bb = __ldg(bias + i);
      reinterpret_cast<float4*>(P.out + so + size_t(which) * C)[i] =
          make_float4(ww.x * ((v.x - mean) / dev) + bb.x, ww.y * ((v.y - mean) / dev) + bb.y, ww.z * ((v.z - mean) / dev) + bb.z,
                      ww.w * ((v.w - mean) / dev) + bb.w);
    }
    return;
  }
  const int c = ((blockIdx.y - 2) * kAdvanceThreads + tid) * 4;
  if (c >= C) return;
  auto four = [&](const float* p) { return *reinterpret_cast<const float4*>(p + c); };
  const float* st = P.state + so;
  float4 a = four(st + 2 * size_t(C)), d = four(st + 3 * size_t(C)), p = four(st + 4 * size_t(C));
  const float4 w = four(par + 4 * size_t(C));
  const float *k = rows(2), *v = rows(3);
#pragma unroll 4
  for (int t = 0; t < n; ++t) {
    const float4 kk = four(k + size_t(t) * C), vv = four(v + size_t(t) * C);
    wkv_advance(kk.x, vv.x, w.x, a.x, d.x, p.x);
    wkv_advance(kk.y, vv.y, w.y, a.y, d.y, p.y);
    wkv_advance(kk.z, vv.z, w.z, a.z, d.z, p.z);
    wkv_advance(kk.w, vv.w, w.w, a.w, d.w, p.w);
  }
  if (n == 0 && P.out == P.state) return;
  float* o = P.out + so + c;
  *reinterpret_cast<float4*>(o + 2 * size_t(C)) = a;
  *reinterpret_cast<float4*>(o + 3 * size_t(C)) = d;
  *reinterpret_cast<float4*>(o + 4 * size_t(C)) = p;
}

}  // namespace b200
