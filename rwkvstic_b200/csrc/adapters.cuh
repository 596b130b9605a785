// Low-rank adapters of many requests beside shared projections: out[row] = y[row] + scale[id] * (x[row] A[id]^T) B[id]^T
// for rows whose stream has adapter id, out[row] = y[row] for the others.  A [rank][K], B [N][rank] per adapter.
//
// h = x A^T has a long sum (K) and few columns (the rank), y + h B^T a short sum and many columns.  Three forms:
//   a cluster of eight CTAs per tile and matrix does both, for calls of a few tiles (adapt_fused_kernel);
//   two launches, the second started before the first ends, over gathered tiles of up to 16 rows (adapt_shrink_kernel and
//   adapt_expand_kernel below, mma.sync);
//   the same over tiles of 128 rows of one stream on tcgen05, where products are many (adapters_tiles.cuh, which has the rules).
// Rows of one adapter share its weights, so a tile is of one adapter.  Streams of 16 rows or more are cut into tiles; shorter
// ones are gathered: CTA s looks through the ids of its window of kAdaptWindow streams, in the order of the streams, and leads
// a tile where a multiple of 16 rows of its adapter ends in front of one of its rows.  So no pass sorts the rows and no count
// travels to the host; CTAs that lead nothing leave.
//
// Operands that are not of one 16-bit type are cut into bfloat16 pieces: a float is exactly three (the upper 8 bits of its
// significand, the next 8, the last 8), a half exactly two.  Products of pieces i and j with i + j of 3 and more are below 2^-21
// of the whole together and left out.  A piece of an infinity is NaN: a row of x that holds an infinity or a NaN comes out as NaN,
// where it has an adapter.
// The tensor cores cut the terms of a sum off at the last place of the largest, and its result, so chains are short before their
// part joins a sum that rounds, with the small products first, while the sum is small: in the first launch 32 k of a lane (64 where
// nothing is cut; tiles of 128 rows twice that), in the second 32 ranks (tiles: all of up to 128).  Lost on average where all terms
// are positive, in units of 2^-23 of the sum, fp32 throughout: 0.2 to 0.8 for any K or rank.  In the order of k one chain of 256
// ranks lost 57, of 128 k 20 and of 64 k 5 to 13, in the same time but for ranks of 256 (4 x 500 rows of 2048 -> 2048, fp32: 110 us
// in one chain, 117 joined).
// What bounds the gathered tiles is what they read and, at rank 64, the lanes that cut pieces (on the GPU alone): 7B key, value and
// receptance for 256 streams of 200 adapters (332 MB) 68 us, the first launch 33, the second 42, overlapping; 3B head for 48 x 5
// rows (115 MB) 33; 7B ffn for 64 streams of 48 adapters (56 MB) 23.  Fragments go from global memory to a lane's own slots of
// shared memory and from there to its registers, without a barrier between warps.  The index along a product is free to permute,
// and is, so that a lane's elements are consecutive: 16 bytes of A, 8 of B.
#pragma once

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

namespace b200 {

constexpr int kAdaptMaxMats = 3;
constexpr int kAdaptWindow = 1024;         // streams
constexpr int kAdaptMaxRank = 256;
constexpr int kAdaptRows = 16;             // of a gathered tile
constexpr int kAdaptMaxSplits = 8;         // of K: a cluster of CTAs
constexpr int kShrinkThreads = 256, kShrinkWarps = kShrinkThreads / 32;
constexpr int kExpandThreads = 256, kExpandWarps = kExpandThreads / 32;

struct AdaptParams {
  const void *a[kAdaptMaxMats], *b[kAdaptMaxMats], *x[kAdaptMaxMats], *y[kAdaptMaxMats];
  void* out[kAdaptMaxMats];
  const float* scale[kAdaptMaxMats];       // null: 1
  float* h[kAdaptMaxMats];                 // [rows][rank]
  int n_out[kAdaptMaxMats];
  int chunk_end[kAdaptMaxMats];            // second launch: column chunks of the matrices up to and including this one
  const long long* ids;
  int nmat, adapters, rank, K, R, T, streams, splits, chunk_cols, stages, ring;
};

__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// d = a b (no sum so far) or d += a b
template <bool HALF>
__device__ __forceinline__ void mma_to(bool first, float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (first) {
    if constexpr (HALF)
      asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
          : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
    else
      asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
          : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
  } else if constexpr (HALF) {
    mma_f16(d, a, b0, b1);
  } else {
    mma_bf16(d, a, b0, b1);
  }
}

// bfloat16 pieces that hold a value exactly.
template <typename T>
struct AdaptType;
template <> struct AdaptType<__nv_bfloat16> { static constexpr int kPieces = 1; };
template <> struct AdaptType<__half> { static constexpr int kPieces = 2; };
template <> struct AdaptType<float> { static constexpr int kPieces = 3; };

// The upper halves of two floats, and what they leave (exactly).
__device__ __forceinline__ uint32_t take_piece(float& lo, float& hi) {
  const uint32_t l = __float_as_uint(lo), u = __float_as_uint(hi);
  lo -= __uint_as_float(l & 0xffff0000u);
  hi -= __uint_as_float(u & 0xffff0000u);
  return __byte_perm(l, u, 0x7632);
}
template <int P>
__device__ __forceinline__ void split_pair(float lo, float hi, uint32_t (&p)[P]) {
#pragma unroll
  for (int i = 0; i < P; ++i) p[i] = take_piece(lo, hi);
}

// N consecutive elements of T, held as loaded.
template <typename T, int N>
struct AdaptRaw {
  static constexpr int kWords = N * int(sizeof(T)) / 4;
  uint32_t w[kWords];
  // pieces of the pair of elements 2i, 2i + 1
  template <int P>
  __device__ __forceinline__ void pair(int i, uint32_t (&p)[P]) const {
    if constexpr (P == 1) {
      p[0] = w[i];
    } else if constexpr (std::is_same<T, float>::value) {
      split_pair<P>(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]), p);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      split_pair<P>(f.x, f.y, p);
    }
  }
  // their first pieces alone
  __device__ __forceinline__ uint32_t first(int i) const {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) return w[i];
    uint32_t p[1];
    if constexpr (std::is_same<T, float>::value) {
      split_pair<1>(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]), p);
    } else if constexpr (std::is_same<T, __half>::value) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      split_pair<1>(f.x, f.y, p);
    }
    return p[0];
  }
};

// The rows of tile `tile` into rows[0..count): returns count, 0 where this CTA leads none.  *id: their adapter, -1: none.
// All threads of the CTA take part; mask: kAdaptWindow / 32 words of shared memory.
__device__ __forceinline__ int adapt_tile(const AdaptParams& P, int tile, int* rows, uint32_t* mask, int* id) {
  constexpr int rt = kAdaptRows;
  const int tid = threadIdx.x, nt = blockDim.x, T = P.T;
  auto id_of = [&](int s) {
    const long long v = __ldg(P.ids + s);
    return v >= 0 && v < P.adapters ? int(v) : -1;
  };
  if (T >= rt) {
    const int per = (T + rt - 1) / rt, s = tile / per, first = (tile - s * per) * rt, n = min(rt, T - first);
    *id = id_of(s);
    for (int i = tid; i < n; i += nt) rows[i] = s * T + first + i;
    __syncthreads();
    return n;
  }
  const int w0 = tile / kAdaptWindow * kAdaptWindow, count = min(kAdaptWindow, P.streams - w0);
  const int mine = id_of(tile);
  const int words = (count + 31) / 32;
  for (int i = tid; i < 32 * words; i += nt) {
    const unsigned m = __ballot_sync(0xffffffffu, i < count && id_of(w0 + i) == mine);
    if ((i & 31) == 0) mask[i >> 5] = m;
  }
  __syncthreads();
  int before = 0, all = 0;                               // streams of this adapter in front of this one, and in the window
  for (int w = 0; w < words; ++w) {
    const uint32_t m = mask[w];
    const int at = tile - w0 - 32 * w;                   // bits of this word in front of the stream's own
    before += __popc(at >= 32 ? m : at > 0 ? m & ((1u << at) - 1u) : 0u);
    all += __popc(m);
  }
  const int lead = (before * T + rt - 1) / rt * rt;      // the first tile that starts at or behind this stream's first row
  if (lead >= (before + 1) * T) return 0;
  const int n = min(rt, all * T - lead);
  *id = mine;
  if (tid < n) {
    int skip = (lead + tid) / T;                         // the stream of this row, counted among the adapter's
    const int token = lead + tid - skip * T;
    int w = 0;
    while (skip >= __popc(mask[w])) skip -= __popc(mask[w++]);
    uint32_t m = mask[w];
    for (; skip > 0; --skip) m &= m - 1;
    rows[tid] = (w0 + 32 * w + __ffs(m) - 1) * T + token;
  }
  __syncthreads();
  return n;
}

// The splits of a tile are a cluster, whose sums meet in shared memory, in the order of the splits:
// put(i, sum over the cluster's CTAs of part_sums[place(i)]) for i < n
template <typename Place, typename Put>
__device__ __forceinline__ void shrink_join(const AdaptParams& P, float* part_sums, int n, Place place, Put put) {
  const int S = P.splits, nt = blockDim.x;
  if (S == 1) {
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += nt) put(i, part_sums[place(i)]);
    return;
  }
  namespace cg = cooperative_groups;
  const cg::cluster_group cluster = cg::this_cluster();
  const int rank = int(cluster.block_rank());
  cluster.sync();
  // every CTA adds up a part of the table; all of a thread's remote reads are in flight at once
  for (int i = rank * nt + threadIdx.x; i < n; i += S * nt) {
    float v[kAdaptMaxSplits];
#pragma unroll
    for (int c = 0; c < kAdaptMaxSplits; ++c) v[c] = c < S ? *cluster.map_shared_rank(part_sums + place(i), c) : 0.f;
    float s = v[0];
#pragma unroll
    for (int c = 1; c < kAdaptMaxSplits; ++c) s += v[c];
    put(i, s);
  }
  cluster.sync();                          // the tables are read before their CTAs leave
}

// 16-byte units of a lane and block, and blocks in flight: as many as half an SM's shared memory holds.
template <typename TX, typename TW, int MT>
struct ShrinkRing {
  static constexpr int kA = int(sizeof(TW)) / 2, kX = int(sizeof(TX)) / 2, kUnits = MT * 2 * kA + 2 * kX, kStage = kUnits * 512;
  static constexpr int kFit = 104 * 1024 / (kShrinkWarps * kStage), kStages = kFit > 6 ? 6 : kFit, kBytes = kShrinkWarps * kStages * kStage;
  static constexpr int kSums = (kShrinkWarps * 16 * (16 * MT + 4) + 16 * 16 * MT) * 4, kSmem = kBytes > kSums ? kBytes : kSums;
  static_assert(kStages >= 2, "a block ahead of the one in use");
};

// The split's sums of a tile as a table [count][16 * MT] in shared memory, to be read after a barrier.
template <typename TX, typename TW, int MT, int NT>
__device__ __forceinline__ float* shrink_sums(const AdaptParams& P, const TX* x, const TW* a, int split, int chunk, const int* rows, int count,
                                              char* shared) {
  using Ring = ShrinkRing<TX, TW, MT>;
  constexpr bool kSame = std::is_same<TX, TW>::value && sizeof(TX) == 2;
  constexpr int PX = kSame ? 1 : AdaptType<TX>::kPieces, PW = kSame ? 1 : AdaptType<TW>::kPieces;
  constexpr int RC = 16 * MT, kStride = RC + 4, kStages = Ring::kStages;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int K = P.K, rank = P.rank;
  const int blocks = (K + 31) / 32, b0 = int((long long)blocks * split / P.splits), b1 = int((long long)blocks * (split + 1) / P.splits);
  const TX* xp[NT];
  uint32_t xok = 0;
#pragma unroll
  for (int q = 0; q < NT; ++q) {
    const int i = q * 8 + g;
    if (i < count) xok |= 1u << q;
    xp[q] = x + size_t(rows[i < count ? i : 0]) * K + 8 * t;
  }
  const TW* ap = a + size_t(chunk * RC + (chunk * RC + g < rank ? g : 0)) * K + 8 * t;
  const int have = (rank - chunk * RC - g + 7) / 8;        // of the lane's 2 MT rows of A, those that exist
  const size_t hop = size_t(8) * K;
  char* slots = shared + warp * (kStages * Ring::kStage) + lane * 16;
  const uint32_t slots_at = smem_u32(slots);
  int ask = b0 + warp;
  uint32_t to = 0;
  auto request = [&] {
    const int k = ask * 32;
    const bool in = ask < b1 && k + 8 * t < K;             // K is a multiple of 8
    const int at = in ? k : 0;
    uint32_t dst = slots_at + to;
#pragma unroll
    for (int m = 0; m < 2 * MT; ++m)
#pragma unroll
      for (int u = 0; u < Ring::kA; ++u, dst += 512) cp_async16(dst, (m < have ? ap + m * hop : ap) + at + u * 4, in && m < have);
#pragma unroll
    for (int q = 0; q < NT; ++q)
#pragma unroll
      for (int u = 0; u < Ring::kX; ++u, dst += 512) cp_async16(dst, xp[q] + at + u * 4, in && (xok >> q & 1));
    cp_async_commit();                                     // a group per block, also an empty one
    ask += kShrinkWarps;
    to = to == (kStages - 1) * Ring::kStage ? 0 : to + Ring::kStage;
  };
  float sum[MT][NT][4];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int q = 0; q < NT; ++q)
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[m][q][i] = 0.f;
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) request();
  const char* from = slots;
  auto take = [&](auto& raw, const char* at) {             // 8 elements
    constexpr int n = sizeof(raw.w) / 16;
#pragma unroll
    for (int u = 0; u < n; ++u) {
      const uint4 v = *reinterpret_cast<const uint4*>(at + u * 512);
      raw.w[4 * u] = v.x; raw.w[4 * u + 1] = v.y; raw.w[4 * u + 2] = v.z; raw.w[4 * u + 3] = v.w;
    }
  };
  for (int kb = b0 + warp; kb < b1; kb += 2 * kShrinkWarps) {   // two blocks; one past the end holds zeros
    float part[MT][NT][4];                                 // the tensor cores cut their sums off; the running sum rounds
    auto join = [&] {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int q = 0; q < NT; ++q)
#pragma unroll
          for (int i = 0; i < 4; ++i) sum[m][q][i] += part[m][q][i];
    };
#pragma unroll
    for (int o = 0; o < 2; ++o) {
      request();
      cp_async_wait<kStages - 1>();
      AdaptRaw<TX, 8> rx[NT];
      AdaptRaw<TW, 8> ra[MT][2];
#pragma unroll
      for (int m = 0; m < 2 * MT; ++m) take(ra[m >> 1][m & 1], from + m * Ring::kA * 512);
#pragma unroll
      for (int q = 0; q < NT; ++q) take(rx[q], from + (2 * MT * Ring::kA + q * Ring::kX) * 512);
      from = from == slots + (kStages - 1) * Ring::kStage ? slots : from + Ring::kStage;
      if constexpr (PX * PW > 1) {                         // small products of the block first, while the sum is small
#pragma unroll
        for (int step = 0; step < 2; ++step) {             // elements 4 step .. 4 step + 3 of every lane
          uint32_t fx[NT][2][PX], fa[MT][PW][4];
#pragma unroll
          for (int q = 0; q < NT; ++q)
#pragma unroll
            for (int i = 0; i < 2; ++i) rx[q].template pair<PX>(2 * step + i, fx[q][i]);
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t f[PW];
              ra[m][i & 1].template pair<PW>(2 * step + (i >> 1), f);
#pragma unroll
              for (int w = 0; w < PW; ++w) fa[m][w][i] = f[w];
            }
          bool first = step == 0;
#pragma unroll
          for (int i = PW - 1; i >= 0; --i)
#pragma unroll
            for (int j = PX - 1; j >= 0; --j) {
              if (i + j >= 3 || i + j == 0) continue;
#pragma unroll
              for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int q = 0; q < NT; ++q) mma_to<false>(first, part[m][q], fa[m][i], fx[q][0][j], fx[q][1][j]);
              first = false;
            }
        }
      }
#pragma unroll
      for (int step = 0; step < 2; ++step) {
        uint32_t fx[NT][2], fa[MT][4];
#pragma unroll
        for (int q = 0; q < NT; ++q)
#pragma unroll
          for (int i = 0; i < 2; ++i) fx[q][i] = kSame ? rx[q].w[2 * step + i] : rx[q].first(2 * step + i);
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int at = 2 * step + (i >> 1);
            fa[m][i] = kSame ? ra[m][i & 1].w[at] : ra[m][i & 1].first(at);
          }
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int q = 0; q < NT; ++q)
            mma_to<std::is_same<TX, __half>::value && kSame>(kSame && o == 0 && step == 0, part[m][q], fa[m], fx[q][0], fx[q][1]);
      }
      if constexpr (PX * PW > 1) join();
    }
    if constexpr (PX * PW == 1) join();
  }
  cp_async_wait<0>();
  __syncthreads();                                         // the slots become the table of sums
  float *red = reinterpret_cast<float*>(shared), *part_sums = red + kShrinkWarps * 16 * kStride;
  // products' rows are ranks (g, g + 8), their columns rows of x (2t, 2t + 1)
  float* mine = red + warp * (16 * kStride);
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int q = 0; q < NT; ++q)
#pragma unroll
      for (int i = 0; i < 4; ++i) mine[(q * 8 + 2 * t + (i & 1)) * kStride + m * 16 + (i >> 1) * 8 + g] = sum[m][q][i];
  __syncthreads();
  for (int i = threadIdx.x; i < count * RC; i += kShrinkThreads) {
    const int r = i / RC, j = i - r * RC;
    float s = 0.f;
    for (int w = 0; w < kShrinkWarps; ++w) s += red[(w * 16 + r) * kStride + j];
    part_sums[i] = s;
  }
  return part_sums;
}

// h[row][j] = sum_k x[row][k] A[id][j][k].  Grid (tiles * splits of K, rank chunks of 16 * MT, matrices).
// For tiles of 16 rows (as columns of the products, 8 at a time), which read little but their adapter.  A warp takes every eighth
// block of 32 k of the split; a lane copies its own 16-byte fragments of A and x into slots of its own, several blocks ahead, so
// that nothing but the end of the sums needs the other warps.
template <typename TX, typename TW, int MT>
__global__ void __launch_bounds__(kShrinkThreads, 2) adapt_shrink_kernel(const AdaptParams P) {
  extern __shared__ __align__(16) char shared[];
  __shared__ int rows[kAdaptRows];
  __shared__ uint32_t mask[kAdaptWindow / 32];
  griddep_launch_dependents();
  int id = -1;
  const int tile = blockIdx.x / P.splits, split = blockIdx.x - tile * P.splits, mat = blockIdx.z;
  const int count = adapt_tile(P, tile, rows, mask, &id);
  if (count == 0 || id < 0) return;        // the whole cluster
  const TX* x = static_cast<const TX*>(P.x[mat]);
  const TW* a = static_cast<const TW*>(P.a[mat]) + size_t(id) * P.rank * P.K;
  constexpr int RC = 16 * MT;
  const int chunk = blockIdx.y;
  float* sums = count <= 8 ? shrink_sums<TX, TW, MT, 1>(P, x, a, split, chunk, rows, count, shared)
                           : shrink_sums<TX, TW, MT, 2>(P, x, a, split, chunk, rows, count, shared);
  shrink_join(P, sums, count * RC, [](int i) { return i; }, [&](int i, float s) {
    const int r = i / RC, j = chunk * RC + i - r * RC;
    if (j < P.rank) P.h[mat][size_t(rows[r]) * P.rank + j] = s;
  });
}

template <typename TY>
__device__ __forceinline__ float adapt_float(TY v) {
  if constexpr (std::is_same<TY, float>::value) return v;
  else if constexpr (std::is_same<TY, __half>::value) return __half2float(v);
  else return __bfloat162float(v);
}
template <typename TY>
__device__ __forceinline__ void adapt_store(TY* p, float v) {
  if constexpr (std::is_same<TY, float>::value) *p = v;
  else if constexpr (std::is_same<TY, __half>::value) *p = __float2half_rn(v);
  else *p = __float2bfloat16_rn(v);
}

// W consecutive elements of a row (1, 2 or 4), held as loaded.
template <typename TY, int W>
struct AdaptFew {
  static constexpr int kBytes = W * int(sizeof(TY));
  using Word = std::conditional_t<kBytes == 16, uint4, std::conditional_t<kBytes == 8, uint2, std::conditional_t<kBytes == 4, uint32_t, unsigned short>>>;
  Word w;
  __device__ __forceinline__ void load(const TY* p) { w = *reinterpret_cast<const Word*>(p); }
  __device__ __forceinline__ void store(TY* p) const { *reinterpret_cast<Word*>(p) = w; }
  // + f[0 .. W), rounded once; W 2 only of fp32
  __device__ __forceinline__ void add_store(TY* p, const float* f) const {
    if constexpr (W == 1) {
      adapt_store(p, adapt_float(*reinterpret_cast<const TY*>(&w)) + f[0]);
    } else if constexpr (W == 2 && sizeof(TY) == 4) {
      const float2 d = *reinterpret_cast<const float2*>(f);
      *reinterpret_cast<float2*>(p) = make_float2(__uint_as_float(w.x) + d.x, __uint_as_float(w.y) + d.y);
    } else {
      const float4 d = *reinterpret_cast<const float4*>(f);
      if constexpr (sizeof(TY) == 4)
        *reinterpret_cast<float4*>(p) = make_float4(__uint_as_float(w.x) + d.x, __uint_as_float(w.y) + d.y, __uint_as_float(w.z) + d.z,
                                                    __uint_as_float(w.w) + d.w);
      else
        *reinterpret_cast<uint2*>(p) = make_uint2(add_pair(w.x, d.x, d.y), add_pair(w.y, d.z, d.w));
    }
  }
  static __device__ __forceinline__ uint32_t add_pair(uint32_t a, float x, float y) {
    if constexpr (std::is_same<TY, __half>::value) {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&a));
      const __half2 r = __floats2half2_rn(v.x + x, v.y + y);
      return *reinterpret_cast<const uint32_t*>(&r);
    } else {
      const __nv_bfloat162 r = __floats2bfloat162_rn(__uint_as_float(a << 16) + x, __uint_as_float(a & 0xffff0000u) + y);
      return *reinterpret_cast<const uint32_t*>(&r);
    }
  }
};

// Columns c_begin .. c_end of `count` rows: a warp per row, several accesses of a lane in flight.
template <typename TY, bool VEC>
__device__ __forceinline__ void adapt_copy(const TY* y, TY* out, const int* rows, int count, int N, int c_begin, int c_end) {
  constexpr int W = VEC ? 4 : 1, U = VEC ? 8 : 16;
  const int lane = threadIdx.x & 31, n = c_end - c_begin;
  for (int i = threadIdx.x >> 5; i < count; i += kExpandWarps) {
    const size_t at = size_t(rows[i]) * N + c_begin;
    const TY* from = y + at;
    TY* to = out + at;
    for (int c = lane * W; c < n; c += U * 32 * W) {
      AdaptFew<TY, W> few[U];
#pragma unroll
      for (int k = 0; k < U; ++k)
        if (c + k * 32 * W < n) few[k].load(from + c + k * 32 * W);
#pragma unroll
      for (int k = 0; k < U; ++k)
        if (c + k * 32 * W < n) few[k].store(to + c + k * 32 * W);
    }
  }
}

// The second launch, for tiles of up to 16 rows.  Shared memory: h in the fragments' own order, [8 rows][step of 16 ranks][piece]
// [lane] of 8 bytes; then per warp the stages of B and the table in which its sums are turned.
// KC: ranks of B per stage.  Stages leave shared memory to L1, which holds the lines of y that are on their way: 3B head for
// 48 x 5 rows 40 us with 4 stages of 16 ranks, 33 with 3 or 2.
template <typename TY, typename TW, int KC>
struct ExpandRing {
  static constexpr int MT = sizeof(TW) == 2 ? 4 : 2, kCols = 16 * MT;        // products of 16 columns that a warp forms at a time
  static constexpr int kLane = KC / 4 * int(sizeof(TW)), kUnit = kLane < 16 ? kLane : 16, kParts = kLane / kUnit;
  static constexpr int kStage = MT * 2 * 32 * kLane, kPitch = kCols + 4, kTurn = 16 * kPitch * 4;
  static constexpr int kStages = KC == 16 ? 3 : sizeof(TW) == 2 ? 2 : 3, kWarp = kStages * kStage + kTurn;
};
// h has all its 24 bits whatever the rows' type: two pieces (16 bits, cut) beside rows of 16 bits put 2.8 % of fp16 and 0.3 % of bf16
// results on a neighbouring value, and saved 2 us of 68 (7B key, value and receptance, 256 streams).
constexpr int kPiecesH = 3;
__host__ __device__ constexpr int expand_h_bytes(int rank, int kc) { return 2 * ((rank + kc - 1) / kc * (kc / 16)) * kPiecesH * 256; }

// Four ranks of a row of h into their fragments: 16 step + 4 t .. + 3 of a step and lane, or with 32 ranks a stage
// 32 (step / 2) + 8 t + 4 (step % 2) .. + 3.
template <int KC>
__device__ __forceinline__ void expand_put_h(char* shared, int ksteps, int r, int j4, float4 s) {
  constexpr int PH = kPiecesH;
  uint32_t lo[PH], hi[PH];
  split_pair<PH>(s.x, s.y, lo);
  split_pair<PH>(s.z, s.w, hi);
  const int ks = KC == 16 ? j4 >> 2 : (j4 >> 3) * 2 + (j4 & 1), t = KC == 16 ? j4 & 3 : (j4 >> 1) & 3;
  uint2* f = reinterpret_cast<uint2*>(shared) + ((r >> 3) * ksteps + ks) * PH * 32 + (r & 7) * 4 + t;
#pragma unroll
  for (int p = 0; p < PH; ++p) f[p * 32] = make_uint2(lo[p], hi[p]);
}

// NT: products of 8 rows; stage_h() puts the tile's h into shared memory.
template <typename TY, typename TW, int KC, bool VEC, int NT, typename StageH>
__device__ __forceinline__ void expand_columns(const AdaptParams& P, const TW* b, const TY* y, TY* out, int c0, int c_end, const size_t* row_at,
                                               int count, const char* shared, char* slots, StageH stage_h) {
  using Ring = ExpandRing<TY, TW, KC>;
  constexpr int PH = kPiecesH, PW = AdaptType<TW>::kPieces;
  constexpr int MT = Ring::MT, COLS = Ring::kCols, kStages = Ring::kStages, kStep = kExpandWarps * COLS;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int rank = P.rank, ksteps = (rank + KC - 1) / KC * (KC / 16);
  const uint2* hf = reinterpret_cast<const uint2*>(shared) + lane;
  float* turn = reinterpret_cast<float*>(slots + kStages * Ring::kStage);
  // a lane's columns of product m are 16 m + g and 16 m + g + 8, its ranks of a stage KC / 4 * t ..
  const bool wide = rank * int(sizeof(TW)) % 16 == 0;      // rows of B start on 16 bytes, else on 8
  const size_t hop = size_t(8) * rank;
  const uint32_t slots_at = smem_u32(slots) + lane * Ring::kUnit;
  int ask = c0, ask_k = 0;                                 // columns and rank that are requested next
  const TW* bp = b + size_t(c0 + g) * rank + KC / 4 * t;
  uint32_t to = 0;
  auto request = [&] {
    if (ask < c_end) {
      const int j = ask_k + KC / 4 * t;                    // the lane's first rank
      const TW* src = bp;
      uint32_t dst = slots_at + to;
#pragma unroll
      for (int u = 0; u < 2 * MT; ++u, src += hop) {
        const bool in = ask + 8 * u + g < c_end;
#pragma unroll
        for (int e = 0; e < Ring::kParts; ++e, dst += 32 * Ring::kUnit) {
          constexpr int n = Ring::kUnit / int(sizeof(TW));
          const bool ok = in && j + e * n < rank;
          const TW* at = ok ? src + e * n : b;
          if (Ring::kUnit == 16 && wide) {
            cp_async16(dst, at, ok);
          } else {
            cp_async8(dst, at, ok);
            if constexpr (Ring::kUnit == 16) {
              const bool second = in && j + e * n + n / 2 < rank;
              cp_async8(dst + 8, second ? src + e * n + n / 2 : b, second);
            }
          }
        }
      }
      ask_k += KC;
      bp += KC;
      if (ask_k >= rank) { bp += size_t(kStep) * rank - ask_k; ask_k = 0; ask += kStep; }
    }
    cp_async_commit();                                     // a group per stage, also an empty one
    to = to == (kStages - 1) * Ring::kStage ? 0 : to + Ring::kStage;
  };
  // VEC: two or four columns per lane; four of fp32 rows cost the loop of 64 columns registers for the addresses of two rows, and
  // it spilled (3B head with rows of 50280: 48 us, 32 with two)
  constexpr int W = !VEC ? 1 : COLS == 64 && sizeof(TY) == 4 ? 2 : 4, kLanes = COLS / W < 32 ? COLS / W : 32, kAtOnce = 32 / kLanes;
  constexpr int kPasses = 8 * NT / kAtOnce, kQ = COLS / (kLanes * W);
  // y of the next columns is requested as this one's sums go out, where a stage is 16 ranks (3B head 42 -> 40 us, with 3 stages of B
  // 33); with 32 ranks its registers are wanted for B (7B key, value and receptance, 256 streams, h in two pieces: 66 us so, 71 ahead)
  constexpr bool kAhead = KC == 16;
  const int my_row = lane / kLanes, my_col = lane % kLanes * W;
  AdaptFew<TY, W> line[kPasses][kQ];
  auto load_y = [&](int i, int c) {                        // pass i of the columns from c
    const int r = i * kAtOnce + my_row;
    const TY* p = y + row_at[r] + c + my_col;
#pragma unroll
    for (int q = 0; q < kQ; ++q)
      if (r < count && c + q * 32 + my_col < c_end) line[i][q].load(p + q * 32);
  };
  // weights and y: no part of what the first launch writes
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) request();
  if constexpr (kAhead) {
#pragma unroll
    for (int i = 0; i < kPasses; ++i)
      if (i * kAtOnce < count) load_y(i, c0);
  }
  stage_h();
  const char* from = slots;
  for (; c0 < c_end; c0 += kStep) {
    if constexpr (!kAhead) {
#pragma unroll
      for (int i = 0; i < kPasses; ++i)
        if (i * kAtOnce < count) load_y(i, c0);
    }
    for (int k0 = 0; k0 < rank; k0 += KC) {
      request();
      cp_async_wait<kStages - 1>();
      AdaptRaw<TW, KC / 4> raw[MT][2];
#pragma unroll
      for (int u = 0; u < 2 * MT; ++u)
#pragma unroll
        for (int e = 0; e < Ring::kParts; ++e) {
          const char* at = from + (u * Ring::kParts + e) * 32 * Ring::kUnit + lane * Ring::kUnit;
          uint32_t* w = raw[u >> 1][u & 1].w;
          if constexpr (Ring::kUnit == 16) {
            const uint4 v = *reinterpret_cast<const uint4*>(at);
            w[4 * e] = v.x; w[4 * e + 1] = v.y; w[4 * e + 2] = v.z; w[4 * e + 3] = v.w;
          } else {
            const uint2 v = *reinterpret_cast<const uint2*>(at);
            w[0] = v.x; w[1] = v.y;
          }
        }
      from = from == slots + (kStages - 1) * Ring::kStage ? slots : from + Ring::kStage;
      // weights that need no cutting: 8 rows at a time, for the registers
      constexpr int NB = PW == 1 ? 1 : NT;
#pragma unroll
      for (int n0 = 0; n0 < NT; n0 += NB) {
        float acc[MT][NB][4];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[m][n][i] = 0.f;
        auto h_of = [&](int n, int s, int p) { return hf[(((n0 + n) * ksteps + k0 / 16 + s) * PH + p) * 32]; };
        // the small products of the stage first, while the sum is small (see the head of this file)
#pragma unroll
        for (int s = 0; s < KC / 16; ++s) {
          uint32_t fa[MT][PW][4];
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t f[PW];
              raw[m][i & 1].template pair<PW>(2 * s + (i >> 1), f);
#pragma unroll
              for (int w = 0; w < PW; ++w) fa[m][w][i] = f[w];
            }
#pragma unroll
          for (int p = PH - 1; p >= 0; --p)
#pragma unroll
            for (int n = 0; n < NB; ++n) {
              if (p == 0 && PW == 1) continue;
              const uint2 h = h_of(n, s, p);
#pragma unroll
              for (int w = PW - 1; w >= 0; --w) {
                if (p + w >= PH || p + w == 0) continue;
#pragma unroll
                for (int m = 0; m < MT; ++m) mma_bf16(acc[m][n], fa[m][w], h.x, h.y);
              }
            }
        }
#pragma unroll
        for (int s = 0; s < KC / 16; ++s) {
          uint32_t fa[MT][4];
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) fa[m][i] = raw[m][i & 1].first(2 * s + (i >> 1));
#pragma unroll
          for (int n = 0; n < NB; ++n) {
            const uint2 h = h_of(n, s, 0);
#pragma unroll
            for (int m = 0; m < MT; ++m) mma_bf16(acc[m][n], fa[m], h.x, h.y);
          }
        }
        if (k0 == 0 && n0 == 0) __syncwarp();              // the table has been read
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float* at = turn + ((n0 + n) * 8 + 2 * t + (i & 1)) * Ring::kPitch + m * 16 + (i >> 1) * 8 + g;
              *at = k0 ? *at + acc[m][n][i] : acc[m][n][i];          // stages join here, rounding
            }
      }
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      if (i * kAtOnce >= count) break;
      const int r = i * kAtOnce + my_row;
      TY* p = out + row_at[r] + c0 + my_col;
#pragma unroll
      for (int q = 0; q < kQ; ++q)
        if (r < count && c0 + q * 32 + my_col < c_end) line[i][q].add_store(p + q * 32, turn + r * Ring::kPitch + q * 32 + my_col);
      if constexpr (kAhead) load_y(i, c0 + kStep);         // in flight until the next columns' sums are there
    }
  }
  cp_async_wait<0>();
}

// out[row][c] = y[row][c] + scale * sum_j h[row][j] B[id][c][j].  Grid (tiles of up to 16 rows, column chunks of all matrices).
// Columns are the rows of the products and rows, 8 at a time, their columns, so that a tile of one row, the common one of a
// decoding step, wastes little.  A lane's fragments of B come by asynchronous copies into slots of its own, some stages ahead;
// sums are turned in the warp's table and leave in lines of a row.  h is scaled, and the sum with y rounded once to TY.
// VEC: all rows of y and out start on boundaries of four elements.
template <typename TY, typename TW, int KC, bool VEC>
__global__ void __launch_bounds__(kExpandThreads, 2) adapt_expand_kernel(const AdaptParams P) {
  using Ring = ExpandRing<TY, TW, KC>;
  extern __shared__ __align__(16) char shared[];
  __shared__ int rows[kAdaptRows];
  __shared__ size_t row_at[16];                            // where they start in y and out
  __shared__ uint32_t mask[kAdaptWindow / 32];
  const int tid = threadIdx.x, warp = tid >> 5;
  int id = -1;
  const int count = adapt_tile(P, blockIdx.x, rows, mask, &id);
  int mat = 0;
  while (mat < P.nmat - 1 && int(blockIdx.y) >= P.chunk_end[mat]) ++mat;
  const int N = P.n_out[mat], chunk = int(blockIdx.y) - (mat ? P.chunk_end[mat - 1] : 0);
  const int c_begin = chunk * P.chunk_cols, c_end = min(N, c_begin + P.chunk_cols);
  const TY* y = static_cast<const TY*>(P.y[mat]);
  TY* out = static_cast<TY*>(P.out[mat]);
  if (count == 0 || id < 0) {
    // no adapter: only a copy, where out is not y
    if (count > 0 && y != out) adapt_copy<TY, VEC>(y, out, rows, count, N, c_begin, c_end);
    // A launch in which nobody waits may end before the first one has read its ids, and what follows the call on the stream may
    // overwrite those, or the workspace.  The first CTA always leads rows: it waits, here or for h.
    if (blockIdx.x == 0 && blockIdx.y == 0) griddep_wait();
    return;
  }
  const int rank = P.rank, ksteps = (rank + KC - 1) / KC * (KC / 16);
  if (tid < 16) row_at[tid] = size_t(rows[tid < count ? tid : 0]) * N;
  __syncthreads();
  auto stage_h = [&] {
    griddep_wait();
    const float scale = P.scale[mat] ? __ldg(P.scale[mat] + id) : 1.f;
    const int r4 = ksteps * 4, padded = (count + 7) / 8 * 8;         // groups of four ranks; rows
    for (int i = tid; i < padded * r4; i += kExpandThreads) {
      const int r = i / r4, j4 = i - r * r4, j = j4 * 4;
      float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r < count && j < rank) s = __ldcg(reinterpret_cast<const float4*>(P.h[mat] + size_t(rows[r]) * rank + j));
      expand_put_h<KC>(shared, ksteps, r, j4, make_float4(s.x * scale, s.y * scale, s.z * scale, s.w * scale));
    }
    __syncthreads();
  };
  const TW* b = static_cast<const TW*>(P.b[mat]) + size_t(id) * N * rank;
  char* slots = shared + expand_h_bytes(rank, KC) + warp * Ring::kWarp;
  const int c0 = c_begin + warp * Ring::kCols;
  if (count <= 8) expand_columns<TY, TW, KC, VEC, 1>(P, b, y, out, c0, c_end, row_at, count, shared, slots, stage_h);
  else expand_columns<TY, TW, KC, VEC, 2>(P, b, y, out, c0, c_end, row_at, count, shared, slots, stage_h);
}

// Both in one launch, for calls of a few tiles, where a launch and the hand-over of h through memory are most of the time: a
// cluster of eight CTAs per tile and matrix, each with an eighth of K, then of the columns; h meets in shared memory.
constexpr int kFusedCtas = 8;
static_assert(kFusedCtas <= kAdaptMaxSplits, "");

template <typename T, typename TW, int MT>
struct FusedShape {
  static constexpr int KC = MT == 1 ? 16 : 32, kH = expand_h_bytes(16 * MT, KC), kRing = kExpandWarps * ExpandRing<T, TW, KC>::kWarp;
  static constexpr int kSmem = kH + kRing + ShrinkRing<T, TW, MT>::kSmem;
  static_assert(kSmem <= 226 * 1024, "");
};

template <typename T, typename TW, int MT, bool VEC>
__global__ void __launch_bounds__(kExpandThreads, 1) adapt_fused_kernel(const AdaptParams P) {
  using F = FusedShape<T, TW, MT>;
  constexpr int KC = F::KC, RC = 16 * MT, kCols = ExpandRing<T, TW, KC>::kCols;
  namespace cg = cooperative_groups;
  const cg::cluster_group cluster = cg::this_cluster();
  extern __shared__ __align__(16) char shared[];
  __shared__ int rows[kAdaptRows];
  __shared__ size_t row_at[16];
  __shared__ uint32_t mask[kAdaptWindow / 32];
  const int tid = threadIdx.x, warp = tid >> 5, tile = blockIdx.x / kFusedCtas, part = blockIdx.x - tile * kFusedCtas, mat = blockIdx.y;
  int id = -1;
  const int count = adapt_tile(P, tile, rows, mask, &id), N = P.n_out[mat], rank = P.rank;
  const int per = (N + kFusedCtas * kCols - 1) / (kFusedCtas * kCols) * kCols, c_begin = part * per, c_end = min(N, c_begin + per);
  const T* y = static_cast<const T*>(P.y[mat]);
  T* out = static_cast<T*>(P.out[mat]);
  if (count == 0) return;                                  // the whole cluster, here and below
  if (id < 0) {
    if (y != out && c_begin < c_end) adapt_copy<T, VEC>(y, out, rows, count, N, c_begin, c_end);
    return;
  }
  if (tid < 16) row_at[tid] = size_t(rows[tid < count ? tid : 0]) * N;
  __syncthreads();
  const int ksteps = (rank + KC - 1) / KC * (KC / 16);
  char *slots = shared + F::kH + warp * ExpandRing<T, TW, KC>::kWarp, *work = shared + F::kH + F::kRing;
  const T* x = static_cast<const T*>(P.x[mat]);
  const TW* a = static_cast<const TW*>(P.a[mat]) + size_t(id) * rank * P.K;
  auto stage_h = [&] {
    float* sums = count <= 8 ? shrink_sums<T, TW, MT, 1>(P, x, a, part, 0, rows, count, work)
                             : shrink_sums<T, TW, MT, 2>(P, x, a, part, 0, rows, count, work);
    cluster.sync();
    const float scale = P.scale[mat] ? __ldg(P.scale[mat] + id) : 1.f;
    const int r4 = ksteps * 4, padded = (count + 7) / 8 * 8;         // groups of four ranks; rows
    for (int i = tid; i < padded * r4; i += kExpandThreads) {
      const int r = i / r4, j4 = i - r * r4;
      float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r < count && j4 * 4 < rank) {
        float4 v[kFusedCtas];
#pragma unroll
        for (int c = 0; c < kFusedCtas; ++c) v[c] = *reinterpret_cast<const float4*>(cluster.map_shared_rank(sums + r * RC + j4 * 4, c));
        s = v[0];
#pragma unroll
        for (int c = 1; c < kFusedCtas; ++c) { s.x += v[c].x; s.y += v[c].y; s.z += v[c].z; s.w += v[c].w; }
      }
      expand_put_h<KC>(shared, ksteps, r, j4, make_float4(s.x * scale, s.y * scale, s.z * scale, s.w * scale));
    }
    cluster.sync();                                        // the tables are read before their CTAs go on or leave
  };
  const TW* b = static_cast<const TW*>(P.b[mat]) + size_t(id) * N * rank;
  const int c0 = c_begin + warp * kCols;
  if (count <= 8) expand_columns<T, TW, KC, VEC, 1>(P, b, y, out, c0, c_end, row_at, count, shared, slots, stage_h);
  else expand_columns<T, TW, KC, VEC, 2>(P, b, y, out, c0, c_end, row_at, count, shared, slots, stage_h);
}

}  // namespace b200
