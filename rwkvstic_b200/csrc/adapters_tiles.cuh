// The two launches of adapters.cuh for streams of many rows, on the 5th-generation tensor cores: tiles of 128 rows of one
// stream, whose adapter is read once per tile.
//
// The operands are the same bfloat16 pieces (or values of one 16-bit type), cut by the threads that bring them and laid out
// in shared memory as the MMAs want them: rows of 64 elements, 128-byte swizzle.  At rank 64 and fp32 rows the pieces are
// 26 multiplications a byte, which mma.sync just about kept up with (and less under the power cap); tcgen05 leaves the
// memory as the bound.  Every wait is bounded; where one runs out the rows concerned come out as NaN and g_adapt_status says so.
#pragma once

#include "adapters.cuh"
#include "dense_gemm.cuh"

namespace b200 {

constexpr int kAdaptTile = 128;            // rows of a tile; columns of a step of the second launch
constexpr int kTileBytes = kAdaptTile * 128;         // 128 rows of 64 elements
constexpr int kTileRankMax = 128;          // of the second launch: two times 64 ranks

// Status bits of expired waits, kept per GPU: a call's workspace is the caller's and holds nothing between calls.
static __device__ int g_adapt_status;

__device__ __forceinline__ void fence_smem_to_mma() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
template <int COLS>
__device__ __forceinline__ void tmem_alloc_cols(uint32_t slot) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "n"(COLS) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
template <int COLS>
__device__ __forceinline__ void tmem_free_cols(uint32_t tmem) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(COLS) : "memory");
}
// 16 consecutive columns of this warp's 32 lanes.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]),
        "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
      : "r"(taddr)
      : "memory");
}
// Where unit `u` (16 bytes) of a row lies in a tile of 128-byte rows.
__device__ __forceinline__ int tile_unit(int row, int u) { return row * 128 + ((u ^ (row & 7)) << 4); }

// Barriers and flags at the front of dynamic shared memory (1024 bytes, so that the tiles behind are aligned).
struct TileControl {
  uint64_t full[8], empty[8], acc_full[2], acc_empty[2];
  int abort;
  uint32_t tmem;
};

// ---------------------------------------------------------------------------------------------- the first launch
// h[row][j] = sum_k x[row][k] A[id][j][k] for 128 rows (the MMAs' M, a TMEM lane each) and up to 64 ranks (their N).  Eight
// warps, or sixteen where they cut pieces (3B ffn, 8192 rows of fp32 50 us with eight, 47 with sixteen; 3B value, 1402 rows of
// fp16 14 and 15), bring 64 k of x and A at a time; one warp issues the MMAs.  x comes by asynchronous copies some stages ahead:
// into the MMAs' own tiles where both operands are of one 16-bit type, else into slots of the thread that asked, which cuts it
// into pieces.  (Loads into registers were bound by the few L1 lines that are left beside this much shared memory: 3B ffn, 8192
// rows 62 us.)  A stage (two, 128 k, where nothing is cut) makes a sum, which those warps add up in registers, rounding, while the
// next one is formed in the other half of the TMEM columns.
// What bounds it: with pieces, shared memory (a stage's 32 KB of x pass it five times), 3.4 TB/s from memory.
constexpr int kShrinkTileRanks = 64;

template <typename TX, typename TW>
struct ShrinkTile {
  static constexpr bool kSame = std::is_same<TX, TW>::value && sizeof(TX) == 2;
  static constexpr int PX = kSame ? 1 : AdaptType<TX>::kPieces, PW = kSame ? 1 : AdaptType<TW>::kPieces;
  static constexpr int kWorkers = kSame ? 256 : 512, kThreads = kWorkers + 32;
  static constexpr int kSums = kShrinkTileRanks / (kWorkers / 128);        // ranks whose sums a thread has, of one row
  static_assert(kSums % 16 == 0, "");
  static constexpr int kBytesX = PX * kTileBytes, kStage = kBytesX + PW * kTileBytes / 2;
  static constexpr int kChain = kSame ? 2 : 1;             // stages whose sum the tensor cores form
  static constexpr int kStages = kSame ? 8 : 2, kRaw = kSame ? 0 : 64 * kAdaptTile * int(sizeof(TX));
  static constexpr int kFit = kSame ? 0 : (226 * 1024 - 1024 - 2 * kStage) / kRaw;
  static constexpr int kRing = kFit > 4 ? 4 : kFit;        // stages of x as it comes
  static constexpr int kPitch = kShrinkTileRanks + 1, kTable = kAdaptTile * kPitch * 4;
  static constexpr int kSmem = 1024 + (kStages * kStage + kRing * kRaw > kTable ? kStages * kStage + kRing * kRaw : kTable);
  // loads of a thread: 16 bytes each
  static constexpr int kUnitX = 16 / int(sizeof(TX)), kRowX = 64 / kUnitX, kHopX = kWorkers / kRowX, kLoadX = kAdaptTile / kHopX;
  static constexpr int kUnitW = 16 / int(sizeof(TW)), kRowW = 64 / kUnitW, kHopW = kWorkers / kRowW, kLoadW = kShrinkTileRanks / kHopW;
};

// One 16-byte load of T as P pieces into tiles `hop` bytes apart: eight elements are a unit, four (fp32) half of one.
template <typename T, int P>
__device__ __forceinline__ void tile_put(char* tile, int hop, int row, int load, uint4 v) {
  if constexpr (P == 1) {
    *reinterpret_cast<uint4*>(tile + tile_unit(row, load)) = v;
  } else if constexpr (sizeof(T) == 4) {
    uint32_t a[P], b[P];
    split_pair<P>(__uint_as_float(v.x), __uint_as_float(v.y), a);
    split_pair<P>(__uint_as_float(v.z), __uint_as_float(v.w), b);
#pragma unroll
    for (int p = 0; p < P; ++p) *reinterpret_cast<uint2*>(tile + p * hop + tile_unit(row, load >> 1) + (load & 1) * 8) = make_uint2(a[p], b[p]);
  } else {
    uint32_t f[4][P];
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      split_pair<P>(x.x, x.y, f[i]);
    }
#pragma unroll
    for (int p = 0; p < P; ++p) *reinterpret_cast<uint4*>(tile + p * hop + tile_unit(row, load)) = make_uint4(f[0][p], f[1][p], f[2][p], f[3][p]);
  }
}

template <typename TX, typename TW>
__global__ void __launch_bounds__(ShrinkTile<TX, TW>::kThreads, 1) adapt_shrink_tile_kernel(const AdaptParams P) {
  using S = ShrinkTile<TX, TW>;
  extern __shared__ __align__(1024) char shared[];
  TileControl& C = *reinterpret_cast<TileControl*>(shared);
  char* stages = shared + 1024;
  const int tid = threadIdx.x, warp = warp_index(), lane = tid & 31;
  const int tile = blockIdx.x / P.splits, split = blockIdx.x - tile * P.splits, mat = blockIdx.z;
  const int per = (P.T + kAdaptTile - 1) / kAdaptTile, s = tile / per, first = (tile - s * per) * kAdaptTile;
  const int count = min(kAdaptTile, P.T - first), row0 = s * P.T + first, K = P.K, rank = P.rank;
  const long long asked = __ldg(P.ids + s);
  if (asked < 0 || asked >= P.adapters) return;            // the whole cluster
  const int j0 = blockIdx.y * kShrinkTileRanks, ranks = min(kShrinkTileRanks, rank - j0), n16 = (ranks + 15) / 16 * 16;
  const int chunks = (K + 63) / 64, c0 = int((long long)chunks * split / P.splits), c1 = int((long long)chunks * (split + 1) / P.splits);
  const uint32_t full = smem_u32(C.full), empty = smem_u32(C.empty), acc_full = smem_u32(C.acc_full), acc_empty = smem_u32(C.acc_empty);
  volatile int* abort_flag = &C.abort;
  if (tid == 0) {
    for (int i = 0; i < S::kStages; ++i) { mbar_init(full + 8 * i, S::kWorkers); mbar_init(empty + 8 * i, 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(acc_full + 8 * i, 1); mbar_init(acc_empty + 8 * i, S::kWorkers / 32); }
    C.abort = 0;
    fence_mbar_init();
  }
  if (warp == S::kWorkers / 32) tmem_alloc_cols<128>(smem_u32(&C.tmem));
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, C.tmem, 0);
  griddep_launch_dependents();                             // only now: the second launch takes tensor memory too
  constexpr int kSums = S::kSums;
  float sum[kSums];
#pragma unroll
  for (int i = 0; i < kSums; ++i) sum[i] = 0.f;
  const int q = warp & 3, r0 = (warp >> 2) * kSums;        // workers: TMEM lanes 32 q .., ranks r0 ..
  if (warp < S::kWorkers / 32) {
    const TX* x = static_cast<const TX*>(P.x[mat]) + size_t(row0) * K;
    const TW* a = static_cast<const TW*>(P.a[mat]) + (size_t(asked) * rank + j0) * K;
    const int ux = tid % S::kRowX, rx = tid / S::kRowX, uw = tid % S::kRowW, rw = tid / S::kRowW;
    uint4 vw[S::kLoadW];
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
    auto load_w = [&](int c) {
      const int k = c * 64 + uw * S::kUnitW;
#pragma unroll
      for (int i = 0; i < S::kLoadW; ++i) {
        const int r = rw + i * S::kHopW;
        vw[i] = r < ranks && k < K ? __ldg(reinterpret_cast<const uint4*>(a + size_t(r) * K + k)) : zero;
      }
    };
    // 16-byte units of x (and of A where nothing is cut) to `at(i)`; past the end of rows, ranks or k zeros
    char* raw = stages + S::kStages * S::kStage + tid * 16;
    auto request = [&](int c, int slot) {
      if (c < c1) {
        const int k = c * 64 + ux * S::kUnitX;
        char* to = stages + slot * S::kStage;
#pragma unroll
        for (int i = 0; i < S::kLoadX; ++i) {
          const int r = rx + i * S::kHopX;
          const bool in = r < count && k < K;
          cp_async16(smem_u32(S::kSame ? to + tile_unit(r, ux) : raw + slot * S::kRaw + i * S::kWorkers * 16), in ? x + size_t(r) * K + k : x, in);
        }
        if constexpr (S::kSame) {
          const int kw = c * 64 + uw * S::kUnitW;
#pragma unroll
          for (int i = 0; i < S::kLoadW; ++i) {
            const int r = rw + i * S::kHopW;
            const bool in = r < ranks && kw < K;
            cp_async16(smem_u32(to + S::kBytesX + tile_unit(r, uw)), in ? a + size_t(r) * K + kw : a, in);
          }
        }
      }
      cp_async_commit();                                   // a group per stage, also an empty one
    };
    bool ok = true;
    auto flush = [&](int g) {                              // the sum of stages kChain g .. kChain g + kChain - 1
      ok = ok && __all_sync(0xffffffffu, mbar_wait_bounded(acc_full + 8 * (g & 1), uint32_t(g >> 1) & 1u, abort_flag));
      if (!ok) return;
      tc_fence_after();
      float v[kSums / 16][16];
#pragma unroll
      for (int i = 0; i < kSums / 16; ++i)
        if (r0 + 16 * i < n16) tmem_ld16(tmem + (uint32_t(q * 32) << 16) + uint32_t((g & 1) * 64 + r0 + 16 * i), v[i]);
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < kSums; ++i)
        if (r0 + (i & ~15) < n16) sum[i] += v[i >> 4][i & 15];
      tc_fence_before();
      if (lane == 0) mbar_arrive(acc_empty + 8 * (g & 1));
    };
    int slot = 0;                                          // of the MMAs' stages
    uint32_t phase = 0;
    // stages ahead: the tiles' own are free again two MMAs later, the slots of x at once
    constexpr int kAhead = S::kSame ? S::kStages - 2 : S::kRing;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) request(c0 + i, i);
    int ask = S::kSame ? kAhead : 0;                       // slot of the next request
    if constexpr (!S::kSame) load_w(c0);
    for (int c = c0; c < c1 && ok; ++c) {
      const int n0 = c - c0;
      if constexpr (S::kSame) {
        if (c + kAhead < c1 && n0 + kAhead >= S::kStages)  // chunk n0 + kAhead takes the stage of n0 + kAhead - kStages = n0 - 2
          ok = __all_sync(0xffffffffu, mbar_wait_bounded(empty + 8 * ask, uint32_t((n0 + kAhead) / S::kStages - 1) & 1u, abort_flag));
        if (!ok) break;
        request(c + kAhead, ask);
        if (++ask == S::kStages) ask = 0;
        cp_async_wait<kAhead>();
      } else {
        cp_async_wait<kAhead - 1>();
        ok = __all_sync(0xffffffffu, mbar_wait_bounded(empty + 8 * slot, phase ^ 1u, abort_flag));
        if (!ok) break;
        char* to = stages + slot * S::kStage;
#pragma unroll
        for (int i = 0; i < S::kLoadX; ++i)
          tile_put<TX, S::PX>(to, kTileBytes, rx + i * S::kHopX, ux, *reinterpret_cast<const uint4*>(raw + ask * S::kRaw + i * S::kWorkers * 16));
#pragma unroll
        for (int i = 0; i < S::kLoadW; ++i) tile_put<TW, S::PW>(to + S::kBytesX, kTileBytes / 2, rw + i * S::kHopW, uw, vw[i]);
        if (c + 1 < c1) load_w(c + 1);
        request(c + kAhead, ask);                          // over what this thread has just read
        if (++ask == S::kRing) ask = 0;
      }
      fence_smem_to_mma();
      mbar_arrive(full + 8 * slot);
      if (++slot == S::kStages) { slot = 0; phase ^= 1u; }
      const int n = c - c0;
      if (n >= S::kChain && n % S::kChain == 0) flush(n / S::kChain - 1);
    }
    if (ok) flush((c1 - c0 + S::kChain - 1) / S::kChain - 1);        // the others have been
    cp_async_wait<0>();
    if (!ok)
#pragma unroll
      for (int i = 0; i < kSums; ++i) sum[i] = NAN;
  } else {
    const uint32_t idesc = umma_idesc_f16(kAdaptTile, n16, !(S::kSame && std::is_same<TX, __half>::value));
    const uint32_t base = smem_u32(stages);
    int slot = 0;
    uint32_t phase = 0;
    for (int c = c0; c < c1; ++c) {
      const int n = c - c0, g = n / S::kChain;
      const bool starts = n % S::kChain == 0, ends = n % S::kChain == S::kChain - 1 || c + 1 == c1;
      if (starts && !warp_wait(acc_empty + 8 * (g & 1), (uint32_t(g >> 1) & 1u) ^ 1u, abort_flag, nullptr, 0)) break;
      if (!warp_wait(full + 8 * slot, phase, abort_flag, nullptr, 0)) break;
      if (elect_one()) {
        tc_fence_after();
        const uint32_t at = base + slot * S::kStage, d = tmem + uint32_t((g & 1) * 64);
        uint32_t more = !starts;
#pragma unroll
        for (int i = S::PW - 1; i >= 0; --i)
#pragma unroll
          for (int j = S::PX - 1; j >= 0; --j) {
            if (i + j >= 3) continue;
            const uint64_t ad = umma_desc(at + j * kTileBytes), bd = umma_desc(at + S::kBytesX + i * (kTileBytes / 2));
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              umma_f16<false>(d, ad + uint64_t(2 * k), bd + uint64_t(2 * k), idesc, more);
              more = 1u;
            }
          }
        umma_commit<false>(empty + 8 * slot);
        if (ends) umma_commit<false>(acc_full + 8 * (g & 1));
      }
      __syncwarp();
      if (++slot == S::kStages) { slot = 0; phase ^= 1u; }
    }
  }
  // every MMA is over (the workers saw the last sum) and no copy on its way: the stages become the table of sums
  float* table = reinterpret_cast<float*>(stages);
  if (warp < S::kWorkers / 32) {
    float* mine = table + (q * 32 + lane) * S::kPitch + r0;
#pragma unroll
    for (int i = 0; i < kSums; ++i) mine[i] = sum[i];
  }
  tc_fence_before();
  float* h = P.h[mat] + size_t(row0) * rank + j0;
  shrink_join(P, table, count * kShrinkTileRanks, [&](int i) { return i / kShrinkTileRanks * S::kPitch + i % kShrinkTileRanks; },
              [&](int i, float v) {
                const int r = i / kShrinkTileRanks, j = i % kShrinkTileRanks;
                if (j < ranks) h[size_t(r) * rank + j] = v;
              });
  if (tid == 0 && *abort_flag) atomicOr(&g_adapt_status, B200RWKV_STATUS_WAIT_FULL);
  if (warp == S::kWorkers / 32) {
    tc_fence_after();
    tmem_free_cols<128>(tmem);
  }
}

// ---------------------------------------------------------------------------------------------- the second launch
// out[row][c] = y[row][c] + scale * sum_j h[row][j] B[id][c][j] for tiles of 128 rows (the MMAs' N) and 128 columns a step (their M,
// a TMEM lane each).  One persistent CTA per SM takes an equal share of all steps of all tiles and matrices, in order; a
// segment is what it has of one tile and matrix, whose pieces of h it lays out once.
//   warps 0..3   bring B and cut it into pieces, a step at a time
//   warps 4..19  add: a warp has 32 columns (lanes) and 16 rows of a half step
//   warp 20      issues the MMAs; two accumulators
//   warp 21      requests y, 64 rows x 128 columns a half step, in TMA boxes of 16 rows, up to four half steps ahead
// Sums are added in place in shared memory, with the lanes along a row, and leave in the same boxes (as bulk copies of single
// rows, 512 bytes each, both ways took 215 us for 8192 rows of a 3B ffn).  What bounds it is memory: 128
// bytes per 16 values pass the SM.  The same tiles with y through registers were bound by the L1 lines that loads in flight
// occupy beside 226 KB of shared memory (3B ffn, 8192 rows: 190 us for 839 MB), mma.sync by its own rate under the power cap.
// A tile without an adapter goes through unchanged, or is left out where out is y.
constexpr int kExpandTileLoaders = 128, kExpandTileAdders = 512, kExpandTileThreads = kExpandTileLoaders + kExpandTileAdders + 64;
constexpr int kExpandTileRing = 4, kExpandHalf = 64;       // half steps of y in shared memory, at most; rows of one

struct ExpandTileControl {
  uint64_t full[4], empty[4], acc_full[2], acc_empty[2], h_full, y_full[kExpandTileRing], y_empty[kExpandTileRing];
  int abort;
  uint32_t tmem;
};

template <typename TY, typename TW>
struct ExpandTile {
  static constexpr int PH = kPiecesH, PW = AdaptType<TW>::kPieces;
  static constexpr int kRow = kAdaptTile * int(sizeof(TY)), kHalfBytes = kExpandHalf * kRow;
  // for `halves` times 64 ranks: half steps of y (2 to 4) that leave room for a stage of B beside h, 0 where none do; then stages
  // of B, at most 4
  __host__ __device__ static constexpr int room(int halves, int ring) { return 226 * 1024 - 1024 - ring * kHalfBytes - PH * halves * kTileBytes; }
  __host__ __device__ static constexpr int ring(int halves) {
    for (int n = kExpandTileRing; n >= 2; --n)
      if (room(halves, n) >= PW * halves * kTileBytes) return n;
    return 0;
  }
  __host__ __device__ static constexpr int stages(int halves) {
    const int n = ring(halves) ? room(halves, ring(halves)) / (PW * halves * kTileBytes) : 0;
    return n > 4 ? 4 : n;
  }
  __host__ __device__ static constexpr int smem(int halves) { return 1024 + ring(halves) * kHalfBytes + (PH + stages(halves) * PW) * halves * kTileBytes; }
};

// A CTA's share of the steps, segment by segment.
struct ExpandSegment {
  int tile, mat, step, steps;              // columns [step, step + steps) * 128 of a matrix for a tile
  int row0, count, id;                     // id -1: none
};
struct ExpandWalk {
  const AdaptParams& P;
  int per, per_tile, at, end;
  __device__ __forceinline__ explicit ExpandWalk(const AdaptParams& P_) : P(P_) {
    per = (P.T + kAdaptTile - 1) / kAdaptTile;
    per_tile = P.chunk_end[P.nmat - 1];                    // steps of all matrices
    const long long all = (long long)P.streams * per * per_tile;
    at = int(all * blockIdx.x / gridDim.x); end = int(all * (blockIdx.x + 1) / gridDim.x);
  }
  __device__ __forceinline__ bool next(ExpandSegment& S) {
    if (at >= end) return false;
    S.tile = at / per_tile;
    const int in_tile = at - S.tile * per_tile;
    S.mat = 0;
    while (S.mat < P.nmat - 1 && in_tile >= P.chunk_end[S.mat]) ++S.mat;
    S.step = in_tile - (S.mat ? P.chunk_end[S.mat - 1] : 0);
    S.steps = min(P.chunk_end[S.mat] - in_tile, end - at);
    at += S.steps;
    const int stream = S.tile / per, first = (S.tile - stream * per) * kAdaptTile;
    S.count = min(kAdaptTile, P.T - first);
    S.row0 = stream * P.T + first;
    const long long v = __ldg(P.ids + stream);
    S.id = v >= 0 && v < P.adapters ? int(v) : -1;
    return true;
  }
  // left out altogether: in place and without an adapter
  __device__ __forceinline__ bool skipped(const ExpandSegment& S) const { return S.id < 0 && P.y[S.mat] == P.out[S.mat]; }
};

// y and out of every matrix as [rows][N], boxes of 16 rows x 128 columns.
struct AdaptMaps {
  CUtensorMap y[kAdaptMaxMats], out[kAdaptMaxMats];
};
constexpr int kExpandBox = 16;
__device__ __forceinline__ void tma_load_rows(uint32_t dst, const CUtensorMap* map, int col, int row, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
               "l"(map), "r"(col), "r"(row), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void tma_store_rows(const CUtensorMap* map, int col, int row, uint32_t src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(col), "r"(row), "r"(src) : "memory");
}
__device__ __forceinline__ void bulk_s2g(void* dst, uint32_t src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

template <typename TY, typename TW>
__global__ void __launch_bounds__(kExpandTileThreads, 1) adapt_expand_tile_kernel(const __grid_constant__ AdaptParams P,
                                                                                const __grid_constant__ AdaptMaps M) {
  using E = ExpandTile<TY, TW>;
  constexpr int PH = E::PH, PW = E::PW;
  extern __shared__ __align__(1024) char shared[];
  ExpandTileControl& C = *reinterpret_cast<ExpandTileControl*>(shared);
  const int tid = threadIdx.x, warp = warp_index(), lane = tid & 31;
  const int rank = P.rank, ksteps = (rank + 15) / 16, halves = (rank + 63) / 64, NS = P.stages, NR = P.ring;
  const int h_piece = halves * kTileBytes, stage_bytes = PW * h_piece;
  char *ring = shared + 1024, *h_tiles = ring + NR * E::kHalfBytes, *stages = h_tiles + PH * h_piece;
  const uint32_t full = smem_u32(C.full), empty = smem_u32(C.empty), acc_full = smem_u32(C.acc_full), acc_empty = smem_u32(C.acc_empty);
  const uint32_t h_full = smem_u32(&C.h_full), y_full = smem_u32(C.y_full), y_empty = smem_u32(C.y_empty);
  volatile int* abort_flag = &C.abort;
  constexpr int kAddWarps = kExpandTileAdders / 32, kAdd0 = kExpandTileLoaders / 32, kMmaWarp = kAdd0 + kAddWarps;
  if (tid == 0) {
    for (int i = 0; i < NS; ++i) { mbar_init(full + 8 * i, kExpandTileLoaders); mbar_init(empty + 8 * i, 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(acc_full + 8 * i, 1); mbar_init(acc_empty + 8 * i, kAddWarps); }
    for (int i = 0; i < NR; ++i) { mbar_init(y_full + 8 * i, 1); mbar_init(y_empty + 8 * i, kAddWarps); }
    mbar_init(h_full, kExpandTileAdders);
    C.abort = 0;
    fence_mbar_init();
  }
  if (warp == kMmaWarp) tmem_alloc_cols<256>(smem_u32(&C.tmem));
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, C.tmem, 0);
  ExpandWalk walk(P);
  ExpandSegment G;
  if (warp < kAdd0) {
    // ---- B: units of eight ranks of a column; neither it nor y comes from the first launch
    const int units = halves * 8, u = tid % units, hop = kExpandTileLoaders / units, j = u * 8;
    const bool wide = rank * int(sizeof(TW)) % 16 == 0, used = u < 2 * ksteps;
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
    int slot = 0;
    uint32_t phase = 0;
    bool ok = true;
    while (ok && walk.next(G)) {
      if (G.id < 0) continue;
      const int N = P.n_out[G.mat];
      const TW* b = static_cast<const TW*>(P.b[G.mat]) + size_t(G.id) * N * rank + j;
      for (int it = 0; it < G.steps; ++it) {
        ok = __all_sync(0xffffffffu, mbar_wait_bounded(empty + 8 * slot, phase ^ 1u, abort_flag));
        if (!ok) break;
        char* to = stages + slot * stage_bytes + (u >> 3) * kTileBytes;
        const int c0 = (G.step + it) * kAdaptTile;
        if (used)
          for (int c = tid / units; c < kAdaptTile; c += 4 * hop) {
            uint4 v[4][sizeof(TW) / 2];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const TW* src = b + size_t(c0 + c + i * hop) * rank;
              const bool in = c + i * hop < kAdaptTile && c0 + c + i * hop < N;
              if constexpr (sizeof(TW) == 4) {
                v[i][0] = in && j < rank ? __ldg(reinterpret_cast<const uint4*>(src)) : zero;
                v[i][1] = in && j + 4 < rank ? __ldg(reinterpret_cast<const uint4*>(src) + 1) : zero;
              } else if (wide) {
                v[i][0] = in && j < rank ? __ldg(reinterpret_cast<const uint4*>(src)) : zero;
              } else {
                const uint2 lo = in && j < rank ? __ldg(reinterpret_cast<const uint2*>(src)) : make_uint2(0u, 0u);
                const uint2 hi = in && j + 4 < rank ? __ldg(reinterpret_cast<const uint2*>(src) + 1) : make_uint2(0u, 0u);
                v[i][0] = make_uint4(lo.x, lo.y, hi.x, hi.y);
              }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (c + i * hop < kAdaptTile) {
                if constexpr (sizeof(TW) == 4) {
                  tile_put<TW, PW>(to, h_piece, c + i * hop, (u & 7) * 2, v[i][0]);
                  tile_put<TW, PW>(to, h_piece, c + i * hop, (u & 7) * 2 + 1, v[i][1]);
                } else {
                  tile_put<TW, PW>(to, h_piece, c + i * hop, u & 7, v[i][0]);
                }
              }
          }
        fence_smem_to_mma();
        mbar_arrive(full + 8 * slot);
        if (++slot == NS) { slot = 0; phase ^= 1u; }
      }
    }
  } else if (warp < kMmaWarp) {
    const int w = warp - kAdd0, q = warp & 3, part = w >> 2;                  // TMEM lanes 32 q ..; rows 16 part .. of a half step
    griddep_wait();
    bool ok = true;
    int slot = 0, uses = 0, last_slot = -1;                // uses: accumulators taken so far
    uint32_t phase = 0;
    while (walk.next(G)) {
      if (walk.skipped(G)) continue;
      const int N = P.n_out[G.mat], n16 = (G.count + 15) / 16 * 16;
      if (G.id >= 0) {                                     // every MMA of the segment before is over: its sums have been read
        const float scale = P.scale[G.mat] ? __ldg(P.scale[G.mat] + G.id) : 1.f;
        const int r4 = ksteps * 4;                         // groups of four ranks
        for (int i = tid - kExpandTileLoaders; i < n16 * r4; i += kExpandTileAdders) {
          const int r = i / r4, j4 = i - r * r4, jj = j4 * 4;
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
          if (r < G.count && jj < rank) v = __ldcg(reinterpret_cast<const float4*>(P.h[G.mat] + size_t(G.row0 + r) * rank + jj));
          uint32_t lo[PH], hi[PH];
          split_pair<PH>(v.x * scale, v.y * scale, lo);
          split_pair<PH>(v.z * scale, v.w * scale, hi);
          char* at = h_tiles + (j4 >> 4) * kTileBytes + tile_unit(r, (j4 & 15) >> 1) + (j4 & 1) * 8;
#pragma unroll
          for (int p = 0; p < PH; ++p) *reinterpret_cast<uint2*>(at + p * h_piece) = make_uint2(lo[p], hi[p]);
        }
        fence_smem_to_mma();
        mbar_arrive(h_full);
      }
      TY* out = static_cast<TY*>(P.out[G.mat]);
      const int n_half = (G.count + kExpandHalf - 1) / kExpandHalf;
      for (int it = 0; it < G.steps; ++it) {
        const int c0 = (G.step + it) * kAdaptTile, bytes = min(kAdaptTile, N - c0) * int(sizeof(TY)), buf = uses & 1;
        if (G.id >= 0) {
          ok = ok && __all_sync(0xffffffffu, mbar_wait_bounded(acc_full + 8 * buf, uint32_t(uses >> 1) & 1u, abort_flag));
          tc_fence_after();
        }
        for (int hf = 0; hf < n_half; ++hf) {
          ok = ok && __all_sync(0xffffffffu, mbar_wait_bounded(y_full + 8 * slot, phase, abort_flag));
          char* half = ring + slot * E::kHalfBytes;
          const int rows = min(kExpandHalf, G.count - hf * kExpandHalf);
          const int r0 = part * 16;
          if (r0 < rows) {
            if (G.id >= 0 || !ok) {
              float d[16];
              if (ok) {
                tmem_ld16(tmem + (uint32_t(q * 32) << 16) + uint32_t(buf * kAdaptTile + hf * kExpandHalf + r0), d);
                tmem_ld_wait();
              } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) d[i] = NAN;
              }
              TY* mine = reinterpret_cast<TY*>(half + r0 * E::kRow) + q * 32 + lane;
#pragma unroll
              for (int i = 0; i < 16; ++i) d[i] += adapt_float(mine[i * kAdaptTile]);
#pragma unroll
              for (int i = 0; i < 16; ++i) adapt_store(mine + i * kAdaptTile, d[i]);
              fence_smem_to_mma();
            }
            named_bar_sync(1 + part, 128);                 // the four warps of these 16 rows
            const int row = G.row0 + hf * kExpandHalf;
            if (r0 + kExpandBox <= rows) {
              if (q == 0 && lane == 0) tma_store_rows(&M.out[G.mat], c0, row + r0, smem_u32(half + r0 * E::kRow));
            } else {                                       // the last rows of a stream, one by one
              const int r = r0 + q * 4 + lane;
              if (lane < 4 && r < rows) bulk_s2g(out + size_t(row + r) * N + c0, smem_u32(half + r * E::kRow), uint32_t(bytes));
            }
          }
          if (lane < 4) bulk_commit();
          if (hf == n_half - 1 && G.id >= 0) {             // this warp has read the accumulator
            tc_fence_before();
            if (lane == 0) mbar_arrive(acc_empty + 8 * buf);
            ++uses;
          }
          if (last_slot >= 0) {                            // the half step before has left shared memory
            if (lane < 4) bulk_wait_read<1>();
            __syncwarp();
            if (lane == 0) mbar_arrive(y_empty + 8 * last_slot);
          }
          last_slot = slot;
          if (++slot == NR) { slot = 0; phase ^= 1u; }
        }
      }
    }
    if (lane < 4) bulk_wait_all();                         // out is written when the kernel ends
  } else if (warp == kMmaWarp) {
    const uint32_t h_at = smem_u32(h_tiles), base = smem_u32(stages);
    int slot = 0, uses = 0, segs = 0;
    uint32_t phase = 0;
    bool ok = true;
    while (ok && walk.next(G)) {
      if (G.id < 0) continue;
      const uint32_t idesc = umma_idesc_f16(kAdaptTile, (G.count + 15) / 16 * 16, 1);
      ok = warp_wait(h_full, uint32_t(segs) & 1u, abort_flag, nullptr, 0);
      ++segs;
      for (int it = 0; it < G.steps && ok; ++it, ++uses) {
        const int buf = uses & 1;
        ok = warp_wait(acc_empty + 8 * buf, (uint32_t(uses >> 1) & 1u) ^ 1u, abort_flag, nullptr, 0) && warp_wait(full + 8 * slot, phase, abort_flag, nullptr, 0);
        if (!ok) break;
        if (elect_one()) {
          tc_fence_after();
          const uint32_t d = tmem + uint32_t(buf * kAdaptTile);
          uint32_t more = 0u;
#pragma unroll
          for (int p = PH - 1; p >= 0; --p)
#pragma unroll
            for (int w = PW - 1; w >= 0; --w) {            // the small products first
              if (p + w >= PH) continue;
              for (int k = 0; k < ksteps; ++k) {
                const uint32_t off = uint32_t((k >> 2) * kTileBytes + (k & 3) * 32);
                umma_f16<false>(d, umma_desc(base + slot * stage_bytes + w * h_piece + off), umma_desc(h_at + p * h_piece + off), idesc, more);
                more = 1u;
              }
            }
          umma_commit<false>(empty + 8 * slot);
          umma_commit<false>(acc_full + 8 * buf);
        }
        __syncwarp();
        if (++slot == NS) { slot = 0; phase ^= 1u; }
      }
    }
  } else {
    int slot = 0;
    uint32_t phase = 0;
    bool ok = true;
    while (ok && walk.next(G)) {
      if (walk.skipped(G)) continue;
      const int N = P.n_out[G.mat], n_half = (G.count + kExpandHalf - 1) / kExpandHalf;
      const TY* y = static_cast<const TY*>(P.y[G.mat]) + size_t(G.row0) * N;
      for (int it = 0; it < G.steps && ok; ++it) {
        const int c0 = (G.step + it) * kAdaptTile, bytes = min(kAdaptTile, N - c0) * int(sizeof(TY));
        for (int hf = 0; hf < n_half && ok; ++hf) {
          ok = warp_wait(y_empty + 8 * slot, phase ^ 1u, abort_flag, nullptr, 0);
          if (!ok) break;
          const int rows = min(kExpandHalf, G.count - hf * kExpandHalf);
          const int boxed = rows / kExpandBox * kExpandBox;          // the last rows of a stream come one by one
          if (lane == 0) mbar_arrive_expect_tx(y_full + 8 * slot, uint32_t(boxed * E::kRow + (rows - boxed) * bytes));
          __syncwarp();
          const uint32_t to = smem_u32(ring + slot * E::kHalfBytes);
          if (lane * kExpandBox < boxed)
            tma_load_rows(to + lane * kExpandBox * E::kRow, &M.y[G.mat], c0, G.row0 + hf * kExpandHalf + lane * kExpandBox, y_full + 8 * slot);
          else if (lane >= 16 && boxed + lane - 16 < rows)
            bulk_g2s(to + (boxed + lane - 16) * E::kRow, y + size_t(hf * kExpandHalf + boxed + lane - 16) * N + c0, uint32_t(bytes), y_full + 8 * slot);
          if (++slot == NR) { slot = 0; phase ^= 1u; }
        }
      }
    }
    // after an abort copies may still be on their way into shared memory
    if (*abort_flag) {
      const unsigned long long t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < kWaitLimitNs / 100) {
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && *abort_flag) atomicOr(&g_adapt_status, B200RWKV_STATUS_WAIT_FULL);
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_free_cols<256>(tmem);
  }
}

struct AdaptShape {
  bool fused;                              // one launch
  bool tiles1, tiles2;                     // the forms for 128 rows of a stream, else for gathered tiles of 16
  int n1, n2;                              // tiles that a launch has at most; CTAs of the second launch's form for tiles
  int splits, mt;                          // first launch: CTAs that share K; gathered: ranks of a CTA in 16
  int kc, chunk_cols, chunks;              // second launch: ranks per stage (gathered), columns of a CTA or step, those of all matrices
};

// SMs that clusters of one CTA per SM can take at once.  A cluster stays inside a GPC and GPCs have SMs over: 15 clusters of eight
// run together on 148 SMs, not 18 (a 16th costs a second pass: rank 16, 10240 -> 2560, 240 rows 7.3 us, 256 rows 12.8), 32 of four.
inline int cluster_room(int ctas, int sms) { return ctas >= 8 ? sms * 13 / 16 : ctas >= 4 ? sms * 7 / 8 : sms; }

// Products of pieces i and j with i + j < limit.
inline int piece_products(int a, int b, int limit) {
  int n = 0;
  for (int i = 0; i < a; ++i)
    for (int j = 0; j < b; ++j) n += i + j < limit;
  return n;
}

// Which form.  Calls whose tiles' clusters of eight all run at once, with at most 64 KB of B per CTA, take one launch (1.5B key,
// value and receptance, one row: 5.1 us against 6.2 in two; rank 16, 10240 -> 2560, 240 rows 7.3 against 10.9).
// Tiles of 128 rows are for streams of 64 rows or more, where the products are many: each launch by itself, since gathered tiles
// start sooner and tcgen05 takes products faster.  Time of gathered tiles beside that of these, 64 to 8192 rows in 1 to 8 streams,
// 768 to 10240 wide, ranks 8 to 128, all types (least, median, most):
//   first launch, by products of 16 ranks x rows x K
//     about 8M -29, -16, -4 %;  16M -18, -8, +22;  32M -7, +4, +25;  64M 0, +16, +108;  256M and more +14, +106, +148
//   second launch, by products of 16 ranks x rows x N x bytes of y
//     about 32M -23, -11, +3 %;  64M -14, -2, +15;  128M -7, +16, +41;  512M +6, +29, +84;  2000M +40, +76, +110
//     (rows of 16 bits: without the third piece of h, which costs gathered tiles less than a product: 10240 -> 2560 for 2 x 701 rows,
//     fp16, rank 32, 43M so and 72M with it: 22.6 us, 24.8 as tiles; bf16, rank 64, 57M and 86M: 27.1 and 25.5)
// Ranks up to 128 and rows that start on 16 bytes for the second (`aligned`; y passes as bulk copies), one CTA per SM.
// Splits of K: a power of two that leaves the launch one wave (of one CTA per SM for tiles, else of two), 256 or more k each.
// Columns of a CTA of the second launch, gathered: the number of steps for which the rounds of the two CTAs that an SM holds take
// the least, a start being worth a step, by the number of tiles where streams spread evenly over the adapters.  Time follows
// the rounds: 3B head for 48 x 5 rows of 20 adapters, 4 6 7 8 10 12 16 steps (2 2 2 1 1 1 1 rounds) 33.5 37.9 38.1 32.4 34.8 38.4 47
// us; 7B ffn for 64 streams of 48 adapters, 4 6 8 12 16 steps 24.6 26.6 23.1 26.9 32.
inline AdaptShape adapt_shape(int nmat, const int* n_out, int adapters, int rank, int K, int streams, int T, int w_pieces, int row_bytes, bool same16,
                              bool aligned, int sms) {
  AdaptShape s;
  auto cut = [&](int rows) { return T < rows ? streams : streams * ((T + rows - 1) / rows); };
  long long columns = 0;
  for (int i = 0; i < nmat; ++i) columns += n_out[i];
  const long long work = (long long)streams * T * ((rank + 15) / 16);
  const int shrink_products = same16 ? 1 : piece_products(row_bytes == 4 ? 3 : w_pieces, w_pieces, 3);
  const int expand_products = piece_products(row_bytes == 4 ? 3 : 2, w_pieces, row_bytes == 4 ? 3 : 2);
  s.tiles1 = T >= 64 && work * shrink_products * K * nmat >= 24000000;
  s.tiles2 = T >= 64 && work * expand_products * columns * row_bytes >= 60000000 && rank <= kTileRankMax && aligned;
  s.n1 = s.tiles1 ? streams * ((T + kAdaptTile - 1) / kAdaptTile) : cut(kAdaptRows);
  auto busy = [&](int n, bool tiled) {                   // tiles that lead rows
    const long long most = adapters + (long long)streams * T / kAdaptRows + 1;
    return !tiled && T < kAdaptRows && most < n ? most : (long long)n;
  };
  // fp16 and fp32: 32 ranks, for the registers of a lane that cuts them (also beside fp16 rows, where nothing is cut)
  s.mt = rank <= 16 ? 1 : rank <= 32 || w_pieces > 1 ? 2 : 4;
  s.kc = rank <= 16 ? 16 : 32;
  s.fused = !s.tiles1 && rank <= 16 * s.mt && (long long)s.n1 * nmat * kFusedCtas <= cluster_room(kFusedCtas, sms);
  for (int i = 0; i < nmat; ++i) s.fused = s.fused && (long long)n_out[i] * rank * (w_pieces == 3 ? 4 : 2) <= kFusedCtas * 64 * 1024;
  const int per_cta = s.tiles1 ? kShrinkTileRanks : 16 * s.mt;
  const long long ctas = busy(s.n1, s.tiles1) * nmat * ((rank + per_cta - 1) / per_cta);
  s.splits = 1;
  while (s.splits < kAdaptMaxSplits && ctas * 2 * s.splits <= (s.tiles1 ? 1LL : 2LL) * cluster_room(2 * s.splits, sms) && K >= 512 * s.splits) s.splits *= 2;
  s.chunks = 0;
  if (s.tiles2) {                                        // steps of all matrices for a tile, and CTAs
    s.chunk_cols = kAdaptTile;
    for (int i = 0; i < nmat; ++i) s.chunks += (n_out[i] + kAdaptTile - 1) / kAdaptTile;
    const long long steps = (long long)streams * ((T + kAdaptTile - 1) / kAdaptTile) * s.chunks;
    s.n2 = int(steps < sms ? steps : sms);
    return s;
  }
  s.n2 = cut(kAdaptRows);
  const int unit = kExpandWarps * (w_pieces < 3 ? 64 : 32);
  const long long shared_by = adapters < streams ? adapters : streams, filled = (long long)streams * T / kAdaptRows + shared_by / 2;
  const long long tiles = T >= kAdaptRows ? s.n2 : filled > shared_by ? filled : shared_by;        // about as many as lead rows
  long long least = 0;
  for (int per = 64; per >= 1; --per) {                  // rounds of two CTAs per SM, times units of a CTA and one for its start
    long long chunks = 0;
    for (int i = 0; i < nmat; ++i) chunks += (n_out[i] + per * unit - 1) / (per * unit);
    const long long cost = (chunks * tiles + 2 * sms - 1) / (2 * sms) * (per + 1);
    if (least && cost >= least) continue;
    least = cost;
    s.chunk_cols = per * unit;
  }
  for (int i = 0; i < nmat; ++i) s.chunks += (n_out[i] + s.chunk_cols - 1) / s.chunk_cols;
  return s;
}

}  // namespace b200
