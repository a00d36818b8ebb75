// Products of 8-bit integer matrices with a scale per token and per channel.
//
//   acc[t, n] = sum_k xq[t, k] * wq[n, k]                 (int32, exact)
//   y[t, n]   = fp32(acc) * (xs[t] * ws[n]) + bias[n]     rounded once
// and, for the gated form (wq holds the gate rows 0..N-1, then the up rows),
//   y[t, n]   = silu(g) * u  with g, u the two products of channel n.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "qcc_common.cuh"
#include "qcc_host.h"
#include "qcc_tc.cuh"

namespace qcc {
namespace {

constexpr int kMaxCols = 131071;  // |q| <= 128: the int32 sum stays below 2^31
constexpr int kMaxTokens = 1 << 20, kMaxChannels = 1 << 19;

struct Int8Args {
  const int8_t* x;
  int64_t ldx;
  const float* xs;
  const int8_t* w;
  int64_t ldw;
  const float* ws;
  const void* bias;
  int bias_dtype;
  int tokens, channels, cols;  // channels: output columns (the weight has twice as many rows when gated)
  void* y;
  int64_t ldy;
  int y_dtype;
  bool y_vec4 = false;  // y's rows take stores of four values
};

__device__ __forceinline__ float silu(float g) { return g / (1.f + expf(-g)); }

__device__ __forceinline__ float bias_value(const void* bias, int dtype, int n) {
  if (bias == nullptr) return 0.f;
  if (dtype == QCC_DTYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(bias)[n]);
  if (dtype == QCC_DTYPE_F16) return __half2float(static_cast<const __half*>(bias)[n]);
  return static_cast<const float*>(bias)[n];
}

// ---------------------------------------------------------------------------
// Stream kernel: one CTA computes 128 weight rows x BN tokens of the product
// over its share of the columns.  The weight rows are the M operand of
// tcgen05.mma kind::i8 (TMEM lanes), the tokens its N operand (TMEM columns),
// so one decoded token costs 16 columns of N, not 128 rows of M.  A cluster of
// S CTAs splits the columns; every CTA leaves its int32 partial sums in its own
// shared memory, and the cluster adds them over distributed shared memory --
// integer sums, so the split changes no bit of the result, and no workspace.
// Gated: the 128 rows are 64 gate rows and the 64 up rows of the same channels.
//
// Waits are bounded; a tile whose wait ran out is written as NaN.
// ---------------------------------------------------------------------------

constexpr int kTileRows = 128;   // TMEM lanes
constexpr int kTileCols = 128;   // bytes of K per stage (one swizzled row)
constexpr uint64_t kWaitNs = 2000000000ull;

template <int BN, int STAGES>
struct StreamSmem {
  static constexpr int kWBytes = kTileRows * kTileCols, kXBytes = BN * kTileCols;
  static constexpr int kStage = kWBytes + kXBytes;
  static constexpr int kPartial = BN * kTileRows * 4;
  static constexpr int kRing = STAGES * kStage;
  static constexpr int kBody = kRing > kPartial ? kRing : kPartial;
  static constexpr int kBytes = 1024 + kBody;  // ring aligned to 1024
};

__device__ __forceinline__ int4 cluster_load4(uint32_t smem, uint32_t rank) {
  uint32_t remote;
  int4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem), "r"(rank));
  asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(remote)
               : "memory");
  return v;
}

__device__ __forceinline__ int cluster_load1(uint32_t smem, uint32_t rank) {
  uint32_t remote;
  int v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem), "r"(rank));
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(remote) : "memory");
  return v;
}

__device__ __forceinline__ void store4(const Int8Args& a, int t, int n, const float (&v)[4]) {
  const int64_t at = static_cast<int64_t>(t) * a.ldy + n;
  if (a.y_vec4 && n + 4 <= a.channels) {
    if (a.y_dtype == QCC_DTYPE_F32) {
      *reinterpret_cast<float4*>(static_cast<float*>(a.y) + at) = make_float4(v[0], v[1], v[2], v[3]);
    } else if (a.y_dtype == QCC_DTYPE_BF16) {
      const __nv_bfloat162 lo = __floats2bfloat162_rn(v[0], v[1]), hi = __floats2bfloat162_rn(v[2], v[3]);
      *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.y) + at) =
          make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    } else {
      const __half2 lo = __floats2half2_rn(v[0], v[1]), hi = __floats2half2_rn(v[2], v[3]);
      *reinterpret_cast<uint2*>(static_cast<__half*>(a.y) + at) =
          make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (n + j < a.channels) store_as(a.y, at + j, a.y_dtype, v[j]);
}

template <bool GATED, int BN, int STAGES>
__global__ void __launch_bounds__(128) int8_stream_kernel(const Int8Args a, const __grid_constant__ CUtensorMap tm_x,
                                                          const __grid_constant__ CUtensorMap tm_w) {
  using S = StreamSmem<BN, STAGES>;
  constexpr int kChannels = GATED ? kTileRows / 2 : kTileRows;
  constexpr uint32_t kTmemCols = BN < 32 ? 32 : BN;
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t full[STAGES], empty[STAGES], done;
  __shared__ uint32_t tmem_slot;
  __shared__ int failed;
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int warp = threadIdx.x >> 5;
  uint32_t rank, splits;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(splits));
  const int n0 = static_cast<int>(blockIdx.x / splits) * kChannels, t0 = static_cast<int>(blockIdx.y) * BN;
  const int blocks = (a.cols + kTileCols - 1) / kTileCols;
  const int first = static_cast<int>(static_cast<int64_t>(blocks) * rank / splits);
  const int count = static_cast<int>(static_cast<int64_t>(blocks) * (rank + 1) / splits) - first;

  if (warp == 0) {
    if (threadIdx.x == 0) {
      tma_prefetch_map(&tm_x);
      tma_prefetch_map(&tm_w);
      for (int s = 0; s < STAGES; ++s) {
        mbar_init(&full[s], 1);
        mbar_init(&empty[s], 1);
      }
      mbar_init(&done, 1);
      failed = 0;
      fence_barrier_init();
    }
  }
  // Tensor memory is taken only once the launches ahead have finished: a CTA
  // of theirs that still waits for its own columns must not wait for ours.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (warp == 1) {
    tmem_alloc(&tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = tmem_slot;

  if (threadIdx.x == 0) {
    const uint64_t keep = policy_evict_last(), stream = policy_evict_first();
    int issued = 0;
    for (; issued < count; ++issued) {
      const int s = issued % STAGES;
      if (issued >= STAGES && !mbar_wait_bounded(&empty[s], (issued / STAGES - 1) & 1, kWaitNs)) {
        failed = 1;
        break;
      }
      uint8_t* w = ring + s * S::kStage;
      mbar_arrive_expect_tx(&full[s], S::kStage);
      const int k = (first + issued) * kTileCols;
      if (GATED) {
        tma_load_2d_hint(w, &tm_w, k, n0, &full[s], stream);
        tma_load_2d_hint(w + S::kWBytes / 2, &tm_w, k, a.channels + n0, &full[s], stream);
      } else {
        tma_load_2d_hint(w, &tm_w, k, n0, &full[s], stream);
      }
      tma_load_2d_hint(w + S::kWBytes, &tm_x, k, t0, &full[s], keep);
    }
    // A copy must not land after this CTA has gone: after a wait that ran out, see the issued ones in.
    if (issued < count)
      for (int i = issued - STAGES < 0 ? 0 : issued - STAGES; i < issued; ++i)
        mbar_wait_bounded(&full[i % STAGES], (i / STAGES) & 1, kWaitNs);
  } else if (threadIdx.x == 32) {
    constexpr uint32_t idesc = idesc_s8(kTileRows, BN);
    for (int i = 0; i < count; ++i) {
      const int s = i % STAGES;
      if (!mbar_wait_bounded(&full[s], (i / STAGES) & 1, kWaitNs)) {
        failed = 1;
        break;
      }
      tc_fence_after_sync();
      const uint32_t w = smem_addr(ring + s * S::kStage);
      const uint64_t wd = smem_desc_sw128(w, 16, 1024), xd = smem_desc_sw128(w + S::kWBytes, 16, 1024);
#pragma unroll
      for (int k = 0; k < kTileCols / 32; ++k)
        tc_mma_i8(tmem, wd + k * 2, xd + k * 2, idesc, (i | k) != 0 ? 1u : 0u);
      tc_commit(&empty[s]);
    }
    tc_commit(&done);
  }
  __syncwarp();
  if (!mbar_wait_bounded(&done, 0, 4 * kWaitNs)) failed = 1;
  tc_fence_after_sync();

  // TMEM -> this CTA's shared memory as [token][row] int32 (the ring is free: every MMA has completed).
  int* partial = reinterpret_cast<int*>(ring);
  const int tokens = min(BN, a.tokens - t0);
#pragma unroll 1
  for (int c = 0; c < tokens; c += 16) {
    float v[16];
    tmem_load16(tmem + (static_cast<uint32_t>(warp * 32) << 16) + c, v);
#pragma unroll
    for (int j = 0; j < 16; ++j) partial[(c + j) * kTileRows + threadIdx.x] = count > 0 ? __float_as_int(v[j]) : 0;
  }
  tc_fence_before_sync();
  cluster_sync();
  tc_fence_after_sync();
  if (warp == 1) tmem_dealloc(tmem, kTmemCols);

  // Sum over the cluster, scale and store: 4 channels of one token a thread at a time.
  constexpr int kVecs = kChannels / 4;
  const uint32_t base = smem_addr(partial);
  int broken = 0;
  for (uint32_t r = 0; r < splits; ++r) broken |= cluster_load1(smem_addr(&failed), r);
  for (int i = static_cast<int>(rank) * 128 + static_cast<int>(threadIdx.x); i < tokens * kVecs;
       i += 128 * static_cast<int>(splits)) {
    const int t = i / kVecs, c = i % kVecs * 4;
    int g[4] = {}, u[4] = {};
    for (uint32_t r = 0; r < splits; ++r) {
      const int4 p = cluster_load4(base + (t * kTileRows + c) * 4, r);
      g[0] += p.x, g[1] += p.y, g[2] += p.z, g[3] += p.w;
      if (GATED) {
        const int4 q = cluster_load4(base + (t * kTileRows + kChannels + c) * 4, r);
        u[0] += q.x, u[1] += q.y, u[2] += q.z, u[3] += q.w;
      }
    }
    const float xs = a.xs[t0 + t];
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = min(n0 + c + j, a.channels - 1);
      v[j] = static_cast<float>(g[j]) * (xs * a.ws[n]);
      if (GATED)
        v[j] = silu(v[j]) * (static_cast<float>(u[j]) * (xs * a.ws[a.channels + n]));
      else
        v[j] += bias_value(a.bias, a.bias_dtype, n);
      if (broken) v[j] = NAN;
    }
    store4(a, t0 + t, n0 + c, v);
  }
  cluster_sync();  // the other CTAs have read this one's sums
}

// ---------------------------------------------------------------------------
// Pair kernel: persistent CTA pairs (cta_group::2), tiles of 256 weight rows x
// up to 256 tokens over all columns, for token counts that make the product
// compute bound.  Warp 0 loads, warp 1 of the even CTA issues the MMAs, warps
// 2-5 drain the accumulators; two accumulators (2 x 256 of the 512 TMEM
// columns) let a tile's epilogue run beside the next tile's MMAs.  A pair reads
// each operand byte of its tile once (128 rows of each per CTA), half of what
// two single CTAs would.
// Gated: the rows of a tile alternate 16 gate and 16 up rows, so that lane l
// of a warp holds the gate and lane l + 16 the up product of one channel and
// one shuffle brings two tokens' pairs together.
// ---------------------------------------------------------------------------

constexpr int kPairStages = 6;
constexpr int kPairTokens = 256;                       // most tokens of a tile
constexpr int kPairStage = 2 * 128 * kTileCols;        // bytes a CTA loads per stage, at most
constexpr int kPairSmem = 1024 + kPairStages * kPairStage;
constexpr int kPairThreads = 192;

struct PairPlan {
  int row_tiles, token_tiles, tile_tokens;  // tile_tokens: multiple of 32, up to kPairTokens
  int group;                                // token tiles that are walked through together
};

// Tile i of the walk: groups of `group` token tiles, within a group the token tiles of one row tile next to each
// other, so that concurrent pairs share weight rows and a group's tokens stay in L2.
__device__ __forceinline__ void pair_tile(const PairPlan& p, int i, int& row, int& token) {
  const int per_group = p.group * p.row_tiles;
  const int g = i / per_group, in = i - g * per_group;
  const int width = min(p.group, p.token_tiles - g * p.group);
  row = in / width;
  token = g * p.group + in - row * width;
}

template <bool GATED>
__global__ void __launch_bounds__(kPairThreads, 1)
    int8_pair_kernel(const Int8Args a, const PairPlan plan, const __grid_constant__ CUtensorMap tm_x,
                     const __grid_constant__ CUtensorMap tm_w) {
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t full[kPairStages], empty[kPairStages], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int failed;
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t rank;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int tiles = plan.row_tiles * plan.token_tiles;
  const int blocks = (a.cols + kTileCols - 1) / kTileCols;
  const int half_tokens = plan.tile_tokens / 2;
  constexpr int kChannels = GATED ? 128 : 256;  // output channels of a tile, half of them in each CTA

  if (threadIdx.x == 0) {
    tma_prefetch_map(&tm_x);
    tma_prefetch_map(&tm_w);
    for (int s = 0; s < kPairStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&acc_full[s], 1);
      mbar_init(&acc_empty[s], 8);  // the four epilogue warps of both CTAs
    }
    failed = 0;
    fence_barrier_init();
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");  // before tensor memory is taken, as in the stream kernel
  if (warp == 1) {
    tmem_alloc_pair(&tmem_slot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync();  // both CTAs' barriers are initialised
  tc_fence_after_sync();
  const uint32_t tmem = tmem_slot;

  if (threadIdx.x == 0) {
    const uint64_t keep = policy_evict_last();
    int n = 0;  // stage uses so far
    bool ok = true;
    for (int i = pair; i < tiles && ok; i += pairs) {
      int row, token;
      pair_tile(plan, i, row, token);
      for (int b = 0; b < blocks; ++b, ++n) {
        const int s = n % kPairStages;
        if (n >= kPairStages && !mbar_wait_bounded(&empty[s], (n / kPairStages - 1) & 1, kWaitNs)) {
          ok = false;
          break;
        }
        uint8_t* w = ring + s * kPairStage;
        const uint32_t bar = cluster_addr(&full[s], 0);
        if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * (128 + half_tokens) * kTileCols);
        const int k = b * kTileCols;
        if (GATED) {
          const int n0 = row * kChannels + static_cast<int>(rank) * 64;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            tma_load_2d_pair(w + q * 32 * kTileCols, &tm_w, k, n0 + q * 16, bar, keep);
            tma_load_2d_pair(w + (q * 32 + 16) * kTileCols, &tm_w, k, a.channels + n0 + q * 16, bar, keep);
          }
        } else {
          tma_load_2d_pair(w, &tm_w, k, row * kChannels + static_cast<int>(rank) * 128, bar, keep);
        }
        tma_load_2d_pair(w + 128 * kTileCols, &tm_x, k, token * plan.tile_tokens + static_cast<int>(rank) * half_tokens,
                         bar, keep);
      }
    }
    if (!ok) {
      failed = 1;
      // Copies in flight land before the cluster's last barrier: the even CTA's barriers count both CTAs' bytes.
      if (rank == 0)
        for (int i = max(0, n - kPairStages); i < n; ++i)
          mbar_wait_bounded(&full[i % kPairStages], (i / kPairStages) & 1, kWaitNs);
    }
  } else if (threadIdx.x == 32 && rank == 0) {
    const uint32_t idesc = idesc_s8(256, plan.tile_tokens);
    int n = 0, done = 0;
    bool ok = true;
    for (int i = pair; i < tiles && ok; i += pairs, ++done) {
      const int acc = done & 1;
      if (done >= 2 && !mbar_wait_bounded(&acc_empty[acc], (done / 2 - 1) & 1, kWaitNs)) {
        ok = false;
        break;
      }
      tc_fence_after_sync();
      for (int b = 0; b < blocks; ++b, ++n) {
        const int s = n % kPairStages;
        if (!mbar_wait_bounded(&full[s], (n / kPairStages) & 1, kWaitNs)) {
          ok = false;
          break;
        }
        tc_fence_after_sync();
        const uint32_t w = smem_addr(ring + s * kPairStage);
        const uint64_t wd = smem_desc_sw128(w, 16, 1024), xd = smem_desc_sw128(w + 128 * kTileCols, 16, 1024);
#pragma unroll
        for (int k = 0; k < kTileCols / 32; ++k)
          tc_mma_i8_pair(tmem + acc * 256, wd + k * 2, xd + k * 2, idesc, (b | k) != 0 ? 1u : 0u);
        tc_commit_pair(&empty[s]);
      }
      tc_commit_pair(&acc_full[acc]);
    }
    if (!ok) failed = 1;
  } else if (warp >= 2) {
    const int quarter = warp & 3;  // TMEM lanes 32 * quarter .. + 31
    int done = 0;
    for (int i = pair; i < tiles; i += pairs, ++done) {
      const int acc = done & 1;
      if (failed || !mbar_wait_bounded(&acc_full[acc], (done / 2) & 1, 4 * kWaitNs)) failed = 1;
      tc_fence_after_sync();
      int row, token;
      pair_tile(plan, i, row, token);
      const int t0 = token * plan.tile_tokens, tokens = min(plan.tile_tokens, a.tokens - t0);
      const int n = row * kChannels + static_cast<int>(rank) * (kChannels / 2) +
                    (GATED ? quarter * 16 + (lane & 15) : quarter * 32 + lane);
      const bool in = n < a.channels;
      const int wrow = GATED && lane >= 16 ? a.channels + n : n;
      const float ws = in ? a.ws[wrow] : 0.f;
      const float bias = !GATED && in ? bias_value(a.bias, a.bias_dtype, n) : 0.f;
      const uint32_t from = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + acc * 256;
      for (int c = 0; c < tokens; c += 32) {
        float v[32];
        tmem_load32(from + c, v);
        const float xs = c + lane < tokens ? a.xs[t0 + c + lane] : 0.f;
        if (c + 32 >= tokens) {  // the accumulator's last columns are in registers
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(cluster_addr(&acc_empty[acc], 0));
        }
#pragma unroll
        for (int j = 0; j < 32; ++j)
          v[j] = static_cast<float>(__float_as_int(v[j])) * (__shfl_sync(0xffffffffu, xs, j) * ws);
        if (GATED) {
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            // Lanes 0-15 finish token j, lanes 16-31 token j + 1.
            const float other = __shfl_xor_sync(0xffffffffu, lane < 16 ? v[j + 1] : v[j], 16);
            float h = silu(lane < 16 ? v[j] : other) * (lane < 16 ? other : v[j + 1]);
            if (failed) h = NAN;
            const int t = c + j + (lane >> 4);
            if (in && t < tokens) store_as(a.y, static_cast<int64_t>(t0 + t) * a.ldy + n, a.y_dtype, h);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            float y = v[j] + bias;
            if (failed) y = NAN;
            if (in && c + j < tokens) store_as(a.y, static_cast<int64_t>(t0 + c + j) * a.ldy + n, a.y_dtype, y);
          }
        }
      }
    }
  }
  __syncwarp();
  tc_fence_before_sync();
  cluster_sync();  // no barrier of this CTA is signalled and none of its memory read after this
  tc_fence_after_sync();
  if (warp == 1) tmem_dealloc_pair(tmem, 512);
}

PFN_cuTensorMapEncodeTiled_v12000 encode_tiled() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    cudaGetLastError();
    return static_cast<PFN_cuTensorMapEncodeTiled_v12000>(nullptr);
  }();
  return fn;
}

// int8 rows [rows, cols], ld bytes apart, read in boxes of box_rows x 128 bytes (zeros outside).
bool make_map(CUtensorMap* map, const int8_t* base, int64_t rows, int64_t cols, int64_t ld, int box_rows) {
  auto fn = encode_tiled();
  if (fn == nullptr) return false;
  const uint64_t dims[2] = {static_cast<uint64_t>(cols), static_cast<uint64_t>(rows)};
  const uint64_t strides[1] = {static_cast<uint64_t>(ld)};
  const uint32_t box[2] = {kTileCols, static_cast<uint32_t>(box_rows)}, elem[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t*>(base), dims, strides, box, elem,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool GATED, int BN, int STAGES>
int launch_stream(const Int8Args& a, int device, cudaStream_t stream) {
  using S = StreamSmem<BN, STAGES>;
  auto* kernel = int8_stream_kernel<GATED, BN, STAGES>;
  CUtensorMap tm_x, tm_w;
  const int64_t rows = GATED ? 2ll * a.channels : a.channels;
  if (!make_map(&tm_x, a.x, a.tokens, a.cols, a.ldx, BN) ||
      !make_map(&tm_w, a.w, rows, a.cols, a.ldw, GATED ? kTileRows / 2 : kTileRows))
    return QCC_ERR_UNSUPPORTED;
  if (!ensure_max_dynamic_smem(reinterpret_cast<const void*>(kernel), device)) return QCC_ERR_CUDA;
  const int channels = GATED ? kTileRows / 2 : kTileRows;
  const int tiles = (a.channels + channels - 1) / channels, token_tiles = (a.tokens + BN - 1) / BN;
  const int slots = device_info(device).num_sms * std::max(1, (225 << 10) / (S::kBytes + 2048));
  const int blocks = (a.cols + kTileCols - 1) / kTileCols;
  const int split = std::max(1, std::min({8, blocks, static_cast<int>(slots / (static_cast<int64_t>(tiles) * token_tiles))}));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(tiles * split, token_tiles);
  cfg.blockDim = dim3(128);
  cfg.dynamicSmemBytes = S::kBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = split;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cuda_ok(cudaLaunchKernelEx(&cfg, kernel, a, tm_x, tm_w)) ? QCC_OK : QCC_ERR_CUDA;
}

// The token width of a tile: the one that needs the fewest columns of MMA work in the longest-running pair.
int pair_tile_tokens(int tokens, int row_tiles, int pairs) {
  int best = kPairTokens;
  int64_t best_cost = INT64_MAX;
  for (int width = kPairTokens; width >= 128; width -= 32) {
    const int64_t tiles = static_cast<int64_t>(row_tiles) * ((tokens + width - 1) / width);
    const int64_t cost = (tiles + pairs - 1) / pairs * width;
    if (cost < best_cost) best = width, best_cost = cost;
  }
  return best;
}

template <bool GATED>
int launch_pair(const Int8Args& a, int device, cudaStream_t stream) {
  auto* kernel = int8_pair_kernel<GATED>;
  const int channels = GATED ? 128 : 256;
  const int pairs = device_info(device).num_sms / 2;
  PairPlan plan;
  plan.row_tiles = (a.channels + channels - 1) / channels;
  plan.tile_tokens = pair_tile_tokens(a.tokens, plan.row_tiles, pairs);
  plan.token_tiles = (a.tokens + plan.tile_tokens - 1) / plan.tile_tokens;
  plan.group = 8;
  CUtensorMap tm_x, tm_w;
  if (!make_map(&tm_x, a.x, a.tokens, a.cols, a.ldx, plan.tile_tokens / 2) ||
      !make_map(&tm_w, a.w, GATED ? 2ll * a.channels : a.channels, a.cols, a.ldw, GATED ? 16 : 128))
    return QCC_ERR_UNSUPPORTED;
  if (!ensure_max_dynamic_smem(reinterpret_cast<const void*>(kernel), device)) return QCC_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * static_cast<unsigned>(std::min<int64_t>(pairs, static_cast<int64_t>(plan.row_tiles) *
                                                                            plan.token_tiles)));
  cfg.blockDim = dim3(kPairThreads);
  cfg.dynamicSmemBytes = kPairSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cuda_ok(cudaLaunchKernelEx(&cfg, kernel, a, plan, tm_x, tm_w)) ? QCC_OK : QCC_ERR_CUDA;
}

template <bool GATED>
int launch(const Int8Args& a, int device, cudaStream_t stream) {
  if (a.tokens <= 16) return launch_stream<GATED, 16, 4>(a, device, stream);
  if (a.tokens <= 32) return launch_stream<GATED, 32, 4>(a, device, stream);
  if (a.tokens <= 64) return launch_stream<GATED, 64, 4>(a, device, stream);
  if (a.tokens <= 128) return launch_stream<GATED, 128, 3>(a, device, stream);
  return launch_pair<GATED>(a, device, stream);
}

int run_int8_linear(Int8Args a, bool gated, cudaStream_t stream) {
  if (!valid_dtype(a.y_dtype) || (a.bias != nullptr && !valid_dtype(a.bias_dtype))) return QCC_ERR_DTYPE;
  if (a.tokens < 0 || a.channels < 1 || a.cols < 1 || a.ldx < a.cols || a.ldw < a.cols || a.ldy < a.channels)
    return QCC_ERR_SHAPE;
  if (a.cols > kMaxCols || a.channels > kMaxChannels || a.tokens > kMaxTokens) return QCC_ERR_UNSUPPORTED;
  if (a.tokens == 0) return QCC_OK;
  if (a.x == nullptr || a.xs == nullptr || a.w == nullptr || a.ws == nullptr || a.y == nullptr)
    return QCC_ERR_INVALID_ARGUMENT;
  if (!aligned16(a.x) || !aligned16(a.w) || a.ldx % 16 != 0 || a.ldw % 16 != 0) return QCC_ERR_ALIGNMENT;
  int device = 0;
  if (!cuda_ok(cudaGetDevice(&device))) return QCC_ERR_CUDA;
  a.y_vec4 = reinterpret_cast<uintptr_t>(a.y) % (4 * dtype_bytes(a.y_dtype)) == 0 && a.ldy % 4 == 0;
  clear_stale_error();
  return gated ? launch<true>(a, device, stream) : launch<false>(a, device, stream);
}

}  // namespace
}  // namespace qcc

extern "C" int qcc_int8_linear(const int8_t* x, int64_t ldx, const float* x_scale, const int8_t* w, int64_t ldw,
                               const float* w_scale, const void* bias, int bias_dtype, int tokens, int channels,
                               int cols, void* y, int64_t ldy, int y_dtype, cudaStream_t stream) {
  return qcc::run_int8_linear({x, ldx, x_scale, w, ldw, w_scale, bias, bias_dtype, tokens, channels, cols, y, ldy,
                               y_dtype}, false, stream);
}

extern "C" int qcc_int8_gated_linear(const int8_t* x, int64_t ldx, const float* x_scale, const int8_t* w, int64_t ldw,
                                     const float* w_scale, int tokens, int channels, int cols, void* y, int64_t ldy,
                                     int y_dtype, cudaStream_t stream) {
  return qcc::run_int8_linear({x, ldx, x_scale, w, ldw, w_scale, nullptr, QCC_DTYPE_F32, tokens, channels, cols, y,
                               ldy, y_dtype}, true, stream);
}
