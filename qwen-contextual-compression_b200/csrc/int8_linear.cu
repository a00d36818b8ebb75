// Products of 8-bit integer matrices with a scale per token and per channel.
//
//   acc[t, n] = sum_k xq[t, k] * wq[n, k]                 (int32, exact)
//   y[t, n]   = fp32(acc) * (xs[t] * ws[n]) + bias[n]     rounded once (scales at the ends of fp32: see scaled())
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
  uint64_t wait_ns;  // bound of the waits for copies and for free slots
};

// silu with the fast exponential and quotient, from exp(-|g|), at most 1: exp's argument rounds once (an error of |g|
// roundings in exp), exp and the quotient are off by 2 ulp each, and the divisor is between 1 and 2 (beyond 2^126, as
// 1 + exp(-g) is below g = -87.3, the fast quotient is 0).
__device__ __forceinline__ float silu(float g) {
  const float e = __expf(-fabsf(g));
  return __fdividef(g < 0.f ? g * e : g, 1.f + e);
}

// Scales whose product is a normal number whatever the other one is: fp32(sum) * (xs * ws) then rounds three times.
__device__ __forceinline__ bool ordinary_scale(float s) {
  return s == 0.f || (fabsf(s) >= 0x1p-62f && fabsf(s) <= 0x1p62f);
}

// sum * xs * ws for other scales, whose product can leave the normal range though the result does not: it would lose
// places or become 0 (rows of values near 2^-119), or infinity, and NaN for a sum of 0.  The smaller scale first then:
// it shrinks the sum, or xs * ws and with it the result are beyond the range anyway.
__device__ __forceinline__ float scaled(int sum, float xs, float ws) {
  const float v = static_cast<float>(sum);
  const float product = xs * ws;
  if (fabsf(product) >= 0x1p-126f && fabsf(product) <= 0x1.fffffep127f) return v * product;
  const bool x_first = fabsf(xs) < fabsf(ws);
  return v * (x_first ? xs : ws) * (x_first ? ws : xs);
}

__device__ __forceinline__ float bias_value(const void* bias, int dtype, int n) {
  if (bias == nullptr) return 0.f;
  if (dtype == QCC_DTYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(bias)[n]);
  if (dtype == QCC_DTYPE_F16) return __half2float(static_cast<const __half*>(bias)[n]);
  return static_cast<const float*>(bias)[n];
}

// ---------------------------------------------------------------------------
// Both kernels keep weight rows in TMEM lanes (the M operand of tcgen05.mma
// kind::i8) and tokens in TMEM columns (the N operand), so one decoded token
// costs 16 columns of N, not 128 rows of M.  Lane l of a warp finishes one
// weight row's products with a run of tokens; a warp's store of one token is
// 32 consecutive channels.
// Gated: 32 lanes are 16 gate rows and the up rows of the same 16 channels, so
// one shuffle brings two tokens' gate and up together and every lane has one
// output of the two to finish.
// Waits are bounded.  A CTA (or pair) whose wait ran out starts nothing more,
// sees its MMAs and copies in (copies would land in the shared memory of a
// later block) and writes NaN: the stream kernel its tile, a pair all its tiles.
// ---------------------------------------------------------------------------

constexpr int kTileRows = 128;  // weight rows of a CTA's tile: TMEM lanes
constexpr int kTileCols = 128;  // bytes of K per stage (one swizzled row)
constexpr uint32_t kMaxSplit = 8;  // CTAs of a stream kernel's cluster, at most
constexpr int kAhead = 6;       // blocks of the weight that a stream kernel's CTA brings to L2 before it waits
constexpr uint64_t kDrainNs = 2000000000ull;  // for MMAs and copies in flight after a wait that ran out

// What one lane needs to finish its weight row's outputs.
template <bool GATED, typename O>
struct RowOutput {
  O* y;  // the first token's output of this lane's channel
  int64_t ldy;
  float ws, ws_up, bias;
  bool in;  // the channel exists
  bool ordinary;  // its scales are ordinary ones

  // row0: the first weight row (gated: channel) of the 32-lane group.
  __device__ __forceinline__ RowOutput(const Int8Args& a, int row0, int t0, int lane) {
    const int n = row0 + (GATED ? lane & 15 : lane);
    in = n < a.channels;
    ldy = a.ldy;
    y = static_cast<O*>(a.y) + static_cast<int64_t>(t0) * a.ldy + n;
    ws = in ? a.ws[n] : 0.f;
    ws_up = GATED && in ? a.ws[a.channels + n] : 0.f;
    bias = !GATED && in ? bias_value(a.bias, a.bias_dtype, n) : 0.f;
    ordinary = ordinary_scale(ws) && ordinary_scale(ws_up);
  }

  // For a tile whose wait ran out: its scales become NaN, and so do its outputs.
  __device__ __forceinline__ void break_off() { ws = NAN, ordinary = false; }

  // The same as finish for scales that are not ordinary, in few instructions rather than in short time.
  template <int J>
  __device__ __forceinline__ void finish_extreme(const int (&acc)[J], int c, int tokens, float xs, int lane) const {
#pragma unroll 1
    for (int k = 0; k < J && c + k < tokens; ++k) {
      int sum = 0;
#pragma unroll
      for (int j = 0; j < J; ++j) sum = j == k ? acc[j] : sum;
      const float scale = __shfl_sync(0xffffffffu, xs, k);
      O* to = y + static_cast<int64_t>(c + k) * ldy;
      if (GATED) {  // lanes 0-15 hold the gate's sums, lanes 16-31 the up rows'
        const int up = __shfl_xor_sync(0xffffffffu, sum, 16);
        if (lane < 16 && in) *to = static_cast<O>(silu(scaled(sum, scale, ws)) * scaled(up, scale, ws_up));
      } else if (in) {
        *to = static_cast<O>(scaled(sum, scale, ws) + bias);
      }
    }
  }

  // Finishes tokens c .. c + J - 1 (those below `tokens`) from their sums; lane j holds token c + j's scale.
  template <int J>
  __device__ __forceinline__ void finish(const int (&acc)[J], int c, int tokens, float xs, int lane) const {
    if (!__all_sync(0xffffffffu, ordinary && ordinary_scale(xs))) {
      finish_extreme(acc, c, tokens, xs, lane);
      return;
    }
    O* to = y + static_cast<int64_t>(c) * ldy;
    if (GATED) {
      // Lanes 0-15 finish the even tokens, lanes 16-31 the odd ones.
      const bool low = lane < 16;
      if (!low) to += ldy;
      const int left = in ? tokens - c - (low ? 0 : 1) : 0;
#pragma unroll
      for (int j = 0; j < J; j += 2) {
        const int other = __shfl_xor_sync(0xffffffffu, low ? acc[j + 1] : acc[j], 16);
        const float scale = __shfl_sync(0xffffffffu, xs, j + (low ? 0 : 1));
        const float g = static_cast<float>(low ? acc[j] : other) * (scale * ws);
        const float u = static_cast<float>(low ? other : acc[j + 1]) * (scale * ws_up);
        if (j < left) *to = static_cast<O>(silu(g) * u);
        to += 2 * ldy;
      }
    } else {
      const int left = in ? tokens - c : 0;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const float v = static_cast<float>(acc[j]) * (__shfl_sync(0xffffffffu, xs, j) * ws);
        if (j < left) *to = static_cast<O>(v + bias);
        to += ldy;
      }
    }
  }
};

// ---------------------------------------------------------------------------
// Stream kernel: one CTA computes 128 weight rows x BN tokens over its share of
// the columns; bound by the weight's bytes.  A cluster of S CTAs splits the
// columns when there are few rows: every CTA leaves its int32 partial sums in
// its own shared memory, and the cluster adds them over distributed shared
// memory -- integer sums, so the split changes no bit of the result, and there
// is no workspace that two calls could share.
// Measured: gate|up 34816 x 5120, 1 token 28.3 us (6.3 of 6.45 TB/s), 64 tokens
// 29.5 us, 128 tokens 33.6; down 5120 x 17408, 1 token 16.8 us (5.3 TB/s:
// filling the rings and joining the cluster take 3 us), 128 tokens 22.5 us, 256
// 33.2 (twice its floor: 128 x 128 tiles load 3.7 times the operands from L2).
// ---------------------------------------------------------------------------

template <int BN, int STAGES>
struct StreamShape {
  static constexpr int kWBytes = kTileRows * kTileCols, kXBytes = BN * kTileCols;
  static constexpr int kStage = kWBytes + kXBytes;
  static constexpr int kRing = STAGES * kStage;
  static_assert(BN * kTileRows * 4 <= kRing, "the ring holds the partial sums as [token][row] int32");
  static constexpr int kSmem = 1024 + kRing;  // ring aligned to 1024
  static constexpr uint32_t kTmemCols = BN < 32 ? 32 : BN;
};

__device__ __forceinline__ int cluster_load(uint32_t smem, uint32_t rank) {
  uint32_t remote;
  int v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem), "r"(rank));
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(remote) : "memory");
  return v;
}

template <bool GATED, typename O, int BN, int STAGES>
__global__ void __launch_bounds__(128)
    int8_stream_kernel(const Int8Args a, const __grid_constant__ CUtensorMap tm_x,
                       const __grid_constant__ CUtensorMap tm_w) {
  using S = StreamShape<BN, STAGES>;
  constexpr int kChannels = GATED ? kTileRows / 2 : kTileRows;
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t full[STAGES], empty[STAGES], done;
  __shared__ uint32_t tmem_slot;
  __shared__ int failed;
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t rank, splits;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(splits));
  const int n0 = static_cast<int>(blockIdx.x / splits) * kChannels, t0 = static_cast<int>(blockIdx.y) * BN;
  const int blocks = (a.cols + kTileCols - 1) / kTileCols;
  const int first = static_cast<int>(static_cast<int64_t>(blocks) * rank / splits);
  const int count = static_cast<int>(static_cast<int64_t>(blocks) * (rank + 1) / splits) - first;  // >= 1

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
    // The weight's first blocks start for L2 while the launches ahead finish (usually the one that makes x): a
    // prefetch moves no value into this kernel, so it may run ahead of a launch that writes the weight.  Norm and
    // gate|up of one token: 32.2 us without it, 30.9 with 4 or 8 blocks, 32.8 with 16.
    for (int i = 0; i < min(count, kAhead); ++i) {
      const int k = (first + i) * kTileCols;
      if (GATED) {
#pragma unroll
        for (int q = 0; q < 4; ++q) tma_prefetch_3d(&tm_w, k, n0 + q * 16, 0);
      } else {
        tma_prefetch_2d(&tm_w, k, n0);
      }
    }
  }
  // Tensor memory is taken only once the launches ahead have finished: a CTA
  // of theirs that still waits for its own columns must not wait for ours.
  // Beside launches of other streams an SM's 512 columns suffice: shared memory
  // admits three of these CTAs at most (two with 128 columns each), and neither
  // the pair kernel nor the prefill (197 and 205 KB) beside one.
  grid_dependency_wait();
  if (warp == 1) {
    tmem_alloc(&tmem_slot, S::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = tmem_slot;
  grid_dependency_trigger();

  // What the outputs need besides the sums arrives while those are made.
  const int tokens = min(BN, a.tokens - t0);
  RowOutput<GATED, O> out(a, n0 + warp * (GATED ? 16 : 32), t0, lane);
  const auto token_scale = [&](int c) { return c + lane < tokens ? a.xs[t0 + c + lane] : 0.f; };
  constexpr int kRun = 4;  // of a split: tokens a warp sums at a time; the cluster's CTAs take runs in turn
  float xs = token_scale(splits == 1 ? 0 : static_cast<int>(rank) * kRun);

  int issued = 0;  // thread 0: blocks whose copies it started
  if (threadIdx.x == 0) {
    const uint64_t keep = policy_evict_last(), stream = policy_evict_first();
    for (; issued < count; ++issued) {
      const int s = issued % STAGES;
      if (issued >= STAGES && !mbar_wait_suspended(&empty[s], (issued / STAGES - 1) & 1, a.wait_ns)) {
        failed = 1;
        break;
      }
      uint8_t* w = ring + s * S::kStage;
      mbar_arrive_expect_tx(&full[s], S::kStage);
      const int k = (first + issued) * kTileCols;
      if (GATED) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          tma_load_3d_hint(w + q * 32 * kTileCols, &tm_w, k, n0 + q * 16, 0, &full[s], stream);
      } else {
        tma_load_2d_hint(w, &tm_w, k, n0, &full[s], stream);
      }
      tma_load_2d_hint(w + S::kWBytes, &tm_x, k, t0, &full[s], keep);
    }
  } else if (threadIdx.x == 32) {
    constexpr uint32_t idesc = idesc_s8(kTileRows, BN);
    for (int i = 0; i < count; ++i) {
      const int s = i % STAGES;
      if (!mbar_wait_suspended(&full[s], (i / STAGES) & 1, a.wait_ns)) {
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
  if (!mbar_wait_suspended(&done, 0, 4 * max(a.wait_ns, kDrainNs))) failed = 1;
  tc_fence_after_sync();
  __syncthreads();

  const uint32_t from = tmem + (static_cast<uint32_t>(warp * 32) << 16);
  if (splits == 1) {
    if (failed != 0) out.break_off();
#pragma unroll 1
    for (int c = 0; c < tokens; c += 16) {
      const float xs_next = token_scale(c + 16);
      int acc[16];
      tmem_load16(from + c, acc);
      out.finish(acc, c, tokens, xs, lane);
      xs = xs_next;
    }
    tc_fence_before_sync();
    __syncthreads();
  } else {
    // The ring is free: every MMA has completed (where a wait ran out copies may still land in it, and all is NaN).
    int* partial = reinterpret_cast<int*>(ring);
#pragma unroll 1
    for (int c = 0; c < tokens; c += 16) {
      int acc[16];
      tmem_load16(from + c, acc);
#pragma unroll
      for (int j = 0; j < 16; ++j) partial[(c + j) * kTileRows + threadIdx.x] = acc[j];
    }
    tc_fence_before_sync();
    __syncwarp();
    cluster_sync();
    tc_fence_after_sync();
    // Remote loads take about 250 cycles: those of all ranks are in flight together.
    const uint32_t base = smem_addr(partial) + threadIdx.x * 4;
    int flags[kMaxSplit];
#pragma unroll
    for (uint32_t r = 0; r < kMaxSplit; ++r) flags[r] = r < splits ? cluster_load(smem_addr(&failed), r) : 0;
    const int step = static_cast<int>(splits) * kRun;
    for (int c = static_cast<int>(rank) * kRun; c < tokens; c += step) {
      const float xs_next = token_scale(c + step);
      int part[kMaxSplit][kRun];
#pragma unroll
      for (uint32_t r = 0; r < kMaxSplit; ++r)
#pragma unroll
        for (int j = 0; j < kRun; ++j)
          part[r][j] = r < splits && c + j < tokens ? cluster_load(base + (c + j) * kTileRows * 4, r) : 0;
      int acc[kRun] = {};
#pragma unroll
      for (uint32_t r = 0; r < kMaxSplit; ++r) {
        if (flags[r] != 0) out.break_off();
#pragma unroll
        for (int j = 0; j < kRun; ++j) acc[j] += part[r][j];
      }
      out.finish(acc, c, tokens, xs, lane);
      xs = xs_next;
    }
    __syncwarp();
    cluster_sync();  // the other CTAs have read this one's sums
  }
  if (failed != 0 && threadIdx.x == 0)
    for (int i = max(0, issued - STAGES); i < issued; ++i)
      mbar_wait_suspended(&full[i % STAGES], (i / STAGES) & 1, kDrainNs);
  if (warp == 1) tmem_dealloc(tmem, S::kTmemCols);
}

// ---------------------------------------------------------------------------
// Pair kernel: persistent CTA pairs (cta_group::2), tiles of 256 weight rows x
// up to 256 tokens over all columns, for token counts that make the product
// compute bound.  Warp 0 loads, warp 1 of the even CTA issues the MMAs, warps
// 2-9 drain the accumulators; two accumulators (2 x 256 of the 512 TMEM
// columns) let a tile's epilogue run beside the next tile's MMAs.  A pair reads
// each operand byte of its tile once (128 rows of each per CTA), half of what
// two single CTAs would.
// Measured at 4096 tokens: gate|up 34816 x 5120 454 us (3.2 POP/s), down 5120 x
// 17408 230 us (3.2 POP/s; 320 tiles are 4.3 rounds of 74 pairs).  In runs of
// seconds, with the launches before them, 561 to 593 and 309 to 329 us: the
// card sits at its 1000 W then, as in cuBLAS's bf16 product (1.4 PFLOP/s
// sustained): power bounds it.
// ---------------------------------------------------------------------------

constexpr int kPairStages = 6;
constexpr int kPairTokens = 256;                       // most tokens of a tile
constexpr int kPairStage = 2 * 128 * kTileCols;        // bytes a CTA loads per stage, at most
constexpr int kPairSmem = 1024 + kPairStages * kPairStage;
constexpr int kPairThreads = 320;
constexpr int kPairGroup = 8;  // token tiles walked through together (4096 tokens: 4, 8 or 16 within 4 %)

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

// Notes a wait that ran out in both CTAs of the pair, before the commits that follow.
__device__ __forceinline__ void note_failure(int* failed, uint32_t rank) {
  *static_cast<volatile int*>(failed) = 1;
  const uint32_t other = cluster_addr(failed, rank ^ 1u);
  asm volatile("st.shared::cluster.s32 [%0], %1;\n\tfence.acq_rel.cluster;" ::"r"(other), "r"(1) : "memory");
}

template <bool GATED, typename O>
__global__ void __launch_bounds__(kPairThreads, 1)
    int8_pair_kernel(const Int8Args a, const PairPlan plan, const __grid_constant__ CUtensorMap tm_x,
                     const __grid_constant__ CUtensorMap tm_w) {
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t full[kPairStages], empty[kPairStages], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int failed, issued;  // issued: column blocks whose copies this CTA started
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
      mbar_init(&acc_empty[s], 16);  // the eight epilogue warps of both CTAs
    }
    failed = 0;
    fence_barrier_init();
  }
  grid_dependency_wait();  // before tensor memory is taken, as in the stream kernel
  if (warp == 1) {
    tmem_alloc_pair(&tmem_slot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync();  // both CTAs' barriers are initialised
  tc_fence_after_sync();
  const uint32_t tmem = tmem_slot;
  grid_dependency_trigger();

  // This CTA's copies of column block b of a tile into stage s, counted with the other CTA's on the even one's barrier.
  const auto load = [&](int row, int token, int b, int s) {
    const uint64_t keep = policy_evict_last();
    uint8_t* w = ring + s * kPairStage;
    const uint32_t bar = cluster_addr(&full[s], 0);
    if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * (128 + half_tokens) * kTileCols);
    const int k = b * kTileCols;
    if (GATED) {
      const int n0 = row * kChannels + static_cast<int>(rank) * 64;
#pragma unroll
      for (int q = 0; q < 4; ++q)
        tma_load_3d_pair(w + q * 32 * kTileCols, &tm_w, k, n0 + q * 16, 0, bar, keep);
    } else {
      tma_load_2d_pair(w, &tm_w, k, row * kChannels + static_cast<int>(rank) * 128, bar, keep);
    }
    tma_load_2d_pair(w + 128 * kTileCols, &tm_x, k, token * plan.tile_tokens + static_cast<int>(rank) * half_tokens,
                     bar, keep);
  };

  if (threadIdx.x == 0) {
    int n = 0;  // stage uses so far
    bool ok = true;
    for (int i = pair; i < tiles && ok; i += pairs) {
      int row, token;
      pair_tile(plan, i, row, token);
      for (int b = 0; b < blocks; ++b, ++n) {
        const int s = n % kPairStages;
        if (n >= kPairStages && !mbar_wait_suspended(&empty[s], (n / kPairStages - 1) & 1, a.wait_ns)) {
          note_failure(&failed, rank);
          ok = false;
          break;
        }
        load(row, token, b, s);
      }
    }
    issued = n;
  } else if (threadIdx.x == 32 && rank == 0) {
    const uint32_t idesc = idesc_s8(256, plan.tile_tokens);
    int n = 0, done = 0;
    bool ok = true;
    for (int i = pair; i < tiles && ok; i += pairs, ++done) {
      const int acc = done & 1;
      if (done >= 2 && !mbar_wait_suspended(&acc_empty[acc], (done / 2 - 1) & 1, a.wait_ns)) {
        note_failure(&failed, rank);
        ok = false;
        break;
      }
      tc_fence_after_sync();
      for (int b = 0; b < blocks; ++b, ++n) {
        const int s = n % kPairStages;
        if (!mbar_wait_suspended(&full[s], (n / kPairStages) & 1, a.wait_ns)) {
          note_failure(&failed, rank);
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
    if (!ok && done > 0) mbar_wait_suspended(&acc_full[(done - 1) & 1], ((done - 1) / 2) & 1, kDrainNs);
  } else if (warp >= 2) {
    const int quarter = warp & 3;  // TMEM lanes 32 * quarter .. + 31
    int done = 0;
    bool broken = false;
    for (int i = pair; i < tiles; i += pairs, ++done) {
      const int acc = done & 1;
      if (!broken && !mbar_wait_suspended(&acc_full[acc], (done / 2) & 1, 4 * max(a.wait_ns, kDrainNs)))
        note_failure(&failed, rank);
      broken = *static_cast<volatile int*>(&failed) != 0;  // and all tiles after it: their waits would run out too
      tc_fence_after_sync();
      int row, token;
      pair_tile(plan, i, row, token);
      const int t0 = token * plan.tile_tokens, tokens = min(plan.tile_tokens, a.tokens - t0);
      RowOutput<GATED, O> out(
          a, row * kChannels + static_cast<int>(rank) * (kChannels / 2) + quarter * (GATED ? 16 : 32), t0, lane);
      if (broken) out.break_off();
      const uint32_t from = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + acc * 256;
      int c = (warp - 2) / 4 * 32;
      for (; c < tokens; c += 64) {
        int sums[32];
        tmem_load32(from + c, sums);
        const float xs = c + lane < tokens ? a.xs[t0 + c + lane] : 0.f;
        if (c + 64 >= tokens) {  // this warp's last columns are in registers
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(cluster_addr(&acc_empty[acc], 0));
        }
        out.finish(sums, c, tokens, xs, lane);
      }
      if (tokens <= 32 && c == 32) {  // the second four warps had no column of this tile
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(cluster_addr(&acc_empty[acc], 0));
      }
    }
  }
  __syncwarp();
  tc_fence_before_sync();
  cluster_sync();  // no barrier of this CTA is signalled and none of its memory read after this
  tc_fence_after_sync();
  if (*static_cast<volatile int*>(&failed) != 0) {  // in both CTAs or in neither
    if (threadIdx.x == 0) {
      // The even CTA's barriers complete by both CTAs' bytes: the CTA that started fewer blocks starts the others,
      // whose stages are free (the other CTA found them so), and the even one sees all of them in.
      const int most = max(issued, cluster_load(smem_addr(&issued), rank ^ 1u));
      for (int n = issued; n < most; ++n) {
        int row, token;
        pair_tile(plan, pair + n / blocks * pairs, row, token);
        load(row, token, n % blocks, n % kPairStages);
      }
      if (rank == 0)
        for (int i = max(0, most - kPairStages); i < most; ++i)
          mbar_wait_suspended(&full[i % kPairStages], (i / kPairStages) & 1, kDrainNs);
    }
    for (int i = pair; i < tiles; i += pairs) {
      int row, token;
      pair_tile(plan, i, row, token);
      const int n0 = row * kChannels + static_cast<int>(rank) * (kChannels / 2), t0 = token * plan.tile_tokens;
      const int channels = min(kChannels / 2, a.channels - n0), tokens = min(plan.tile_tokens, a.tokens - t0);
      for (int e = threadIdx.x; e < channels * tokens; e += kPairThreads)
        static_cast<O*>(a.y)[(t0 + e / channels) * a.ldy + n0 + e % channels] = static_cast<O>(NAN);
    }
    __syncwarp();
    cluster_sync();
  }
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

// The gate and the up rows of a fused weight as two planes: a box holds 16 rows of each, one warp's 32 lanes (one copy
// for both: two copies of 16 rows took 15 % longer at 4096 tokens).
bool make_gated_map(CUtensorMap* map, const int8_t* base, int64_t channels, int64_t cols, int64_t ld) {
  auto fn = encode_tiled();
  if (fn == nullptr) return false;
  const uint64_t dims[3] = {static_cast<uint64_t>(cols), static_cast<uint64_t>(channels), 2};
  const uint64_t strides[2] = {static_cast<uint64_t>(ld), static_cast<uint64_t>(channels * ld)};
  const uint32_t box[3] = {kTileCols, 16, 2}, elem[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<int8_t*>(base), dims, strides, box, elem,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// A launch on `stream` as clusters of `cluster` CTAs that may start while the launch ahead of it finishes.
template <typename... P, typename... A>
int launch_clusters(void (*kernel)(P...), dim3 grid, int threads, int smem, int cluster, cudaStream_t stream,
                    const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cuda_ok(cudaLaunchKernelEx(&cfg, kernel, args...)) ? QCC_OK : QCC_ERR_CUDA;
}

template <bool GATED, typename O, int BN, int STAGES>
int launch_stream(const Int8Args& a, int device, cudaStream_t stream) {
  using S = StreamShape<BN, STAGES>;
  constexpr int kChannels = GATED ? kTileRows / 2 : kTileRows;
  auto* kernel = int8_stream_kernel<GATED, O, BN, STAGES>;
  CUtensorMap tm_x, tm_w;
  if (!make_map(&tm_x, a.x, a.tokens, a.cols, a.ldx, BN) ||
      !(GATED ? make_gated_map(&tm_w, a.w, a.channels, a.cols, a.ldw)
              : make_map(&tm_w, a.w, a.channels, a.cols, a.ldw, kTileRows)))
    return QCC_ERR_UNSUPPORTED;
  if (!ensure_max_dynamic_smem(reinterpret_cast<const void*>(kernel), device)) return QCC_ERR_CUDA;
  const int tiles = (a.channels + kChannels - 1) / kChannels, token_tiles = (a.tokens + BN - 1) / BN;
  // Columns are split while all CTAs still run at once: a second wave costs more than the split brings (17408 columns
  // to 5120 channels, 32 tokens, two CTAs an SM: 240 CTAs 19.1 us, 320 CTAs 25.2 us).  Clusters leave part of a
  // GPC's slots empty, hence 85 %.
  const int slots = device_info(device).num_sms * std::max(1, (225 << 10) / (S::kSmem + 2048)) * 85 / 100;
  const int blocks = (a.cols + kTileCols - 1) / kTileCols;
  const int split = static_cast<int>(
      std::max<int64_t>(1, std::min<int64_t>({kMaxSplit, blocks, slots / (1ll * tiles * token_tiles)})));
  return launch_clusters(kernel, dim3(tiles * split, token_tiles), 128, S::kSmem, split, stream, a, tm_x, tm_w);
}

template <bool GATED, typename O>
int launch_pair(const Int8Args& a, int device, cudaStream_t stream) {
  auto* kernel = int8_pair_kernel<GATED, O>;
  const int channels = GATED ? 128 : 256;
  const int pairs = device_info(device).num_sms / 2;
  PairPlan plan;
  plan.row_tiles = (a.channels + channels - 1) / channels;
  // As few token tiles as fit, of equal width: a tile's time hardly falls with its width (4096 tokens of the 34816 x
  // 5120 gated product: 458 us at 256 wide, 559 at 192, 741 at 128), its weight rows' loads stay.
  plan.token_tiles = (a.tokens + kPairTokens - 1) / kPairTokens;
  plan.tile_tokens = ((a.tokens + plan.token_tiles - 1) / plan.token_tiles + 31) / 32 * 32;
  plan.group = kPairGroup;
  CUtensorMap tm_x, tm_w;
  if (!make_map(&tm_x, a.x, a.tokens, a.cols, a.ldx, plan.tile_tokens / 2) ||
      !(GATED ? make_gated_map(&tm_w, a.w, a.channels, a.cols, a.ldw)
              : make_map(&tm_w, a.w, a.channels, a.cols, a.ldw, 128)))
    return QCC_ERR_UNSUPPORTED;
  if (!ensure_max_dynamic_smem(reinterpret_cast<const void*>(kernel), device)) return QCC_ERR_CUDA;
  const unsigned grid = 2u * static_cast<unsigned>(std::min<int64_t>(
                                 pairs, static_cast<int64_t>(plan.row_tiles) * plan.token_tiles));
  return launch_clusters(kernel, dim3(grid), kPairThreads, kPairSmem, 2, stream, a, plan, tm_x, tm_w);
}

// Bytes that the stream kernel's CTAs load with tiles of `bn` tokens.
int64_t stream_loads(const Int8Args& a, bool gated, int bn) {
  const int channels = gated ? kTileRows / 2 : kTileRows;
  const int64_t tiles = static_cast<int64_t>((a.channels + channels - 1) / channels) * ((a.tokens + bn - 1) / bn);
  return tiles * ((a.cols + kTileCols - 1) / kTileCols) * (kTileRows + bn) * kTileCols;
}

template <bool GATED, typename O>
int launch(const Int8Args& a, int device, cudaStream_t stream) {
  if (a.tokens <= 16) return launch_stream<GATED, O, 16, 4>(a, device, stream);
  if (a.tokens <= 32) return launch_stream<GATED, O, 32, 4>(a, device, stream);
  if (a.tokens <= 64) return launch_stream<GATED, O, 64, 4>(a, device, stream);
  // Pairs where their tiles fill at least half of the SMs (512 tokens, 17408 columns to 5120 channels, 40 tiles: pairs
  // 48 us, stream 60 us; 256 tokens, 20 tiles: 46 and 33 us; 256 tokens of 4000 x 4000, 16 tiles: 17.3 and 13.4).  Not
  // right everywhere: 256 tokens of 6000 x 6000, 24 tiles, 25.4 and 33.8.
  const int channels = GATED ? 128 : 256;
  const int64_t pair_tiles = static_cast<int64_t>((a.channels + channels - 1) / channels) *
                             ((a.tokens + kPairTokens - 1) / kPairTokens);
  if (a.tokens > 128 && 4 * pair_tiles >= device_info(device).num_sms) return launch_pair<GATED, O>(a, device, stream);
  // Narrow token tiles make more CTAs, wide ones load the weight less often (200 tokens of a 4000 x 4000 weight, 101 MB
  // of loads at 64: 13.4 us, at 128 17.8 us; 256 tokens of 9000 columns to 2560 channels, 140 MB: 24.1 and 20.4; of
  // 17408 to 5120, 535 MB: 43.5 and 33.5).  The number of CTAs counts as well: 100 tokens of 6000 x 6000, 109 MB, 22.1
  // and 18.2.
  if (stream_loads(a, GATED, 64) <= (128 << 20)) return launch_stream<GATED, O, 64, 4>(a, device, stream);
  return launch_stream<GATED, O, 128, 3>(a, device, stream);
}

template <bool GATED>
int launch(const Int8Args& a, int device, cudaStream_t stream) {
  if (a.y_dtype == QCC_DTYPE_BF16) return launch<GATED, __nv_bfloat16>(a, device, stream);
  if (a.y_dtype == QCC_DTYPE_F16) return launch<GATED, __half>(a, device, stream);
  return launch<GATED, float>(a, device, stream);
}

int run_int8_linear(Int8Args a, bool gated, cudaStream_t stream) {
  if (!valid_dtype(a.y_dtype) || (a.bias != nullptr && !valid_dtype(a.bias_dtype))) return QCC_ERR_DTYPE;
  if (a.tokens < 0 || a.channels < 1 || a.cols < 1 || a.ldx < a.cols || a.ldw < a.cols || a.ldy < a.channels)
    return QCC_ERR_SHAPE;
  if (a.cols > kMaxCols || a.channels > kMaxChannels || a.tokens > kMaxTokens) return QCC_ERR_UNSUPPORTED;
  if (a.tokens == 0) return QCC_OK;
  if (a.x == nullptr || a.xs == nullptr || a.w == nullptr || a.ws == nullptr || a.y == nullptr)
    return QCC_ERR_INVALID_ARGUMENT;
  const auto misaligned = [](const void* p, int size) { return reinterpret_cast<uintptr_t>(p) % size != 0; };
  if (!aligned16(a.x) || !aligned16(a.w) || a.ldx % 16 != 0 || a.ldw % 16 != 0 || misaligned(a.xs, 4) ||
      misaligned(a.ws, 4) || misaligned(a.y, dtype_bytes(a.y_dtype)) ||
      (a.bias != nullptr && misaligned(a.bias, dtype_bytes(a.bias_dtype))))
    return QCC_ERR_ALIGNMENT;
  int device = 0;
  if (!cuda_ok(cudaGetDevice(&device))) return QCC_ERR_CUDA;
  clear_stale_error();
  a.wait_ns = wait_limit_ns();
  return gated ? launch<true>(a, device, stream) : launch<false>(a, device, stream);
}

}  // namespace
}  // namespace qcc

extern "C" int qcc_int8_linear(const int8_t* x, int64_t ldx, const float* x_scale, const int8_t* w, int64_t ldw,
                               const float* w_scale, const void* bias, int bias_dtype, int tokens, int channels,
                               int cols, void* y, int64_t ldy, int y_dtype, cudaStream_t stream) {
  return qcc::run_int8_linear({x, ldx, x_scale, w, ldw, w_scale, bias, bias_dtype, tokens, channels, cols, y, ldy,
                               y_dtype, 0}, false, stream);
}

extern "C" int qcc_int8_gated_linear(const int8_t* x, int64_t ldx, const float* x_scale, const int8_t* w, int64_t ldw,
                                     const float* w_scale, int tokens, int channels, int cols, void* y, int64_t ldy,
                                     int y_dtype, cudaStream_t stream) {
  return qcc::run_int8_linear({x, ldx, x_scale, w, ldw, w_scale, nullptr, QCC_DTYPE_F32, tokens, channels, cols, y,
                               ldy, y_dtype, 0}, true, stream);
}
