// Products of 8-bit integer matrices with a scale per token and per channel.
//
//   acc[t, n] = sum_k xq[t, k] * wq[n, k]                 (int32, exact)
//   y[t, n]   = fp32(acc) * (xs[t] * ws[n]) + bias[n]     rounded once
// and, for the gated form (wq holds the gate rows 0..N-1, then the up rows),
//   y[t, n]   = silu(g) * u  with g, u the two products of channel n.
#include <cuda_runtime.h>

#include <algorithm>

#include "qcc_common.cuh"
#include "qcc_host.h"

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
};

__device__ __forceinline__ float silu(float g) { return g / (1.f + expf(-g)); }

__device__ __forceinline__ float bias_value(const void* bias, int dtype, int n) {
  if (bias == nullptr) return 0.f;
  if (dtype == QCC_DTYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(bias)[n]);
  if (dtype == QCC_DTYPE_F16) return __half2float(static_cast<const __half*>(bias)[n]);
  return static_cast<const float*>(bias)[n];
}

// One output a thread, 16 x 16 outputs a CTA, 64 columns of both operands in
// shared memory at a time.
template <bool GATED>
__global__ void __launch_bounds__(256) int8_linear_kernel(const Int8Args a) {
  constexpr int kStep = 64, kRow = kStep / 4 + 1;
  constexpr int kParts = GATED ? 2 : 1;
  __shared__ int xt[16 * kRow], wt[kParts * 16 * kRow];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int t0 = blockIdx.x * 16, n0 = blockIdx.y * 16;
  int acc[kParts] = {};
  for (int k0 = 0; k0 < a.cols; k0 += kStep) {
    for (int i = threadIdx.x; i < 16 * (kStep / 4) * (1 + kParts); i += 256) {
      const int part = i / (16 * (kStep / 4)), r = i / (kStep / 4) % 16, c = i % (kStep / 4);
      const int8_t* base = part == 0 ? a.x : a.w;
      const int64_t row = part == 0 ? t0 + r : n0 + r;
      const bool in = part == 0 ? row < a.tokens : row < a.channels;
      const int64_t at = part == 0 ? row * a.ldx : (row + (part - 1) * static_cast<int64_t>(a.channels)) * a.ldw;
      uint32_t word = 0;
      for (int b = 0; b < 4; ++b) {
        const int k = k0 + c * 4 + b;
        if (in && k < a.cols) word |= static_cast<uint32_t>(static_cast<uint8_t>(base[at + k])) << (8 * b);
      }
      (part == 0 ? xt : wt + (part - 1) * 16 * kRow)[r * kRow + c] = static_cast<int>(word);
    }
    __syncthreads();
    for (int c = 0; c < kStep / 4; ++c)
#pragma unroll
      for (int p = 0; p < kParts; ++p) acc[p] = __dp4a(xt[ty * kRow + c], wt[(p * 16 + tx) * kRow + c], acc[p]);
    __syncthreads();
  }
  const int t = t0 + ty, n = n0 + tx;
  if (t >= a.tokens || n >= a.channels) return;
  const float xs = a.xs[t];
  float v = static_cast<float>(acc[0]) * (xs * a.ws[n]);
  if (GATED)
    v = silu(v) * (static_cast<float>(acc[kParts - 1]) * (xs * a.ws[a.channels + n]));
  else
    v += bias_value(a.bias, a.bias_dtype, n);
  store_as(a.y, t * a.ldy + n, a.y_dtype, v);
}

int run_int8_linear(const Int8Args& a, bool gated, cudaStream_t stream) {
  if (!valid_dtype(a.y_dtype) || (a.bias != nullptr && !valid_dtype(a.bias_dtype))) return QCC_ERR_DTYPE;
  if (a.tokens < 0 || a.channels < 1 || a.cols < 1 || a.ldx < a.cols || a.ldw < a.cols || a.ldy < a.channels)
    return QCC_ERR_SHAPE;
  if (a.cols > kMaxCols || a.channels > kMaxChannels || a.tokens > kMaxTokens) return QCC_ERR_UNSUPPORTED;
  if (a.tokens == 0) return QCC_OK;
  if (a.x == nullptr || a.xs == nullptr || a.w == nullptr || a.ws == nullptr || a.y == nullptr)
    return QCC_ERR_INVALID_ARGUMENT;
  if (!aligned16(a.x) || !aligned16(a.w) || a.ldx % 16 != 0 || a.ldw % 16 != 0) return QCC_ERR_ALIGNMENT;
  const dim3 grid((a.tokens + 15) / 16, (a.channels + 15) / 16);
  clear_stale_error();
  if (gated)
    int8_linear_kernel<true><<<grid, 256, 0, stream>>>(a);
  else
    int8_linear_kernel<false><<<grid, 256, 0, stream>>>(a);
  return launch_ok() ? QCC_OK : QCC_ERR_CUDA;
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
