// Norms before and after an FFN block, fused with the block's gate and
// residual scale, and the int8 quantisation of rows.
//
// For every row t (all sums and products in fp32, each output rounded once):
//   b = N_post(y_t)                                   branch, after its norm
//   r = residual_scale * res_t + branch_scale * act(g_t) * b
//   residual_out_t = r
//   x = N_next(r)                                     input of the next block
//   out_t = x, or q = rint(x * 127 / amax|x|) with row_scale = amax / 127
// N is the identity, the RMS norm v * rsqrt(mean v^2 + eps) * (o + w) + b or
// the layer norm (v - mean) * rsqrt(var + eps) * (o + w) + b.  The next norm
// takes r before residual_out's rounding.
//
// One pass: a row's values stay in registers between the reductions (the
// layer norm's variance is a second sum over centred values, not a difference
// of moments), so DRAM sees each input once and each output once.
#include <cuda_runtime.h>

#include <algorithm>
#include <cfloat>

#include "qcc_common.cuh"
#include "qcc_host.h"

namespace qcc {
namespace {

constexpr int kMaxThreads = 1024;
constexpr int kMaxVecs = 4;                               // 8-element vectors a thread keeps
constexpr int kMaxHidden = kMaxThreads * kMaxVecs * 8;    // 32768
// A row whose largest magnitude is below this is stored as zeros: its scale
// (and 127 / amax) would leave the normal fp32 range.
constexpr float kSmallestAmax = 1.504632769052528e-36f;   // 2^-119

struct BlockNormArgs {
  const void* y;
  int64_t ldy;
  const void* res;  // NULL: r = y (no residual)
  int64_t ld_res;
  int rows, hidden;
  float residual_scale, branch_scale;
  qcc_norm_params post, next;
  qcc_gate_params gate;  // values NULL: none
  void* res_out;
  int64_t ld_res_out;
  void* out;  // NULL: residual_out only
  int64_t ld_out;
  int out_dtype;  // QCC_DTYPE_* or QCC_DTYPE_I8
  float* row_scale;
};

// Element index of value j of vector v: vectors of 8 consecutive elements, or
// (rows that are not 16-byte aligned) single elements a block width apart.
template <bool VEC>
__device__ __forceinline__ int element(int v, int j) {
  const int bd = static_cast<int>(blockDim.x), tid = static_cast<int>(threadIdx.x);
  return VEC ? (v * bd + tid) * 8 + j : (v * 8 + j) * bd + tid;
}

template <typename T, bool VEC>
__device__ __forceinline__ void load_row8(const T* row, int v, int n, float (&f)[8]) {
  if (VEC) {
    const int e = element<true>(v, 0);
    if (e + 8 <= n) {
      widen(load_pack8<T>(row + e), f);
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int e = element<VEC>(v, j);
    f[j] = e < n ? to_f32<T>(row[e]) : 0.f;
  }
}

template <bool VEC>
__device__ __forceinline__ void load_any8(const void* row, int dtype, int v, int n, float (&f)[8]) {
  if (dtype == QCC_DTYPE_BF16)
    load_row8<__nv_bfloat16, VEC>(static_cast<const __nv_bfloat16*>(row), v, n, f);
  else if (dtype == QCC_DTYPE_F16)
    load_row8<__half, VEC>(static_cast<const __half*>(row), v, n, f);
  else
    load_row8<float, VEC>(static_cast<const float*>(row), v, n, f);
}

__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16*) {
  __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&p);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half*) {
  __half2 p = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&p);
}

template <typename T>
__device__ __forceinline__ void store_vec8(T* p, const float* f) {
  uint4 w;
  w.x = pack2(f[0], f[1], p);
  w.y = pack2(f[2], f[3], p);
  w.z = pack2(f[4], f[5], p);
  w.w = pack2(f[6], f[7], p);
  *reinterpret_cast<uint4*>(p) = w;
}
__device__ __forceinline__ void store_vec8(float* p, const float* f) {
  reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
}

template <typename T, bool VEC>
__device__ __forceinline__ void store_row8(T* row, int v, int n, const float* f) {
  if (VEC) {
    const int e = element<true>(v, 0);
    if (e + 8 <= n) {
      store_vec8(row + e, f);
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int e = element<VEC>(v, j);
    if (e < n) row[e] = static_cast<T>(f[j]);
  }
}

template <bool VEC>
__device__ __forceinline__ void store_any8(void* row, int dtype, int v, int n, const float* f) {
  if (dtype == QCC_DTYPE_BF16)
    store_row8<__nv_bfloat16, VEC>(static_cast<__nv_bfloat16*>(row), v, n, f);
  else if (dtype == QCC_DTYPE_F16)
    store_row8<__half, VEC>(static_cast<__half*>(row), v, n, f);
  else
    store_row8<float, VEC>(static_cast<float*>(row), v, n, f);
}

// |f| <= 127 / inverse by construction, so the rounded value fits int8.
template <bool VEC>
__device__ __forceinline__ void store_int8x8(int8_t* row, int v, int n, const float* f, float inverse) {
  uint32_t q[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) q[j] = static_cast<uint32_t>(__float2int_rn(f[j] * inverse)) & 0xFFu;
  if (VEC) {
    const int e = element<true>(v, 0);
    if (e + 8 <= n) {
      uint2 w;
      w.x = q[0] | (q[1] << 8) | (q[2] << 16) | (q[3] << 24);
      w.y = q[4] | (q[5] << 8) | (q[6] << 16) | (q[7] << 24);
      *reinterpret_cast<uint2*>(row + e) = w;
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int e = element<VEC>(v, j);
    if (e < n) row[e] = static_cast<int8_t>(q[j]);
  }
}

struct SumOp {
  static __device__ __forceinline__ float apply(float a, float b) { return a + b; }
};
struct MaxOp {
  static __device__ __forceinline__ float apply(float a, float b) { return fmaxf(a, b); }
};

// Reduction over the block in a fixed order; every thread gets the result.
template <typename Op>
__device__ __forceinline__ float block_reduce(float v, float* scratch) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = Op::apply(v, __shfl_xor_sync(0xffffffffu, v, o));
  const int warps = static_cast<int>(blockDim.x) >> 5;
  if (warps == 1) return v;
  __syncthreads();  // the previous reduction's readers are done
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = static_cast<int>(threadIdx.x & 31) < warps ? scratch[threadIdx.x & 31] : scratch[0];
  if (static_cast<int>(threadIdx.x & 31) >= warps) s = Op::apply(0.f, 0.f);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s = Op::apply(s, __shfl_xor_sync(0xffffffffu, s, o));
  return s;
}

// v <- N(v) over the row's `n` values (entries past the row are 0 on entry and on exit).
template <int VPT, bool VEC>
__device__ __forceinline__ void normalise(float (&v)[VPT][8], const qcc_norm_params& a, int n, float* scratch) {
  if (a.kind == QCC_NORM_NONE) return;
  float mean = 0.f;
  if (a.kind == QCC_NORM_LAYER) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) s += v[i][j];
    mean = block_reduce<SumOp>(s, scratch) / static_cast<float>(n);
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = element<VEC>(i, j) < n ? v[i][j] - mean : 0.f;
  }
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < VPT; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) s += v[i][j] * v[i][j];
  s = block_reduce<SumOp>(s, scratch);
  const float rstd = 1.f / sqrtf(s / static_cast<float>(n) + a.eps);
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    float w[8];
    if (a.weight != nullptr) {
      load_any8<VEC>(a.weight, a.dtype, i, n, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] *= rstd * (a.weight_offset + w[j]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] *= rstd;
    }
    if (a.bias != nullptr) {
      load_any8<VEC>(a.bias, a.dtype, i, n, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] += w[j];
    }
  }
}

__device__ __forceinline__ float gate_value(float g, int act) {
  if (act == QCC_GATE_SIGMOID) return 1.f / (1.f + expf(-g));
  if (act == QCC_GATE_TANH) return tanhf(g);
  return g;
}

// One CTA a row.  T: the branch's type, R: the residual's.
template <typename T, typename R, int VPT, bool VEC>
__global__ void __launch_bounds__(kMaxThreads) block_norm_kernel(const BlockNormArgs a) {
  __shared__ float scratch[32];
  const int64_t t = blockIdx.x;
  const int n = a.hidden;
  float v[VPT][8];
#pragma unroll
  for (int i = 0; i < VPT; ++i) load_row8<T, VEC>(static_cast<const T*>(a.y) + t * a.ldy, i, n, v[i]);
  if (a.res != nullptr) {
    normalise<VPT, VEC>(v, a.post, n, scratch);
    if (a.gate.values != nullptr) {
      const size_t gs = a.gate.dtype == QCC_DTYPE_F32 ? 4 : 2;
      const char* row = static_cast<const char*>(a.gate.values) + (t / a.gate.rows_each) * a.gate.ld * gs;
      if (a.gate.cols == 1) {
        const float g = a.gate.dtype == QCC_DTYPE_BF16
                            ? __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(row))
                        : a.gate.dtype == QCC_DTYPE_F16 ? __half2float(*reinterpret_cast<const __half*>(row))
                                                        : *reinterpret_cast<const float*>(row);
        const float s = gate_value(g, a.gate.act);
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
          for (int j = 0; j < 8; ++j) v[i][j] *= s;
      } else {
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
          float g[8];
          load_any8<VEC>(row, a.gate.dtype, i, n, g);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[i][j] *= gate_value(g[j], a.gate.act);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      float r[8];
      load_row8<R, VEC>(static_cast<const R*>(a.res) + t * a.ld_res, i, n, r);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        v[i][j] = element<VEC>(i, j) < n ? a.residual_scale * r[j] + a.branch_scale * v[i][j] : 0.f;
      if (a.res_out != nullptr) store_row8<R, VEC>(static_cast<R*>(a.res_out) + t * a.ld_res_out, i, n, v[i]);
    }
  }
  if (a.out == nullptr) return;
  normalise<VPT, VEC>(v, a.next, n, scratch);
  if (a.out_dtype != QCC_DTYPE_I8) {
    char* row = static_cast<char*>(a.out) + t * a.ld_out * (a.out_dtype == QCC_DTYPE_F32 ? 4 : 2);
#pragma unroll
    for (int i = 0; i < VPT; ++i) store_any8<VEC>(row, a.out_dtype, i, n, v[i]);
    return;
  }
  // amax with every non-finite value as +inf (fmaxf alone would drop a NaN).
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < VPT; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float m = fabsf(v[i][j]);
      if (element<VEC>(i, j) < n) amax = fmaxf(amax, m <= FLT_MAX ? m : INFINITY);
    }
  amax = block_reduce<MaxOp>(amax, scratch);
  const bool finite = amax <= FLT_MAX, kept = finite && amax >= kSmallestAmax;
  const float inverse = kept ? 127.f / amax : 0.f;
  if (threadIdx.x == 0) a.row_scale[t] = kept ? amax / 127.f : finite ? 0.f : NAN;
  int8_t* row = static_cast<int8_t*>(a.out) + t * a.ld_out;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if (!kept)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
    store_int8x8<VEC>(row, i, n, v[i], inverse);
  }
}

bool row_vectors(const void* p, int64_t ld, int dtype_size) {
  return p == nullptr || (aligned16(p) && (ld * dtype_size) % 16 == 0);
}

int size_of(int dtype) { return dtype == QCC_DTYPE_I8 ? 1 : dtype_bytes(dtype); }

bool norm_vectors(const qcc_norm_params& a) { return row_vectors(a.weight, 0, 1) && row_vectors(a.bias, 0, 1); }

template <typename T, typename R>
bool launch_block_norm(const BlockNormArgs& a, bool vec, cudaStream_t stream) {
  const int vecs = (a.hidden + 7) / 8;
  const int per = vecs <= 256 ? 1 : vecs <= 512 ? 2 : 4;
  const int threads = ((vecs + per - 1) / per + 31) / 32 * 32;
  const dim3 grid(static_cast<unsigned>(a.rows));
  clear_stale_error();
#define QCC_LAUNCH(V)                                                          \
  (vec ? block_norm_kernel<T, R, V, true><<<grid, threads, 0, stream>>>(a)     \
       : block_norm_kernel<T, R, V, false><<<grid, threads, 0, stream>>>(a))
  if (per == 1)
    QCC_LAUNCH(1);
  else if (per == 2)
    QCC_LAUNCH(2);
  else
    QCC_LAUNCH(4);
#undef QCC_LAUNCH
  return launch_ok();
}

bool valid_norm(const qcc_norm_params* p) {
  if (p == nullptr) return true;
  if (p->kind == QCC_NORM_NONE) return p->weight == nullptr && p->bias == nullptr;
  return (p->kind == QCC_NORM_RMS || p->kind == QCC_NORM_LAYER) &&
         ((p->weight == nullptr && p->bias == nullptr) || valid_dtype(p->dtype));
}

int run_block_norm(const BlockNormArgs& a, int dtype, int res_dtype, cudaStream_t stream) {
  const int es = dtype_bytes(dtype), rs = dtype_bytes(res_dtype);
  const bool vec = row_vectors(a.y, a.ldy, es) && row_vectors(a.res, a.ld_res, rs) &&
                   row_vectors(a.res_out, a.ld_res_out, rs) && norm_vectors(a.post) && norm_vectors(a.next) &&
                   (a.gate.cols == 1 || row_vectors(a.gate.values, a.gate.ld, dtype_bytes(a.gate.dtype))) &&
                   row_vectors(a.out, a.ld_out, size_of(a.out_dtype));
  bool ok;
  if (dtype == QCC_DTYPE_BF16)
    ok = res_dtype == QCC_DTYPE_F32 ? launch_block_norm<__nv_bfloat16, float>(a, vec, stream)
                                    : launch_block_norm<__nv_bfloat16, __nv_bfloat16>(a, vec, stream);
  else if (dtype == QCC_DTYPE_F16)
    ok = res_dtype == QCC_DTYPE_F32 ? launch_block_norm<__half, float>(a, vec, stream)
                                    : launch_block_norm<__half, __half>(a, vec, stream);
  else
    ok = launch_block_norm<float, float>(a, vec, stream);
  return ok ? QCC_OK : QCC_ERR_CUDA;
}

}  // namespace
}  // namespace qcc

extern "C" int qcc_norm_rows(const void* x, int64_t ldx, int dtype, int rows, int hidden, const qcc_norm_params* norm,
                             void* out, int64_t ld_out, int out_dtype, float* row_scale, cudaStream_t stream) {
  if (!qcc::valid_dtype(dtype) || !(qcc::valid_dtype(out_dtype) || out_dtype == QCC_DTYPE_I8)) return QCC_ERR_DTYPE;
  if (!qcc::valid_norm(norm)) return QCC_ERR_INVALID_ARGUMENT;
  if (rows < 0 || hidden < 1 || ldx < hidden || ld_out < hidden) return QCC_ERR_SHAPE;
  if (hidden > qcc::kMaxHidden) return QCC_ERR_UNSUPPORTED;
  if (rows == 0) return QCC_OK;
  if (x == nullptr || out == nullptr || (out_dtype == QCC_DTYPE_I8 && row_scale == nullptr))
    return QCC_ERR_INVALID_ARGUMENT;
  qcc::BlockNormArgs a = {};
  a.y = x;
  a.ldy = ldx;
  a.rows = rows;
  a.hidden = hidden;
  if (norm != nullptr) a.next = *norm;
  a.out = out;
  a.ld_out = ld_out;
  a.out_dtype = out_dtype;
  a.row_scale = row_scale;
  return qcc::run_block_norm(a, dtype, dtype, stream);
}

extern "C" int qcc_residual_norm(const void* branch, int64_t ld_branch, int dtype, const void* residual,
                                 int64_t ld_residual, int residual_dtype, int rows, int hidden,
                                 const qcc_norm_params* post, const qcc_gate_params* gate, float residual_scale,
                                 float branch_scale, void* residual_out, int64_t ld_residual_out,
                                 const qcc_norm_params* next, void* out, int64_t ld_out, int out_dtype,
                                 float* row_scale, cudaStream_t stream) {
  if (!qcc::valid_dtype(dtype) || !(residual_dtype == dtype || residual_dtype == QCC_DTYPE_F32)) return QCC_ERR_DTYPE;
  if (!qcc::valid_norm(post) || !qcc::valid_norm(next)) return QCC_ERR_INVALID_ARGUMENT;
  if (rows < 0 || hidden < 1 || ld_branch < hidden || ld_residual < hidden || ld_residual_out < hidden)
    return QCC_ERR_SHAPE;
  if (gate != nullptr) {
    if (!qcc::valid_dtype(gate->dtype)) return QCC_ERR_DTYPE;
    if (gate->act != QCC_GATE_NONE && gate->act != QCC_GATE_SIGMOID && gate->act != QCC_GATE_TANH)
      return QCC_ERR_INVALID_ARGUMENT;
    if (gate->rows_each < 1 || (gate->cols != 1 && gate->cols != hidden) || gate->ld < 0) return QCC_ERR_SHAPE;
  }
  if (out != nullptr) {
    if (!(qcc::valid_dtype(out_dtype) || out_dtype == QCC_DTYPE_I8)) return QCC_ERR_DTYPE;
    if (ld_out < hidden) return QCC_ERR_SHAPE;
    if (out_dtype == QCC_DTYPE_I8 && row_scale == nullptr) return QCC_ERR_INVALID_ARGUMENT;
  }
  if (hidden > qcc::kMaxHidden) return QCC_ERR_UNSUPPORTED;
  if (rows == 0) return QCC_OK;
  if (branch == nullptr || residual == nullptr || residual_out == nullptr ||
      (gate != nullptr && gate->values == nullptr))
    return QCC_ERR_INVALID_ARGUMENT;
  qcc::BlockNormArgs a = {};
  a.y = branch;
  a.ldy = ld_branch;
  a.res = residual;
  a.ld_res = ld_residual;
  a.rows = rows;
  a.hidden = hidden;
  a.residual_scale = residual_scale;
  a.branch_scale = branch_scale;
  if (post != nullptr) a.post = *post;
  if (next != nullptr) a.next = *next;
  if (gate != nullptr) a.gate = *gate;
  a.res_out = residual_out;
  a.ld_res_out = ld_residual_out;
  a.out = out;
  a.ld_out = ld_out;
  a.out_dtype = out == nullptr ? dtype : out_dtype;
  a.row_scale = row_scale;
  return qcc::run_block_norm(a, dtype, residual_dtype, stream);
}
