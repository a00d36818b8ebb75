// The block norms' entry points: checks, and the kernels of the rows' type.
#include "block_norm.h"

#include "qcc_host.h"

namespace qcc {
namespace {

constexpr int kMaxHidden = 32768;
constexpr int kMaxQuantized = 131071;  // rows as they are to int8: the widest that the int8 products take

bool element_aligned(const void* p, int es) { return reinterpret_cast<uintptr_t>(p) % es == 0; }

bool valid_norm(const qcc_norm_params* p) {
  if (p == nullptr) return true;
  if (p->kind == QCC_NORM_NONE) return p->weight == nullptr && p->bias == nullptr;
  return (p->kind == QCC_NORM_RMS || p->kind == QCC_NORM_LAYER) &&
         ((p->weight == nullptr && p->bias == nullptr) || valid_dtype(p->dtype));
}

bool norm_aligned(const qcc_norm_params& p) {
  const int es = dtype_bytes(p.dtype);
  return element_aligned(p.weight, es) && element_aligned(p.bias, es);
}

int run_block_norm(const BlockNormArgs& a, int dtype, int res_dtype, cudaStream_t stream) {
  if (!element_aligned(a.y, dtype_bytes(dtype)) || !element_aligned(a.res, dtype_bytes(res_dtype)) ||
      !element_aligned(a.res_out, dtype_bytes(res_dtype)) || !norm_aligned(a.post) || !norm_aligned(a.next) ||
      (a.gate.values != nullptr && !element_aligned(a.gate.values, dtype_bytes(a.gate.dtype))) ||
      (a.out_dtype != QCC_DTYPE_I8 && !element_aligned(a.out, dtype_bytes(a.out_dtype))) ||
      !element_aligned(a.row_scale, 4))
    return QCC_ERR_ALIGNMENT;
  int device = 0;
  if (!cuda_ok(cudaGetDevice(&device))) return QCC_ERR_CUDA;
  const bool quantize = a.res == nullptr && a.out_dtype == QCC_DTYPE_I8 && a.next.kind == QCC_NORM_NONE;
  const bool ok = dtype == QCC_DTYPE_BF16  ? block_norm_bf16(a, res_dtype, quantize, device, stream)
                  : dtype == QCC_DTYPE_F16 ? block_norm_f16(a, res_dtype, quantize, device, stream)
                                           : block_norm_f32(a, quantize, device, stream);
  return ok ? QCC_OK : QCC_ERR_CUDA;
}

}  // namespace
}  // namespace qcc

extern "C" int qcc_norm_rows(const void* x, int64_t ldx, int dtype, int rows, int hidden, const qcc_norm_params* norm,
                             void* out, int64_t ld_out, int out_dtype, float* row_scale, cudaStream_t stream) {
  if (!qcc::valid_dtype(dtype) || !(qcc::valid_dtype(out_dtype) || out_dtype == QCC_DTYPE_I8)) return QCC_ERR_DTYPE;
  if (!qcc::valid_norm(norm)) return QCC_ERR_INVALID_ARGUMENT;
  if (rows < 0 || hidden < 1 || ldx < hidden || ld_out < hidden) return QCC_ERR_SHAPE;
  const bool as_is = out_dtype == QCC_DTYPE_I8 && (norm == nullptr || norm->kind == QCC_NORM_NONE);
  if (hidden > (as_is ? qcc::kMaxQuantized : qcc::kMaxHidden)) return QCC_ERR_UNSUPPORTED;
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
