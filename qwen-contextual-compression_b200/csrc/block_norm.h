// One launch of the block norms, and its entry point for each type of rows.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "qcc_b200.h"

namespace qcc {

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
  int shift0;             // elements of row 0 before its first 16-byte boundary's granule, 0..7
  bool gate_in_granules;  // the gate's rows, in the branch's type, share its granules
  float inv_hidden;       // 1 / hidden
  uint64_t wait_ns;       // bound of the ring's waits for its copies
};

// Rows of one type; res_dtype as the residual's type in a join (a.res not NULL), quantize: rows as they are to int8.
bool block_norm_bf16(const BlockNormArgs& a, int res_dtype, bool quantize, int device, cudaStream_t stream);
bool block_norm_f16(const BlockNormArgs& a, int res_dtype, bool quantize, int device, cudaStream_t stream);
bool block_norm_f32(const BlockNormArgs& a, bool quantize, int device, cudaStream_t stream);

}  // namespace qcc
