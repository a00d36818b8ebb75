// Block norms of f16 rows.
#include "block_norm.cuh"

namespace qcc {

bool block_norm_f16(const BlockNormArgs& a, int res_dtype, bool quantize, int device, cudaStream_t stream) {
  using T = __half;
  constexpr int kType = QCC_DTYPE_F16;
  if (quantize) return launch_rows<T, T, kQuantize>(a, kType, kType, device, stream);
  if (a.res == nullptr) return launch_rows<T, T, kNorm>(a, kType, kType, device, stream);
  return res_dtype == QCC_DTYPE_F32 ? launch_rows<T, float, kJoin>(a, kType, res_dtype, device, stream)
                                    : launch_rows<T, T, kJoin>(a, kType, res_dtype, device, stream);
}

}  // namespace qcc
