// Block norms of fp32 rows.
#include "block_norm.cuh"

namespace qcc {

bool block_norm_f32(const BlockNormArgs& a, bool quantize, int device, cudaStream_t stream) {
  constexpr int kType = QCC_DTYPE_F32;
  if (quantize) return launch_rows<float, float, kQuantize>(a, kType, kType, device, stream);
  if (a.res != nullptr) return launch_rows<float, float, kJoin>(a, kType, kType, device, stream);
  // The 16-bit type of the parameters or of the output, where there is one.
  const auto any = [&](int type) { return a.out_dtype == type || a.next.dtype == type; };
  if (any(QCC_DTYPE_BF16)) return launch_rows<float, __nv_bfloat16, kNorm>(a, kType, kType, device, stream);
  if (any(QCC_DTYPE_F16)) return launch_rows<float, __half, kNorm>(a, kType, kType, device, stream);
  return launch_rows<float, float, kNorm>(a, kType, kType, device, stream);
}

}  // namespace qcc
