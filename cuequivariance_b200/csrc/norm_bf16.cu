// The norm kernels of one element type (norm_kernels.cuh); a file each, so that they compile side by side.
#include "norm_kernels.cuh"

cueq_norm::Kernel cueq_norm::pick_bf16(int mode, bool q8, bool backward) {
  return q8 ? pick<__nv_bfloat16, float, true>(mode, backward) : pick<__nv_bfloat16, float, false>(mode, backward);
}
