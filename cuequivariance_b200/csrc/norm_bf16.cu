// The norm kernels of one element type (norm_kernels.cuh).
#include "norm_kernels.cuh"

cueq_norm::Kernel cueq_norm::pick_bf16(int mode, bool mul_ir, bool backward) { return pick<__nv_bfloat16, float, false>(mode, mul_ir, backward); }
