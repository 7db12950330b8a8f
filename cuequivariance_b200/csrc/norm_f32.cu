// The norm kernels of one element type (norm_kernels.cuh).
#include "norm_kernels.cuh"

cueq_norm::Kernel cueq_norm::pick_f32(int mode, bool mul_ir, bool backward) { return pick<float, float, false>(mode, mul_ir, backward); }
