// The norm kernels of one element type (norm_kernels.cuh); a file each, so that they compile side by side.
#include "norm_kernels.cuh"

cueq_norm::Kernel cueq_norm::pick_f32(int mode, bool q8, bool mul_ir, bool backward) { return pick<float, float>(mode, q8, mul_ir, backward); }
