// The norm kernels of one element type (norm_kernels.cuh), activations kept in 8 bits.
#include "norm_kernels.cuh"

cueq_norm::Kernel cueq_norm::pick_f32_codes(int mode, bool mul_ir, bool backward) { return pick<float, float, true>(mode, mul_ir, backward); }
