// The norm kernels of one element type (norm_kernels.cuh).
#include "norm_kernels.cuh"

cueq_norm::Kernel cueq_norm::pick_f64(int mode, bool mul_ir, bool backward) { return pick<double, double, false>(mode, mul_ir, backward); }
