// Shared helpers for the cueq_b200 kernels: error reporting, dtype-generic loads, atomics.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdarg>
#include <cstdint>
#include <cstdio>

#include "../../include/cueq_b200.h"

namespace cueq {

// thread-local message returned by cueq_b200_last_error()
char* error_buffer();
int fail(const char* fmt, ...);

#define CUEQ_CUDA_OK(expr)                                                        \
  do {                                                                            \
    cudaError_t e__ = (expr);                                                     \
    if (e__ != cudaSuccess)                                                       \
      return ::cueq::fail("%s failed: %s", #expr, cudaGetErrorString(e__));       \
  } while (0)

static inline int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// One flag per device ordinal.  Function attributes such as the dynamic shared-memory limit
// belong to the device that was current when they were set, so a launcher that has configured
// its kernel on one GPU still has to do it on the next GPU the same process uses.
struct PerDeviceFlag {
  static constexpr int kMax = 64;
  bool done[kMax] = {};
  static int current() {
    int d = -1;
    return cudaGetDevice(&d) == cudaSuccess ? d : -1;
  }
  bool get() const {
    const int d = current();
    return d >= 0 && d < kMax && done[d];
  }
  void set() {
    const int d = current();
    if (d >= 0 && d < kMax) done[d] = true;
  }
};

// Load one element of a buffer whose element type is only known at run time.
template <typename M>
__device__ __forceinline__ M load_as(const void* p, int dtype, int64_t i) {
  switch (dtype) {
    case CUEQ_F32: return (M)__ldg(reinterpret_cast<const float*>(p) + i);
    case CUEQ_F64: return (M)__ldg(reinterpret_cast<const double*>(p) + i);
    case CUEQ_BF16: return (M)__bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
    default: return (M)__half2float(reinterpret_cast<const __half*>(p)[i]);
  }
}

__device__ __forceinline__ int64_t load_index(const void* idx, int is64, int64_t z) {
  return is64 ? __ldg(reinterpret_cast<const long long*>(idx) + z)
              : (int64_t)__ldg(reinterpret_cast<const int*>(idx) + z);
}

// Activations kept in 8 bits: code = rint(v / step), step the smallest power of two (at least 2^-126) of which 127 hold the block's
// largest magnitude.  A power of two costs at most one of the seven bits, code * step is exact in bf16 and TF32, and no code depends on
// how a quotient is rounded.  `top`: bits of the largest magnitude, 127 = 1.984375 * 2^6; an infinity or NaN: step NaN, codes 0.
__device__ __forceinline__ void code_step(unsigned top, float& step, float& inverse) {
  if (top >= 0x7f800000u) { step = __uint_as_float(0x7fc00000u); inverse = 0.f; return; }
  int k = (int)(top >> 23) - 6 + ((top & 0x7fffffu) > 0x7e0000u ? 1 : 0);
  k = k < 1 ? 1 : k;
  step = __uint_as_float((unsigned)k << 23);
  inverse = __uint_as_float((unsigned)(254 - k) << 23);
}
__device__ __forceinline__ signed char to_code(float v, float inverse) { return (signed char)__float2int_rn(v * inverse); }

template <typename M>
__device__ __forceinline__ M warp_sum(M v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

}  // namespace cueq
