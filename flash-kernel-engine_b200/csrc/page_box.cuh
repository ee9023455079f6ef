// Exponents of the int8 page boxes, shared by the kernels that make and score them.
#pragma once

#include <cuda_runtime.h>

namespace fe {
namespace step {

constexpr int kMinBoxExp = -120;  // 2^-e and 2^e stay normal

__device__ __forceinline__ bool is_finite(float x) {
  return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u;
}
// 2^e for -126 <= e <= 127.
__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float((e + 127) << 23); }

// The smallest e >= kMinBoxExp with amax <= 127 * 2^e, amax finite and >= 0.
__device__ __forceinline__ int box_exponent(float amax) {
  int e;
  const float m = frexpf(amax, &e);  // amax = m 2^e, m in [0.5, 1), or 0 = 0 2^0
  e = e - 7 + (m > 127.f / 128.f ? 1 : 0);
  return e < kMinBoxExp ? kMinBoxExp : e;
}

}  // namespace step
}  // namespace fe
