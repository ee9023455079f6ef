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

// The smallest e >= kMinBoxExp with amax <= 127 * 2^e, amax finite and >= 0; -7 for 0.
// amax = m 2^E with m in [0.5, 1): e = E - 7, and one more where m > 127 / 128, that is where
// the 23 bits below the leading one pass 0x7e0000.
__device__ __forceinline__ int box_exponent(float amax) {
  const unsigned u = __float_as_uint(amax);
  if (u == 0) return -7;
  const int e = static_cast<int>(u >> 23) - 126 - 7 + ((u & 0x7fffffu) > 0x7e0000u ? 1 : 0);
  return e < kMinBoxExp ? kMinBoxExp : e;  // subnormal ones too
}

}  // namespace step
}  // namespace fe
