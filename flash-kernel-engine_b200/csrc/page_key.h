// Keys of the pages' scores, in whose order sparse_decode.cu chooses pages. Plain C++, so that
// a host program can go through them too.
#pragma once

#include <cuda_runtime.h>
#include <string.h>

namespace fe {
namespace step {

constexpr unsigned kForced = 0xffffffffu;  // key of an always-chosen page, above every score
constexpr float kInf = __builtin_huge_valf();

// Key of a page with the largest sum `best` of a query head and the scale `sc`: the score
// best * sc in an order-preserving map of the float to 32 bits, -0 as 0, and always strictly
// between 0 (no page) and kForced. +inf for a page with the scale +inf, which has a key that
// is not finite, and where there is no number (a scale that nobody wrote, say): a NaN's own
// bits could be kForced, and more pages than are kept would then count as always chosen.
__host__ __device__ __forceinline__ unsigned page_key(float best, float sc) {
  float x = best * sc + 0.f;
  if (sc == kInf || x != x) x = kInf;
  unsigned u;
  memcpy(&u, &x, 4);
  return u ^ (static_cast<unsigned>(static_cast<int>(u) >> 31) | 0x80000000u);
}

}  // namespace step
}  // namespace fe
