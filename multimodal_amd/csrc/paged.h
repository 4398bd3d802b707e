// paged.h — what the kernels of the paged key-value cache share (paged_attention.hip, paged_pages.hip).
#pragma once
#include "common.h"

namespace mmamd {

// Division of a 32-bit number by a constant that is known at launch (Granlund & Montgomery 1994, "Division by invariant integers using
// multiplication", figure 4.1): exact for every n, two shifts and one high product where a page size need not be a power of two.
struct FastDiv {
  uint32_t d, mul;
  int sh1, sh2;
};
inline FastDiv fast_div(uint32_t d) {
  int l = 0;
  while (l < 32 && (1ull << l) < d) ++l;
  FastDiv f;
  f.d = d;
  f.mul = (uint32_t)(((1ull << 32) * ((1ull << l) - d)) / d + 1);
  f.sh1 = l < 1 ? l : 1;
  f.sh2 = l > 1 ? l - 1 : 0;
  return f;
}
__host__ __device__ __forceinline__ uint32_t div_by(const FastDiv& f, uint32_t n) {
  const uint32_t t = (uint32_t)(((uint64_t)f.mul * n) >> 32);
  return (t + ((n - t) >> f.sh1)) >> f.sh2;
}

__device__ __forceinline__ int clamp_int(int v, int lo, int hi) { return v < lo ? lo : (v > hi ? hi : v); }

}  // namespace mmamd
