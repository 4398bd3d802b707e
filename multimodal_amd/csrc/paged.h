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

// 16-byte pieces past the caches.  A copy's stores: left in the L2, its lines are written back when the kernel ends, which waits for them (36 MB moved within a
// pool: 21.7 us a call with ordinary stores, 11.3 with these; 240 MB: 64.0 and 48.6).
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
__device__ __forceinline__ uint4 load_past(const void* at) { return __builtin_bit_cast(uint4, __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(at))); }
__device__ __forceinline__ void store_past(void* at, const uint4& v) { __builtin_nontemporal_store(__builtin_bit_cast(u32x4, v), reinterpret_cast<u32x4*>(at)); }

__device__ __forceinline__ int clamp_int(int v, int lo, int hi) { return v < lo ? lo : (v > hi ? hi : v); }

}  // namespace mmamd
