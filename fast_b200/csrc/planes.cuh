// fp32 values as three bf16 planes x = x0 + x1 + x2: the leading 8 significant
// bits, the next 8, the last 8.  Cutting bits off is exact and cannot
// overflow; x0 of an infinity or NaN carries it alone.
#pragma once
#include "common.cuh"

namespace fbplanes {

struct Split {
  uint32_t b0, b1, b2;                        // fp32 bits of the planes (low halves zero; b2's are cut on packing)
};
// What a plane leaves of x; `first`: x may be an infinity or NaN, which leaves nothing.
__device__ __forceinline__ float rest(float x, bool first) {
  const uint32_t b = __float_as_uint(x) & 0xFFFF0000u;
  return first && (b & 0x7F800000u) == 0x7F800000u ? 0.f : x - __uint_as_float(b);
}
__device__ __forceinline__ Split split(float x) {
  const float r1 = rest(x, true);
  return Split{__float_as_uint(x) & 0xFFFF0000u, __float_as_uint(r1) & 0xFFFF0000u, __float_as_uint(rest(r1, false))};
}
__device__ __forceinline__ uint32_t pair(uint32_t lo, uint32_t hi) { return __byte_perm(lo, hi, 0x7632); }

// Four consecutive values to 8-byte aligned places `plane` elements apart.
__device__ __forceinline__ void put4(uint16_t *p, int64_t plane, float a, float b, float c, float d) {
  const Split s = split(a), t = split(b), u = split(c), v = split(d);
  *reinterpret_cast<uint2 *>(p) = make_uint2(pair(s.b0, t.b0), pair(u.b0, v.b0));
  *reinterpret_cast<uint2 *>(p + plane) = make_uint2(pair(s.b1, t.b1), pair(u.b1, v.b1));
  *reinterpret_cast<uint2 *>(p + 2 * plane) = make_uint2(pair(s.b2, t.b2), pair(u.b2, v.b2));
}

}  // namespace fbplanes
