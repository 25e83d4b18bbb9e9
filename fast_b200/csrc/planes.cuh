// fp32 values as three bf16 planes x = x0 + x1 + x2: the leading 8 significant
// bits, the next 8, the last 8.  Cutting bits off is exact and cannot overflow.
//
// The products 00, 01, 02, 10, 11, 20 of two operands' planes are summed.  An
// infinity is kept as (+-1, +-1, +-inf): its plane 2 meets the other operand's
// plane 0 alone, which is zero only where the other value is.  As plane 0 it
// would also meet planes 1 and 2, which are zero for every value of few bits
// (1, 0.5), and 0 * inf would make a NaN of an infinite product.  Two
// infinities meet as +-inf times +-1.  A NaN is plane 0 alone.
#pragma once
#include "common.cuh"

namespace fbplanes {

// Plane 0 or 1 as fp32 bits, and what it leaves of x; what plane 1 leaves is
// plane 2.  FINITE: x is no infinity and no NaN (600 x 100 rows against 10,000
// nodes, training: 82 us with the general form for all values, 77 so).
struct Cut {
  uint32_t lead;
  float rest;
};
template <bool FINITE> __device__ __forceinline__ Cut cut(float x) {
  const uint32_t b = __float_as_uint(x), m = b & 0x7FFFFFFFu, lead = b & 0xFFFF0000u;
  if (FINITE || m < 0x7F800000u) return Cut{lead, x - __uint_as_float(lead)};
  return m == 0x7F800000u ? Cut{(b & 0x80000000u) | 0x3F800000u, x} : Cut{b | 0x00400000u, 0.f};
}
// Adds up to 0 over finite values, to NaN over others.
__device__ __forceinline__ float probe(float x, float sum) { return fmaf(x, 0.f, sum); }

struct Split {
  uint32_t b0, b1, b2;                        // b2's low half is cut on packing
};
template <bool FINITE> __device__ __forceinline__ Split split(float x) {
  const Cut c0 = cut<FINITE>(x), c1 = cut<FINITE>(c0.rest);
  return Split{c0.lead, c1.lead, __float_as_uint(c1.rest)};
}
__device__ __forceinline__ uint32_t pair(uint32_t lo, uint32_t hi) { return __byte_perm(lo, hi, 0x7632); }

// Four consecutive values to 8-byte aligned places `plane` elements apart.
template <bool FINITE>
__device__ __forceinline__ void put4_as(uint16_t *p, int64_t plane, float a, float b, float c, float d) {
  const Split s = split<FINITE>(a), t = split<FINITE>(b), u = split<FINITE>(c), v = split<FINITE>(d);
  *reinterpret_cast<uint2 *>(p) = make_uint2(pair(s.b0, t.b0), pair(u.b0, v.b0));
  *reinterpret_cast<uint2 *>(p + plane) = make_uint2(pair(s.b1, t.b1), pair(u.b1, v.b1));
  *reinterpret_cast<uint2 *>(p + 2 * plane) = make_uint2(pair(s.b2, t.b2), pair(u.b2, v.b2));
}
__device__ __forceinline__ void put4(uint16_t *p, int64_t plane, float a, float b, float c, float d) {
  if (probe(a, probe(b, probe(c, probe(d, 0.f)))) == 0.f) put4_as<true>(p, plane, a, b, c, d);
  else put4_as<false>(p, plane, a, b, c, d);
}

}  // namespace fbplanes
