// The gated block's activations: act(g) and act'(g).
#pragma once
#include "common.cuh"

namespace fbact {

enum : int { kSilu = FB_ACT_SILU, kGelu = FB_ACT_GELU, kRelu = FB_ACT_RELU };

// To a few ulp of fp32, of the result: GELU's normal distribution function is
// not 0.5 (1 + erf), which for g < 0 is a small difference of two ones (off by
// 2.7e-4 of itself at -4, zero from -5.5 on).  act' near its zero: a few ulp of
// its terms.
template <int ACT> __device__ __forceinline__ float2 act_exact(float g) {
  if (ACT == kSilu) {
    const float s = 1.f / (1.f + expf(-g));
    return make_float2(g * s, s * (1.f + g * (1.f - s)));
  }
  if (ACT == kGelu) {
    const float phi = normcdff(g);
    return make_float2(g * phi, phi + g * expf(-0.5f * g * g) * 0.39894228040143268f);
  }
  return make_float2(fmaxf(g, 0.f), g > 0.f ? 1.f : 0.f);
}

// With the hardware's fast exponential and division: results that are rounded
// to bf16 next.  2^-20 or so of the result, or of act's terms; GELU's
// exponential adds 2^-24 g^2.
template <int ACT> __device__ __forceinline__ float2 act_fast(float g) {
  if (ACT == kSilu) {
    const float s = __fdividef(1.f, 1.f + __expf(-g));
    return make_float2(g * s, s * (1.f + g * (1.f - s)));
  }
  if (ACT == kGelu) {
    // The normal distribution function of -|g| is 0.5 erfc(x), x = |g| / sqrt(2), and erfc(x) is the density's exponential
    // times a smooth function of t = 1 / (1 + 0.42 x): its polynomial of degree 8 without a constant, fitted (linear
    // program over 1,000 points) to the least relative error for x up to 9.6, where bf16's range ends: 5e-7 in fp32.
    // (A polynomial for erf, 1.5e-7 of one, was off by 1.6e-3 of the result at -5 and 1% at -8; 12,000 x 172 x 688 rows,
    // training: 90.3 us with it, 92.4 with this.)
    const float x = fabsf(g) * 0.70710678118654752f, e = __expf(-0.5f * g * g);
    const float t = __fdividef(1.f, fmaf(0.42f, x, 1.f));
    float p = fmaf(t, 0.06989795714616776f, -0.31880080699920654f);
    p = fmaf(t, p, 0.43804308772087097f);
    p = fmaf(t, p, -0.12798945605754852f);
    p = fmaf(t, p, 0.2673374116420746f);
    p = fmaf(t, p, 0.19517037272453308f);
    p = fmaf(t, p, 0.239512100815773f);
    p = t * fmaf(t, p, 0.23682916164398193f);
    const float q = 0.5f * p * e, phi = g >= 0.f ? 1.f - q : q;
    return make_float2(g * phi, fmaf(g * e, 0.39894228040143268f, phi));
  }
  return make_float2(fmaxf(g, 0.f), g > 0.f ? 1.f : 0.f);
}

}  // namespace fbact
