// The gated block's activations: act(g) and act'(g).
#pragma once
#include "common.cuh"

namespace fbact {

enum : int { kSilu = FB_ACT_SILU, kGelu = FB_ACT_GELU, kRelu = FB_ACT_RELU };

// To a few ulp of fp32.
template <int ACT> __device__ __forceinline__ float2 act_exact(float g) {
  if (ACT == kSilu) {
    const float s = 1.f / (1.f + expf(-g));
    return make_float2(g * s, s * (1.f + g * (1.f - s)));
  }
  if (ACT == kGelu) {
    const float phi = 0.5f * (1.f + erff(g * 0.70710678118654752f));
    return make_float2(g * phi, phi + g * expf(-0.5f * g * g) * 0.39894228040143268f);
  }
  return make_float2(fmaxf(g, 0.f), g > 0.f ? 1.f : 0.f);
}

// With the hardware's fast exponential and division (2^-21 or so of the
// result): results that are rounded to bf16 next.
template <int ACT> __device__ __forceinline__ float2 act_fast(float g) {
  if (ACT == kSilu) {
    const float s = __fdividef(1.f, 1.f + __expf(-g));
    return make_float2(g * s, s * (1.f + g * (1.f - s)));
  }
  if (ACT == kGelu) {
    // normal distribution function by Abramowitz & Stegun 7.1.26 (erf to 1.5e-7): its exponential is the density's
    const float x = fabsf(g) * 0.70710678118654752f, e = __expf(-0.5f * g * g);
    const float t = __fdividef(1.f, fmaf(0.3275911f, x, 1.f));
    const float p = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.061405429f, -1.453152027f), 1.421413741f), -0.284496736f),
                             0.254829592f);
    const float q = 0.5f * p * e, phi = g >= 0.f ? 1.f - q : q;
    return make_float2(g * phi, fmaf(g * e, 0.39894228040143268f, phi));
  }
  return make_float2(fmaxf(g, 0.f), g > 0.f ? 1.f : 0.f);
}

}  // namespace fbact
