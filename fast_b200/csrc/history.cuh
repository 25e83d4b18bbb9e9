// Packed histories: rows of several sequences one after the other.  Sequence s
// takes rows starts[s] .. starts[s + 1] - 1; it may be empty.  Rows in front
// of starts[0] and from starts[S] on belong to none.
//
// What the device holds in `starts` is not checked on the host.  Every index
// made from it is clamped to the rows and sequences of the call, so values out
// of order give wrong sums and no access out of range.
#pragma once
#include <cuda_bf16.h>
#include "common.cuh"

namespace fbq {

using bf16 = __nv_bfloat16;

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f<bf16>(bf16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16 from_f<bf16>(float v) { return __float2bfloat16_rn(v); }

// V elements of T as one aligned memory access.
template <typename T, int V> struct alignas(sizeof(T) * V) Vec {
  T e[V];
};

// Whether every pointer given (null: none) lies at a multiple of `bytes`, a power of two.
template <typename... P> bool aligned(uintptr_t bytes, P... p) { return ((reinterpret_cast<uintptr_t>(p) | ...) & (bytes - 1)) == 0; }

struct Starts {
  const void *p;             // null: one sequence over all rows
  int wide;                  // 64-bit entries
  int seqs;
  int64_t rows;
  __device__ __forceinline__ int64_t operator[](int s) const {
    if (!p) return s > 0 ? rows : 0;
    const int64_t v = wide ? static_cast<const int64_t *>(p)[s] : static_cast<const int32_t *>(p)[s];
    return v < 0 ? 0 : (v > rows ? rows : v);
  }
};

// Sequence of a row: the last s in [0, seqs] with starts[s] <= row; -1 in front
// of them all, seqs behind them all.  The whole warp takes part; 32 probes a
// round, so 1,024 sequences take two dependent loads.
__device__ __forceinline__ int owner(const Starts &st, int64_t row) {
  if (!st.p) return row < 0 ? -1 : (row < st.rows ? 0 : 1);
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = st.seqs + 1;                        // starts[lo - 1] <= row < starts[hi]
  while (hi > lo) {
    const int step = (hi - lo + 31) >> 5, i = lo + lane * step;
    const int c = __popc(__ballot_sync(0xffffffffu, i < hi && st[i] <= row));
    if (c == 0) break;
    const int next = lo + c * step;
    lo = next - step + 1;
    hi = next < hi ? next : hi;
  }
  return lo - 1;
}

// Walks the rows' boundaries upwards, kTile rows at a time.
constexpr int kTile = 8;
struct Walk {
  int next;                  // first entry of starts that may lie behind the current tile's first row
  int base;                  // the lanes' entries of the last tile: starts[base + lane]
  int64_t entry;
  bool all;                  // they are all of the tile's
  __device__ __forceinline__ void begin(const Starts &st, int64_t row) { next = owner(st, row - 1) + 1; }
  // Bit i: row r0 + i begins a sequence (or is the first behind the last one).
  __device__ __forceinline__ unsigned tile(const Starts &st, int64_t r0) {
    unsigned bits = 0;
    const int lane = threadIdx.x & 31;
    if (!st.p) return (r0 == 0 ? 1u : 0u) | (st.rows >= r0 && st.rows < r0 + kTile ? 1u << (st.rows - r0) : 0u);
    for (all = true;; all = false) {
      base = next;
      const int i = next + lane;
      const int64_t b = entry = i <= st.seqs ? st[i] : INT64_MAX;
      const bool in = b < r0 + kTile;
      bits |= __reduce_or_sync(0xffffffffu, in && b >= r0 ? 1u << (int)(b - r0) : 0u);
      const int c = __popc(__ballot_sync(0xffffffffu, in));
      next += c;
      if (c < 32) return bits;
    }
  }
  // owner() of a row of the tile or of the one in front of it, without a load where the lanes hold the tile's entries.
  __device__ __forceinline__ int sequence(const Starts &st, int64_t row) const {
    if (!st.p || !all) return owner(st, row);
    return base + __popc(__ballot_sync(0xffffffffu, entry <= row)) - 1;
  }
};

// The same, downwards: the first tile asked for holds row `top`, the next ones
// lie 8 rows lower each.
struct WalkDown {
  int next;                  // last entry of starts that may lie in the next tile
  int base;                  // the lanes' entries of the last tile: starts[base - lane]
  int64_t entry;
  bool all;                  // they are all of the tile's
  __device__ __forceinline__ void begin(const Starts &st, int64_t top) { next = owner(st, top); }
  __device__ __forceinline__ unsigned tile(const Starts &st, int64_t r0) {
    if (!st.p) return r0 == 0 ? 1u : 0u;
    unsigned bits = 0;
    const int lane = threadIdx.x & 31;
    for (all = true;; all = false) {
      base = next;
      const int i = next - lane;
      const int64_t b = entry = i >= 0 ? st[i] : -1;
      const bool in = b >= r0;
      bits |= __reduce_or_sync(0xffffffffu, in && b < r0 + kTile ? 1u << (int)(b - r0) : 0u);
      const int c = __popc(__ballot_sync(0xffffffffu, in));
      next -= c;
      if (c < 32) return bits;
    }
  }
  __device__ __forceinline__ int sequence(const Starts &st, int64_t row) const {
    if (!st.p || !all) return owner(st, row);
    return base - __popc(__ballot_sync(0xffffffffu, entry > row));
  }
};

// ---- pairs of fp32 values, one instruction for both ------------------------------------------------
struct F2 {
  unsigned long long v;
};
__device__ __forceinline__ F2 pack(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpack(F2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

// ---- functions of one value ------------------------------------------------------------------------
constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ F2 ex2_2(F2 x) {
  const float2 f = unpack(x);
  return pack(ex2(f.x), ex2(f.y));
}
__device__ __forceinline__ float rcp(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ F2 both(float a) { return pack(a, a); }
__device__ __forceinline__ F2 rcp_2(F2 x) {
  const float2 f = unpack(x);
  return pack(rcp(f.x), rcp(f.y));
}
// The smaller and the larger one, NaN if there is one.
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// A log2(e), kept finite so that a row of no sequence (dt 0) leaves the state as it
// is even where A is -infinity.
__device__ __forceinline__ float scaled(float A) { return max_nan(A * kLog2e, -3e38f); }
// exp(dt A) of a pair, A2 = scaled(A).  The exponential unit's results are low by
// 0.6 to 2.4e-8 on average where decays are slow (measured for exponents of -1e-4
// to -1), which a state that remembers a thousand steps adds up a thousand
// times; the summand centres them.
__device__ __forceinline__ F2 decays(F2 dt, F2 A2) { return ex2_2(fma2(dt, A2, both(2e-8f))); }

// What t = -m log2(e), rounded, lacks: m log2(e) + t.
__device__ __forceinline__ F2 exponent_rest2(F2 m, F2 t) {
  return fma2(m, both(1.925963033500011e-8f), fma2(m, both(kLog2e), t));
}

// log(1 + e^x) of a pair and (SLOPE) its derivative, relative accuracy a few
// 2^-24 also where they are small.  With e = e^-|x|: log(1 + e) = 2 artanh(s), s =
// e / (2 + e) <= 1/3, and artanh(s) / s is a polynomial in s^2 (interpolated at
// Chebyshev nodes of [0, 1/9], off by 4e-9).  The product |x| log2(e) is carried
// to two words: its rounding alone would cost e 2^-24 |x|.  Below x = -87.3 e is
// flushed to 0.
template <bool SLOPE> __device__ __forceinline__ F2 softplus2(F2 x, F2 &slope) {
  const float2 f = unpack(x);
  const F2 m = pack(fminf(fabsf(f.x), 100.f), fminf(fabsf(f.y), 100.f));
  const F2 t = mul2(m, both(-kLog2e));
  F2 e = ex2_2(t);
  e = fma2(mul2(exponent_rest2(m, t), both(-0.6931472f)), e, e);
  const F2 s = mul2(e, rcp_2(add2(e, both(2.f)))), w = mul2(s, s);
  F2 p = fma2(w, both(0.14078889787197113f), both(0.13982579112052917f));
  p = fma2(w, p, both(0.20012298226356506f));
  p = fma2(w, p, both(0.3333316147327423f));
  const F2 s2 = add2(s, s), l = fma2(mul2(w, p), s2, s2);
  if constexpr (SLOPE) {
    const float2 r = unpack(rcp_2(add2(e, both(1.f)))), er = unpack(mul2(e, pack(r.x, r.y)));
    slope = pack(f.x >= 0.f ? r.x : er.x, f.y >= 0.f ? r.y : er.y);
  }
  return add2(l, pack(max_nan(f.x, 0.f), max_nan(f.y, 0.f)));
}
__device__ __forceinline__ float softplus(float x) {
  F2 none;
  return unpack(softplus2<false>(both(x), none)).x;
}

// 1 / (1 + e^-x) of a pair in rows of type T, and what it leaves to 1.  For fp32
// rows both keep their relative accuracy, a few 2^-24, where they are small: the
// product x log2(e) is carried to two words, as in softplus2, and the rest is e^-x
// times the first.  x is held to where no step overflows; below -87.3 the sigmoid
// is flushed to 0.  For bf16 rows, whose results are rounded to 2^-8, one word does
// (|x| 2^-24 off), and nothing asks for the rest.
template <typename T> __device__ __forceinline__ F2 sigmoid2(F2 x, F2 &rest) {
  if constexpr (sizeof(T) == 4) {
    const float2 f = unpack(x);
    const F2 m = pack(min_nan(max_nan(f.x, -88.f), 100.f), min_nan(max_nan(f.y, -88.f), 100.f)), t = mul2(m, both(-kLog2e));
    F2 e = ex2_2(t);
    e = fma2(mul2(exponent_rest2(m, t), both(-0.6931472f)), e, e);
    const F2 sg = rcp_2(add2(e, both(1.f)));
    rest = mul2(e, sg);
    return sg;
  } else {
    return rcp_2(add2(ex2_2(mul2(x, both(-kLog2e))), both(1.f)));
  }
}
template <typename T> __device__ __forceinline__ float sigmoid(float x, float &rest) {
  if constexpr (sizeof(T) == 4) {
    const float m = min_nan(max_nan(x, -88.f), 100.f), t = __fmul_rn(m, -kLog2e);
    float e = ex2(t);
    e = fmaf(fmaf(m, 1.925963033500011e-8f, fmaf(m, kLog2e, t)) * -0.6931472f, e, e);
    const float sg = rcp(1.f + e);
    rest = e * sg;
    return sg;
  } else {
    const float sg = rcp(1.f + ex2(-kLog2e * x));
    rest = 1.f - sg;
    return sg;
  }
}
template <typename T> __device__ __forceinline__ float sigmoid(float x) {
  float rest;
  return sigmoid<T>(x, rest);
}

// The derivative of x sigmoid(x) from the sigmoid and its rest: sg (1 + x (1 - sg)).
// Written out, sg + x sg - x sg^2, it cancels for large x, by |x| 2^-24.  For bf16
// rows that is what fits between the loads best (convolution backward of 32,768 x
// 2,048: 121 us, with the difference from 1 124 to 131), so there x ends at 64, where
// the sigmoid is 1.
template <typename T> __device__ __forceinline__ F2 silu_slope2(F2 x, F2 sg, F2 rest) {
  if constexpr (sizeof(T) == 4) return mul2(sg, fma2(x, rest, both(1.f)));
  const float2 f = unpack(x);
  const F2 xs = mul2(pack(fminf(f.x, 64.f), fminf(f.y, 64.f)), sg);
  return fma2(mul2(xs, sg), both(-1.f), add2(sg, xs));
}

}  // namespace fbq
