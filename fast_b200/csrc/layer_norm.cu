// Layer norm over rows of fp32 or bf16, forward and backward, with the
// residual sum in front of it and the reduction of the weight's gradient.
//
//   s = x + res (kept, rounded to the rows' type; s = x without res)
//   mean = sum(s) / D,  rstd = 1 / sqrt(sum((s - mean)^2) / D + eps)
//   y = (s - mean) rstd gamma + beta
//   a = dy gamma,  xhat = (s - mean) rstd
//   ds_in = rstd (a - mean(a) - xhat mean(a xhat)) (+ ds)
//   dgamma = sum_rows dy xhat,  dbeta = sum_rows dy
//
// A row is read once and held in registers (32 bytes of each operand a
// thread), so the variance is the exact two-pass one.  G threads share a row
// (G = 8 .. 1024, the smallest that hold it) and a CTA of at least 256 threads
// works on 256 / G rows at once.  The grid is a fixed number of CTAs per SM
// that walk the rows: gamma and beta stay in shared memory as fp32 (registers
// are what limits the rows in flight), and a row's loads are
// issued before the row ahead of it is reduced, which keeps memory busy
// through the reductions.  Rows of 2 KB and more with 16-byte aligned operands
// (BULK) come by bulk copies into a ring of rows in shared memory instead, up
// to kRing bytes ahead of the row in work (backward of 16,384 x 4,096 bf16 rows
// with a residual: 185 us by register prefetch, 112 by the ring).  The forward's
// ring and registers are small enough for four CTAs an SM: what is left is the
// latency of a row's two reductions, and more rows in work cover it (88 us for
// the same rows, 6.1 TB/s; 99 us with a ring of 64 KB and two CTAs).  Elements move in the widest power-of-two groups (up
// to 16 bytes) that every operand's base, pitch and width allow.  All sums are
// fp32.
//
// Backward keeps dgamma / dbeta partials of a CTA's rows in registers (in
// shared memory for G = 1024, where registers would spill), writes one
// partial row per CTA and a second kernel adds them in a fixed order, so
// results repeat bit for bit.  Up to kFusedElems elements it runs as one
// cluster of at most eight CTAs, which add their partials themselves behind a
// cluster barrier: one launch less where launches are what a call costs
// (forward and backward of 64 x 1,024 bf16 rows 17.2 us with a second
// launch, 14.9 so).
#include <cuda_bf16.h>
#include <algorithm>
#include "runtime.cuh"
#include "tc_common.cuh"

namespace {

using bf16 = __nv_bfloat16;

constexpr int kMaxD = 16384;
constexpr size_t kSmemSm = 228 * 1024, kSmemCta = 227 * 1024 - 1024;   // shared memory of an SM; dynamic, of a CTA
template <int G> __host__ __device__ constexpr int threads_of() { return G < 256 ? 256 : G; }

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

// Elements of a group as floats and back; bf16 in pairs.
template <typename T, int V> __device__ __forceinline__ void unpack(float (&o)[V], const Vec<T, V> &v) {
  if constexpr (sizeof(T) == 2 && V > 1) {
    const uint32_t *w = reinterpret_cast<const uint32_t *>(v.e);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      o[2 * i] = __uint_as_float(w[i] << 16);
      o[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] = to_f(v.e[e]);
  }
}
template <typename T, int V> __device__ __forceinline__ void pack(Vec<T, V> &v, const float (&o)[V]) {
  if constexpr (sizeof(T) == 2 && V > 1) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i)
      reinterpret_cast<__nv_bfloat162 *>(v.e)[i] = __floats2bfloat162_rn(o[2 * i], o[2 * i + 1]);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) v.e[e] = from_f<T>(o[e]);
  }
}

// Rows on their way into shared memory: `stages` stages of R rows of each of
// `ops` operands, filled by bulk copies that thread 0 issues.  A stage is
// consumed into registers before a CTA barrier, after which it is refilled, so
// it needs no second barrier.
constexpr int kRing = 32 * 1024;
constexpr int kMaxStages = 8;
struct Ring {
  uint8_t *base;
  uint64_t *full;
  volatile int *abort_flag;
  int32_t *err;
  int stages, ops, row_bytes;
};
__device__ __forceinline__ void bulk_load(void *dst, const void *src, uint32_t bytes, uint64_t *bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   fbtc::smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(fbtc::smem_u32(bar))
               : "memory");
}
// Thread 0: rows r0 .. r0 + R - 1 (those below n) of each operand into stage s.
template <typename T, int R, int OPS>
__device__ __forceinline__ void fill(const Ring &g, int s, const T *const (&p)[OPS], const int64_t (&ld)[OPS],
                                     int64_t r0, int64_t n) {
  const int rows = (int)min((int64_t)R, n - r0);
  if (rows <= 0) return;
  fbtc::mbar_expect_tx(g.full + s, (uint32_t)(rows * g.ops * g.row_bytes));
  for (int o = 0; o < g.ops; ++o)
    for (int q = 0; q < rows; ++q)
      bulk_load(g.base + ((s * g.ops + o) * R + q) * g.row_bytes, p[o] + (r0 + q) * ld[o], g.row_bytes, g.full + s);
}
// Time for copies in flight to land before the CTA's shared memory goes away (after a wait that ran out).
__device__ __forceinline__ void let_land() {
  const long long t0 = clock64();
  while (clock64() - t0 < 4000000) {
  }
}
// This thread's groups of operand o, row `sub` of stage s.
template <typename T, int V, int G, int R, int C>
__device__ __forceinline__ void from_ring(Vec<T, V> (&x)[C], const Ring &g, int s, int o, int sub, int t, int D) {
  const T *p = reinterpret_cast<const T *>(g.base + ((s * g.ops + o) * R + sub) * g.row_bytes);
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int i = (c * G + t) * V;
    if (i < D) x[c] = *reinterpret_cast<const Vec<T, V> *>(p + i);
    else
#pragma unroll
      for (int e = 0; e < V; ++e) x[c].e[e] = T(0.f);
  }
}

// This thread's C groups of a row (group c at column (c G + t) V; none at or past D).
template <typename T, int V, int G, int C>
__device__ __forceinline__ void load_row(Vec<T, V> (&o)[C], const void *base, int64_t at, int t, int D, bool live) {
  const T *p = static_cast<const T *>(base) + at;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int i = (c * G + t) * V;
    if (live && i < D) o[c] = *reinterpret_cast<const Vec<T, V> *>(p + i);
    else
#pragma unroll
      for (int e = 0; e < V; ++e) o[c].e[e] = T(0.f);
  }
}

// A parameter vector as fp32 in shared memory (`none` without one), by the
// whole CTA.  Groups of 8 are kept as two halves of the vector, so that the
// lanes' 16-byte reads lie side by side.
template <int V> __device__ __forceinline__ int param_at(int i, int D) {
  return V == 8 ? (i >> 3) * 4 + (i & 3) + ((i >> 2) & 1) * (D / 2) : i;
}
template <typename T, int V>
__device__ __forceinline__ void stage_param(float *o, const void *p, int wide, int D, float none) {
  for (int i = threadIdx.x; i < D; i += blockDim.x)
    o[param_at<V>(i, D)] = !p ? none : (wide ? static_cast<const float *>(p)[i] : to_f(static_cast<const T *>(p)[i]));
}
template <int V> __device__ __forceinline__ void group(float (&o)[V], const float *p, int i, int D) {
  if constexpr (V == 8) {
    *reinterpret_cast<float4 *>(o) = *reinterpret_cast<const float4 *>(p + i / 2);
    *reinterpret_cast<float4 *>(o + 4) = *reinterpret_cast<const float4 *>(p + i / 2 + D / 2);
  } else if constexpr (V == 4) {
    *reinterpret_cast<float4 *>(o) = *reinterpret_cast<const float4 *>(p + i);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] = p[i + e];
  }
}

// Sums of `a` and `b` over the G threads of a row.  G <= 32: shuffles; larger
// G: a row's warp sums meet in `sm` (two buffers used in turn, so that one
// barrier per call is enough).
template <int G> __device__ __forceinline__ float2 row_sum(float a, float b, float2 *sm, int &turn) {
#pragma unroll
  for (int o = (G < 32 ? G : 32) / 2; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  if (G <= 32) return make_float2(a, b);
  float2 *buf = sm + turn * 32;
  turn ^= 1;
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = make_float2(a, b);
  __syncthreads();
  float2 t = make_float2(0.f, 0.f);
  const int w0 = threadIdx.x / G * (G / 32); // this row's warps
#pragma unroll
  for (int w = 0; w < G / 32; ++w) {
    t.x += buf[w0 + w].x;
    t.y += buf[w0 + w].y;
  }
  return t;
}

// Floats between two parameter vectors in shared memory.
__host__ __device__ constexpr int pitch_of(int D) { return (D + 3) / 4 * 4; }

struct FwdArgs {
  const void *x, *res, *gamma, *beta;
  void *sum, *y;
  float *mean, *rstd;
  int64_t ldx, ldr, lds, ldy, n;
  int D, wide;
  float eps;
  int stages;                                // BULK
  int32_t *err;
};

template <typename T, int V, int G, int E, bool BULK>
__global__ void __launch_bounds__(threads_of<G>(), G < 512 ? 4 : 1024 / G) k_layer_norm_fwd(const FwdArgs a) {
  constexpr int kRows = threads_of<G>() / G, C = E / V;
  extern __shared__ __align__(16) float dyn[];   // gamma, beta
  __shared__ float2 sm[64];
  fb::pdl_enter();
  int turn = 0;
  const int t = threadIdx.x % G;
  const int64_t step = (int64_t)gridDim.x * kRows;
  int64_t r = (int64_t)blockIdx.x * kRows + threadIdx.x / G;
  float *const gm = dyn, *const bt = dyn + pitch_of(a.D);
  __shared__ uint64_t bars[BULK ? kMaxStages : 1];
  __shared__ int gave_up;
  const Ring ring{reinterpret_cast<uint8_t *>(dyn + 2 * pitch_of(a.D)), bars, &gave_up, a.err, a.stages,
                  a.res ? 2 : 1, (int)(a.D * sizeof(T))};
  const T *const src[2] = {static_cast<const T *>(a.x), static_cast<const T *>(a.res)};
  const int64_t lds[2] = {a.ldx, a.ldr};
  Vec<T, V> nx[C], nr[C];
  if constexpr (BULK) {
    if (threadIdx.x == 0) {
      for (int q = 0; q < a.stages; ++q) fbtc::mbar_init(bars + q, 1);
      gave_up = 0;
      fbtc::fence_barrier_init();
      for (int q = 0; q < a.stages; ++q)
        fill<T, kRows, 2>(ring, q, src, lds, (int64_t)blockIdx.x * kRows + q * step, a.n);
    }
  } else {
    load_row<T, V, G>(nx, a.x, r * a.ldx, t, a.D, r < a.n);
    if (a.res) load_row<T, V, G>(nr, a.res, r * a.ldr, t, a.D, r < a.n);
  }
  stage_param<T, V>(gm, a.gamma, a.wide, a.D, 0.f);
  stage_param<T, V>(bt, a.beta, a.wide, a.D, 0.f);
  __syncthreads();
  int stage = 0;
  uint32_t lap = 0;
  bool ok = true;
  // every thread of the CTA makes the same number of turns (shuffles, barriers)
  for (int64_t r0 = (int64_t)blockIdx.x * kRows; r0 < a.n; r0 += step, r += step) {
    if (BULK) ok = ok && fbtc::mbar_wait(bars + stage, lap & 1, &gave_up, a.err);
    const bool live = r < a.n && ok;         // after a wait that ran out (recorded) nothing more is written
    Vec<T, V> x[C];
    if constexpr (BULK) {
      from_ring<T, V, G, kRows>(nx, ring, stage, 0, threadIdx.x / G, t, a.D);
      if (a.res) from_ring<T, V, G, kRows>(nr, ring, stage, 1, threadIdx.x / G, t, a.D);
    }
    float s = 0.f, v[C][V];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      x[c] = nx[c];
      const int i = (c * G + t) * V;
      unpack<T, V>(v[c], x[c]);
      if (a.res) {
        float q[V];
        unpack<T, V>(q, nr[c]);
#pragma unroll
        for (int e = 0; e < V; ++e) q[e] += v[c][e];
        pack<T, V>(x[c], q);
        if (live && i < a.D) *reinterpret_cast<Vec<T, V> *>(static_cast<T *>(a.sum) + r * a.lds + i) = x[c];
        unpack<T, V>(v[c], x[c]);            // what is kept is what is normalised
      }
      if (i < a.D)
#pragma unroll
        for (int e = 0; e < V; ++e) s += v[c][e];
    }
    if constexpr (!BULK) {
      const int64_t rn = r + step;
      load_row<T, V, G>(nx, a.x, rn * a.ldx, t, a.D, rn < a.n);
      if (a.res) load_row<T, V, G>(nr, a.res, rn * a.ldr, t, a.D, rn < a.n);
    }
    const float mean = row_sum<G>(s, 0.f, sm, turn).x / (float)a.D;
    if constexpr (BULK) {                    // row_sum's barrier: every thread has its part of the stage
      if (threadIdx.x == 0 && ok) fill<T, kRows, 2>(ring, stage, src, lds, r0 + a.stages * step, a.n);
      if (++stage == a.stages) stage = 0, ++lap;
    }
    s = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c)
      if ((c * G + t) * V < a.D)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          v[c][e] -= mean;
          s = fmaf(v[c][e], v[c][e], s);
        }
    const float var = row_sum<G>(s, 0.f, sm, turn).x / (float)a.D;
    const float rstd = 1.f / sqrtf(var + a.eps);
    if (!live) continue;
    if (t == 0) {
      if (a.mean) a.mean[r] = mean;
      if (a.rstd) a.rstd[r] = rstd;
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int i = (c * G + t) * V;
      if (i >= a.D) continue;
      float g[V], b[V];
      group<V>(g, gm, i, a.D);
      group<V>(b, bt, i, a.D);
#pragma unroll
      for (int e = 0; e < V; ++e) b[e] = fmaf(v[c][e] * rstd, g[e], b[e]);
      pack<T, V>(x[c], b);
      *reinterpret_cast<Vec<T, V> *>(static_cast<T *>(a.y) + r * a.ldy + i) = x[c];
    }
  }
  if (BULK && !ok) let_land();
}

// Floats of the CTA's weight-gradient partials in shared memory.
template <int G> __host__ __device__ constexpr int acc_floats(int D) {
  const int groups = threads_of<G>() / (G < 32 ? 32 : G);
  return G == 1024 || groups > 1 ? pitch_of(groups * 2 * D) : 0;
}

struct BwdArgs {
  const void *dy, *x, *gamma, *ds;
  const float *mean, *rstd;
  void *dx;
  float *part;                               // [gridDim.x][2][D]
  int64_t lddy, ldx, ldds, lddx, n;
  int D, wide, weights;                      // weights: dgamma / dbeta wanted
  int stages;                                // BULK
  int32_t *err;
  int fused;                                 // one cluster: it also adds the partials, into
  void *dgamma, *dbeta;
  int accumulate;
};

// One column's dgamma (i < D) or dbeta.
__device__ __forceinline__ void put_weight(void *dgamma, void *dbeta, int i, int D, int wide, int accumulate, float s) {
  void *o = i < D ? dgamma : dbeta;
  if (!o) return;
  const int k = i < D ? i : i - D;
  if (wide) {
    float *f = static_cast<float *>(o) + k;
    *f = accumulate ? *f + s : s;
  } else {
    static_cast<bf16 *>(o)[k] = __float2bfloat16_rn(s);
  }
}

template <typename T, int V, int G, int E, bool BULK>
__global__ void __launch_bounds__(threads_of<G>(), G < 512 ? 2 : 1) k_layer_norm_bwd(const BwdArgs a) {
  constexpr int kRows = threads_of<G>() / G, C = E / V;
  constexpr bool kShared = G == 1024;        // partials in shared memory
  extern __shared__ __align__(16) float dyn[];   // gamma; kShared: [2][D]; else [groups][2][D] for the final sum
  float *const gm = dyn, *const acc = dyn + pitch_of(a.D);
  __shared__ float2 sm[64];
  fb::pdl_enter();
  int turn = 0;
  const int t = threadIdx.x % G;
  float dg[kShared ? 1 : C][V], db[kShared ? 1 : C][V];
  stage_param<T, V>(gm, a.gamma, a.wide, a.D, 0.f);
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int i = (c * G + t) * V + e;
      if (!kShared) dg[c][e] = db[c][e] = 0.f;
      else if (i < a.D) acc[i] = acc[a.D + i] = 0.f;
    }
  const int64_t step = (int64_t)gridDim.x * kRows;
  int64_t r = (int64_t)blockIdx.x * kRows + threadIdx.x / G;
  Vec<T, V> nx[C], ny[C], ns[C];
  float nmean = 0.f, nrstd = 0.f;
  __shared__ uint64_t bars[BULK ? kMaxStages : 1];
  __shared__ int gave_up;
  const Ring ring{reinterpret_cast<uint8_t *>(dyn + pitch_of(a.D) + acc_floats<G>(a.D)), bars, &gave_up, a.err,
                  a.stages, a.ds ? 3 : 2, (int)(a.D * sizeof(T))};
  const T *const src[3] = {static_cast<const T *>(a.x), static_cast<const T *>(a.dy), static_cast<const T *>(a.ds)};
  const int64_t lds[3] = {a.ldx, a.lddy, a.ldds};
  auto fetch = [&](int64_t q) {
    const bool in = q < a.n;
    if constexpr (!BULK) {
    load_row<T, V, G>(nx, a.x, q * a.ldx, t, a.D, in);
    load_row<T, V, G>(ny, a.dy, q * a.lddy, t, a.D, in);
    if (a.ds) load_row<T, V, G>(ns, a.ds, q * a.ldds, t, a.D, in);
    }
    nmean = in ? a.mean[q] : 0.f;
    nrstd = in ? a.rstd[q] : 0.f;            // rows past the end: xhat = 0, dy = 0
  };
  if constexpr (BULK) {
    if (threadIdx.x == 0) {
      for (int q = 0; q < a.stages; ++q) fbtc::mbar_init(bars + q, 1);
      gave_up = 0;
      fbtc::fence_barrier_init();
      for (int q = 0; q < a.stages; ++q)
        fill<T, kRows, 3>(ring, q, src, lds, (int64_t)blockIdx.x * kRows + q * step, a.n);
    }
  }
  fetch(r);
  __syncthreads();
  int stage = 0;
  uint32_t lap = 0;
  bool ok = true;
  for (int64_t r0 = (int64_t)blockIdx.x * kRows; r0 < a.n; r0 += step, r += step) {
    if (BULK) ok = ok && fbtc::mbar_wait(bars + stage, lap & 1, &gave_up, a.err);
    const bool live = r < a.n && ok;
    const float mean = nmean, rstd = nrstd;
    Vec<T, V> ds[C];
    float xh[C][V], g[C][V];                 // xhat, dy gamma
    float s1 = 0.f, s2 = 0.f;
    if constexpr (BULK) {
      from_ring<T, V, G, kRows>(nx, ring, stage, 0, threadIdx.x / G, t, a.D);
      from_ring<T, V, G, kRows>(ny, ring, stage, 1, threadIdx.x / G, t, a.D);
      if (a.ds) from_ring<T, V, G, kRows>(ns, ring, stage, 2, threadIdx.x / G, t, a.D);
      if (!live)                             // a stage's rows past the end were not loaded
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int e = 0; e < V; ++e) nx[c].e[e] = ny[c].e[e] = T(0.f);
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
      unpack<T, V>(xh[c], nx[c]);
      unpack<T, V>(g[c], ny[c]);
      if (a.ds) ds[c] = ns[c];
    }
    fetch(r + step);
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if ((c * G + t) * V >= a.D) continue;
      float gv[V];
      group<V>(gv, gm, (c * G + t) * V, a.D);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float d = g[c][e];
        xh[c][e] = (xh[c][e] - mean) * rstd;
        g[c][e] = d * gv[e];
        s1 += g[c][e];
        s2 = fmaf(g[c][e], xh[c][e], s2);
        if (!kShared) {
          dg[c][e] = fmaf(d, xh[c][e], dg[c][e]);
          db[c][e] += d;
        } else if (a.weights) {
          const int i = (c * G + t) * V + e;
          acc[i] = fmaf(d, xh[c][e], acc[i]);
          acc[a.D + i] += d;
        }
      }
    }
    const float2 s = row_sum<G>(s1, s2, sm, turn);
    if constexpr (BULK) {
      if (threadIdx.x == 0 && ok) fill<T, kRows, 3>(ring, stage, src, lds, r0 + a.stages * step, a.n);
      if (++stage == a.stages) stage = 0, ++lap;
    }
    const float m1 = s.x / (float)a.D, m2 = s.y / (float)a.D;
    if (!live) continue;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int i = (c * G + t) * V;
      if (i >= a.D) continue;
      Vec<T, V> o;
      float q[V];
      if (a.ds) unpack<T, V>(q, ds[c]);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float v = fmaf(-xh[c][e], m2, g[c][e] - m1);
        q[e] = a.ds ? fmaf(rstd, v, q[e]) : rstd * v;
      }
      pack<T, V>(o, q);
      *reinterpret_cast<Vec<T, V> *>(static_cast<T *>(a.dx) + r * a.lddx + i) = o;
    }
  }
  if (BULK && !ok) let_land();
  if (!a.weights) return;
  float *out = a.part + (int64_t)blockIdx.x * 2 * a.D;
  // rows of a warp meet by shuffles, the CTA's groups in shared memory
  constexpr int kGroups = threads_of<G>() / (G < 32 ? 32 : G);
  const int grp = threadIdx.x / (G < 32 ? 32 : G);
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int i = (c * G + t) * V + e;
      float g = kShared ? (i < a.D ? acc[i] : 0.f) : dg[kShared ? 0 : c][e];
      float b = kShared ? (i < a.D ? acc[a.D + i] : 0.f) : db[kShared ? 0 : c][e];
#pragma unroll
      for (int o = G; o < 32; o <<= 1) {
        g += __shfl_xor_sync(0xffffffffu, g, o);
        b += __shfl_xor_sync(0xffffffffu, b, o);
      }
      float *mine = kGroups > 1 ? acc + (int64_t)grp * 2 * a.D : out;
      if (i < a.D && (G >= 32 || (threadIdx.x & 31) < G)) mine[i] = g, mine[a.D + i] = b;
    }
  if (kGroups > 1) {
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * a.D; i += blockDim.x) {
      float v = 0.f;
#pragma unroll
      for (int q = 0; q < kGroups; ++q) v += acc[q * 2 * a.D + i];
      out[i] = v;
    }
  }
  if (!a.fused) return;
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < 2 * a.D; i += gridDim.x * blockDim.x) {
    float v = 0.f;
    for (int q = 0; q < (int)gridDim.x; ++q) v += a.part[(int64_t)q * 2 * a.D + i];
    put_weight(a.dgamma, a.dbeta, i, a.D, a.wide, a.accumulate, v);
  }
}

// dgamma / dbeta from the CTA partials: 32 columns x 32 warps per CTA; a warp
// adds every 32nd partial, the warps meet in order.
__global__ void __launch_bounds__(1024) k_layer_norm_reduce(const float *part, int parts, int D, void *dgamma,
                                                            void *dbeta, int wide, int accumulate) {
  __shared__ float sm[32][33];
  fb::pdl_enter();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int i = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (i < 2 * D) {
    const float *p = part + i;
    const int64_t row = 2 * D;
    int q = w;
    for (; q + 96 < parts; q += 128) {
      const float v0 = p[q * row], v1 = p[(q + 32) * row], v2 = p[(q + 64) * row], v3 = p[(q + 96) * row];
      s += v0, s += v1, s += v2, s += v3;
    }
    for (; q < parts; q += 32) s += p[q * row];
  }
  sm[w][lane] = s;
  __syncthreads();
  if (w || i >= 2 * D) return;
#pragma unroll
  for (int q = 1; q < 32; ++q) s += sm[q][lane];
  put_weight(dgamma, dbeta, i, D, wide, accumulate, s);
}

// Widest power-of-two element group (at most 16 bytes) that divides the row
// width and every pitch and keeps every base aligned.
struct Align {
  int64_t m = 0;
  int es;
  explicit Align(int es_) : es(es_) {}
  void add(const void *p, int64_t ld) {
    if (!p) return;
    m |= (int64_t)(reinterpret_cast<uintptr_t>(p) | (uintptr_t)(ld * es));
  }
  int vec(int D) const {
    int v = 16 / es;
    while (v > 1 && (D % v || (m & (v * es - 1)))) v >>= 1;
    return es == 4 && v == 2 ? 1 : v;        // built for 16-byte groups, 8- and 4-byte ones of bf16, single ones
  }
};

// Elements of a row per thread: 32 bytes in vectors; 8 single ones (each takes
// a register of its own); twice that where 1024 threads would not hold the row.
int elems_of(int type, int V, int D) {
  const int e = type == FB_BF16 && V > 1 ? 16 : 8;
  return D <= 1024 * e ? e : 16;
}
int group_of(int type, int V, int D) {
  const int e = elems_of(type, V, D);
  for (int g : {8, 32, 64, 128, 256, 512})
    if (D <= g * e) return g;
  return 1024;
}

template <template <typename, int, int, int, bool> class K, typename T, int V, int E, typename... A>
int by_group(int G, A &&...a) {
  switch (G) {
    case 8: return K<T, V, 8, E, false>::go(a...);
    case 32: return K<T, V, 32, E, false>::go(a...);
    case 64: return K<T, V, 64, E, false>::go(a...);
    case 128: return K<T, V, 128, E, false>::go(a...);
    case 256: return K<T, V, 256, E, false>::go(a...);
    case 512: return K<T, V, 512, E, false>::go(a...);
    default: return K<T, V, 1024, E, false>::go(a...);
  }
}
// Rows of at least 2 KB in 16-byte groups come through the ring of bulk copies.
// (past 8192 columns the parameters and partials leave no room for one)
bool bulk_of(int type, int V, int D) {
  return D <= 8192 && (type == FB_F32 ? V == 4 && D >= 512 : V == 8 && D >= 1024);
}

template <template <typename, int, int, int, bool> class K, typename T, int V, int E, typename... A>
int by_group_bulk(int G, A &&...a) {
  switch (G) {
    case 64: return K<T, V, 64, E, true>::go(a...);
    case 128: return K<T, V, 128, E, true>::go(a...);
    case 256: return K<T, V, 256, E, true>::go(a...);
    default:
      if constexpr (E == 8)
        if (G == 1024) return K<T, V, 1024, E, true>::go(a...);
      return K<T, V, 512, E, true>::go(a...);
  }
}
template <template <typename, int, int, int, bool> class K, typename... A> int by_type(int type, int V, int D, A &&...a) {
  const int G = group_of(type, V, D);
  const bool wide = elems_of(type, V, D) == 16;
  if (bulk_of(type, V, D)) {
    return type == FB_BF16 ? by_group_bulk<K, bf16, 8, 16>(G, a...) : by_group_bulk<K, float, 4, 8>(G, a...);
  }
  if (type == FB_F32) {
    if (V == 4) return wide ? K<float, 4, 1024, 16, false>::go(a...) : by_group<K, float, 4, 8>(G, a...);
    return wide ? K<float, 1, 1024, 16, false>::go(a...) : by_group<K, float, 1, 8>(G, a...);
  }
  if (V == 8) return by_group<K, bf16, 8, 16>(G, a...);
  if (V == 4) return by_group<K, bf16, 4, 16>(G, a...);
  if (V == 2) return by_group<K, bf16, 2, 16>(G, a...);
  return wide ? K<bf16, 1, 1024, 16, false>::go(a...) : by_group<K, bf16, 1, 8>(G, a...);
}

int num_sms() {
  static int n[64] = {0};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!n[dev & 63]) {
    int v = 0;
    cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev);
    n[dev & 63] = v > 0 ? v : 148;
  }
  return n[dev & 63];
}

// CTAs that walk n rows: what fits on the SMs at the kernels' register use.
int ctas_of(int64_t n, int G, int per_sm) {
  const int rows = std::max(1, 256 / G);
  return (int)std::max<int64_t>(1, std::min<int64_t>((n + rows - 1) / rows, (int64_t)num_sms() * per_sm));
}
constexpr int64_t kFusedElems = 128 * 1024;
constexpr int kFusedCtas = 8;
int bwd_ctas(int type, int V, int64_t n, int D) {
  const int G = group_of(type, V, D);
  const int c = ctas_of(n, G, G >= 512 ? 1 : 2);
  return n * D <= kFusedElems ? std::min(c, kFusedCtas) : c;
}

// More than the default dynamic shared memory, once per kernel and device.
template <auto kernel> int want_smem(size_t smem) {
  static bool set[64] = {false};
  int dev = 0;
  if (smem <= 40 * 1024) return FB_OK;       // the 48 KB that need no asking include the static arrays
  cudaGetDevice(&dev);
  if (!set[dev & 63]) {
    FB_TRY_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     (int)kSmemCta));
    set[dev & 63] = true;
  }
  return FB_OK;
}

// Ring stages of `unit` bytes beside `smem` bytes: kRing in all, what fits.
int stages_of(int unit, size_t smem) {
  int n = std::max(2, std::min(kMaxStages, kRing / unit));
  while (n > 1 && smem + (size_t)n * unit > kSmemCta) --n;
  return n;
}

template <typename T, int V, int G, int E, bool BULK> struct Fwd {
  static int go(FwdArgs a, cudaStream_t st) {
    constexpr auto k = k_layer_norm_fwd<T, V, G, E, BULK>;
    size_t smem = 2 * sizeof(float) * pitch_of(a.D);
    int per_sm = G < 512 ? 4 : 1024 / G;
    if (BULK) {
      const int unit = (a.res ? 2 : 1) * (threads_of<G>() / G) * a.D * (int)sizeof(T);
      a.stages = stages_of(unit, smem);
      a.err = fbtc::err_word();
      smem += (size_t)a.stages * unit;
      per_sm = std::max(1, std::min(per_sm, (int)(kSmemSm / (smem + 2048))));
    }
    const int rc = want_smem<k>(smem);
    if (rc) return rc;
    FB_TRY_CUDA(fb::launch(k, (unsigned)ctas_of(a.n, G, per_sm), threads_of<G>(), smem, st, a));
    FB_LAUNCHED("k_layer_norm_fwd");
    return FB_OK;
  }
};

// fb::launch as one cluster of `grid` CTAs.
template <typename K, typename A>
cudaError_t launch_cluster(K kernel, unsigned grid, unsigned block, size_t smem, cudaStream_t stream, const A &a) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = grid;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = fb::pdl_enabled() ? 2 : 1;
  ++fb::launches();
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <typename T, int V, int G, int E, bool BULK> struct Bwd {
  static int go(BwdArgs a, int ctas, cudaStream_t st) {
    constexpr auto k = k_layer_norm_bwd<T, V, G, E, BULK>;
    size_t smem = sizeof(float) * (pitch_of(a.D) + acc_floats<G>(a.D));
    if (BULK) {
      const int unit = (a.ds ? 3 : 2) * (threads_of<G>() / G) * a.D * (int)sizeof(T);
      a.stages = stages_of(unit, smem);
      a.err = fbtc::err_word();
      smem += (size_t)a.stages * unit;
    }
    const int rc = want_smem<k>(smem);
    if (rc) return rc;
    FB_TRY_CUDA(a.fused ? launch_cluster(k, (unsigned)ctas, threads_of<G>(), smem, st, a)
                        : fb::launch(k, (unsigned)ctas, threads_of<G>(), smem, st, a));
    FB_LAUNCHED("k_layer_norm_bwd");
    return FB_OK;
  }
};

bool type_ok(int t) { return t == FB_F32 || t == FB_BF16; }
int elem(int t) { return t == FB_F32 ? 4 : 2; }

}  // namespace

extern "C" int fb_layer_norm_fwd(int type, const void *x, int64_t ldx, const void *res, int64_t ldr,
                                 const void *gamma, const void *beta, int param_type, float eps, void *sum,
                                 int64_t lds, void *y, int64_t ldy, float *mean, float *rstd, int64_t n, int D,
                                 cudaStream_t stream) {
  if (!type_ok(type) || (param_type != FB_F32 && param_type != type))
    return fb::set_error(FB_ERR_ARG, "layer_norm_fwd: rows are fp32 or bf16, parameters fp32 or the rows' type");
  if (n < 0 || D < 1 || !gamma || (n > 0 && (!x || !y)) || ldx < D || ldy < D || (res && (!sum || ldr < D || lds < D)) ||
      !(eps >= 0.f))
    return fb::set_error(FB_ERR_ARG, "layer_norm_fwd: bad pointer, size or leading dimension");
  if (D > kMaxD) return fb::set_error(FB_ERR_UNSUPPORTED, "layer_norm_fwd: rows wider than 16384");
  if (n > (int64_t)INT32_MAX) return fb::set_error(FB_ERR_UNSUPPORTED, "layer_norm_fwd: more than 2^31 - 1 rows");
  if (n == 0) return FB_OK;
  Align al(elem(type));
  al.add(x, ldx);
  al.add(y, ldy);
  if (res) al.add(res, ldr), al.add(sum, lds);
  const FwdArgs a{x, res, gamma, beta, sum, y, mean, rstd, ldx, ldr, lds, ldy, n, D, param_type == FB_F32, eps, 0, nullptr};
  return by_type<Fwd>(type, al.vec(D), D, a, stream);
}

extern "C" size_t fb_layer_norm_bwd_ws_bytes(int64_t n, int D) {
  if (n < 1 || D < 1 || D > kMaxD) return 256;
  int most = 1;
  for (int type : {FB_F32, FB_BF16})
    for (int V : {1, 4}) most = std::max(most, bwd_ctas(type, V, n, D));
  return (size_t)most * 2 * D * sizeof(float) + 256;
}

extern "C" int fb_layer_norm_bwd(int type, const void *dy, int64_t lddy, const void *x, int64_t ldx,
                                 const void *gamma, int param_type, const float *mean, const float *rstd,
                                 const void *ds, int64_t ldds, void *dx, int64_t lddx, void *dgamma, void *dbeta,
                                 int accumulate, int64_t n, int D, void *ws, size_t ws_bytes, cudaStream_t stream) {
  if (!type_ok(type) || (param_type != FB_F32 && param_type != type))
    return fb::set_error(FB_ERR_ARG, "layer_norm_bwd: rows are fp32 or bf16, parameters fp32 or the rows' type");
  if (n < 0 || D < 1 || !gamma || (n > 0 && (!dy || !x || !mean || !rstd || !dx)) || lddy < D || ldx < D ||
      lddx < D || (ds && ldds < D))
    return fb::set_error(FB_ERR_ARG, "layer_norm_bwd: bad pointer, size or leading dimension");
  if (accumulate && param_type != FB_F32)
    return fb::set_error(FB_ERR_UNSUPPORTED, "layer_norm_bwd: only fp32 weight gradients accumulate");
  if (D > kMaxD) return fb::set_error(FB_ERR_UNSUPPORTED, "layer_norm_bwd: rows wider than 16384");
  const bool weights = dgamma || dbeta;
  if (weights && n > 0 && (!ws || ws_bytes < fb_layer_norm_bwd_ws_bytes(n, D)))
    return fb::set_error(FB_ERR_ARG, "layer_norm_bwd: workspace too small");
  if (weights && n > 0 && (reinterpret_cast<uintptr_t>(ws) & 15u))
    return fb::set_error(FB_ERR_ARG, "layer_norm_bwd: the workspace must be 16-byte aligned");
  if (n == 0) {                              // an empty sum is zero
    const size_t pb = (size_t)D * elem(param_type);
    if (dgamma && !accumulate) FB_TRY_CUDA(cudaMemsetAsync(dgamma, 0, pb, stream));
    if (dbeta && !accumulate) FB_TRY_CUDA(cudaMemsetAsync(dbeta, 0, pb, stream));
    return FB_OK;
  }
  Align al(elem(type));
  al.add(dy, lddy);
  al.add(x, ldx);
  al.add(dx, lddx);
  if (ds) al.add(ds, ldds);
  const int V = al.vec(D), ctas = bwd_ctas(type, V, n, D);
  float *part = static_cast<float *>(ws);
  const bool fused = weights && n * D <= kFusedElems;
  const BwdArgs a{dy, x, gamma, ds, mean, rstd, dx, part, lddy, ldx, ldds, lddx, n, D, param_type == FB_F32, weights, 0, nullptr,
                  fused, dgamma, dbeta, accumulate};
  const int rc = by_type<Bwd>(type, V, D, a, ctas, stream);
  if (rc || !weights || fused) return rc;
  FB_TRY_CUDA(fb::launch(k_layer_norm_reduce, (unsigned)((2 * D + 31) / 32), 1024, 0, stream, (const float *)part, ctas,
                         D, dgamma, dbeta, (int)(param_type == FB_F32), accumulate));
  FB_LAUNCHED("k_layer_norm_reduce");
  return FB_OK;
}
