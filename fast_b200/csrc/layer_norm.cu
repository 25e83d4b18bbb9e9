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
// A row is read once and held in registers, so the variance is the exact
// two-pass one.  G threads share a row (G = 8 .. 1024, the smallest that hold
// it) and a CTA works on several rows at once when G is small.  Elements move
// in the widest power-of-two groups (up to 16 bytes) that every operand's
// base, row pitch and width allow.  All sums are fp32.
//
// Backward keeps dgamma / dbeta partials of a CTA's rows in registers (in
// shared memory for G = 1024, where registers would spill), writes one
// partial row per CTA and a second kernel adds them in CTA order, so results
// repeat bit for bit.
#include <cuda_bf16.h>
#include <algorithm>
#include "runtime.cuh"

namespace {

using bf16 = __nv_bfloat16;

constexpr int kMaxD = 16384;
constexpr int kElems = 16;                 // row elements a thread holds
constexpr int kBwdCtasPerSm = 2;

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

template <typename T, int V> __device__ __forceinline__ void load(float (&o)[V], const T *p) {
  const Vec<T, V> v = *reinterpret_cast<const Vec<T, V> *>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) o[i] = to_f(v.e[i]);
}
template <typename T, int V> __device__ __forceinline__ void store(T *p, const float (&o)[V]) {
  Vec<T, V> v;
#pragma unroll
  for (int i = 0; i < V; ++i) v.e[i] = from_f<T>(o[i]);
  *reinterpret_cast<Vec<T, V> *>(p) = v;
}

// A parameter (gamma, beta) element: fp32, or the rows' type.
template <typename T> __device__ __forceinline__ float param(const void *p, int wide, int i) {
  return wide ? static_cast<const float *>(p)[i] : to_f(static_cast<const T *>(p)[i]);
}

// Sums of `a` and `b` over the G threads of a row.  G <= 32: shuffles; larger
// G: the CTA is one row, warp sums meet in `sm` (2 x 32 floats, two buffers
// used in turn so that one barrier per call is enough).
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
#pragma unroll
  for (int w = 0; w < G / 32; ++w) {
    t.x += buf[w].x;
    t.y += buf[w].y;
  }
  return t;
}

struct FwdArgs {
  const void *x, *res, *gamma, *beta;
  void *sum, *y;
  float *mean, *rstd;
  int64_t ldx, ldr, lds, ldy, n;
  int D, wide;
  float eps;
};

template <int G> __host__ __device__ constexpr int threads_of() { return G < 128 ? 128 : G; }

template <typename T, int V, int G>
__global__ void __launch_bounds__(threads_of<G>()) k_layer_norm_fwd(const FwdArgs a) {
  constexpr int kRows = threads_of<G>() / G, kC = kElems / V;
  __shared__ float2 sm[64];
  fb::pdl_enter();
  int turn = 0;
  const int t = threadIdx.x % G;
  const int64_t r = (int64_t)blockIdx.x * kRows + threadIdx.x / G;
  const bool live = r < a.n;                 // dead rows stay for the shuffles
  const T *x = static_cast<const T *>(a.x) + (live ? r : 0) * a.ldx;
  float v[kC][V];
  float s = 0.f;
#pragma unroll
  for (int c = 0; c < kC; ++c) {
    const int i = (c * G + t) * V;
#pragma unroll
    for (int e = 0; e < V; ++e) v[c][e] = 0.f;
    if (live && i < a.D) {
      load<T, V>(v[c], x + i);
      if (a.res) {
        float q[V];
        load<T, V>(q, static_cast<const T *>(a.res) + r * a.ldr + i);
#pragma unroll
        for (int e = 0; e < V; ++e) v[c][e] = to_f(from_f<T>(v[c][e] + q[e]));
        store<T, V>(static_cast<T *>(a.sum) + r * a.lds + i, v[c]);
      }
    }
#pragma unroll
    for (int e = 0; e < V; ++e) s += v[c][e];
  }
  const float mean = row_sum<G>(s, 0.f, sm, turn).x / (float)a.D;
  s = 0.f;
#pragma unroll
  for (int c = 0; c < kC; ++c)
    if ((c * G + t) * V < a.D)
#pragma unroll
      for (int e = 0; e < V; ++e) s += (v[c][e] - mean) * (v[c][e] - mean);
  const float var = row_sum<G>(s, 0.f, sm, turn).x / (float)a.D;
  const float rstd = 1.f / sqrtf(var + a.eps);
  if (!live) return;
  if (t == 0) {
    if (a.mean) a.mean[r] = mean;
    if (a.rstd) a.rstd[r] = rstd;
  }
#pragma unroll
  for (int c = 0; c < kC; ++c) {
    const int i = (c * G + t) * V;
    if (i >= a.D) continue;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float b = a.beta ? param<T>(a.beta, a.wide, i + e) : 0.f;
      v[c][e] = (v[c][e] - mean) * rstd * param<T>(a.gamma, a.wide, i + e) + b;
    }
    store<T, V>(static_cast<T *>(a.y) + r * a.ldy + i, v[c]);
  }
}

struct BwdArgs {
  const void *dy, *x, *gamma, *ds;
  const float *mean, *rstd;
  void *dx;
  float *part;                               // [gridDim.x][2][D]
  int64_t lddy, ldx, ldds, lddx, n;
  int D, wide, weights;                      // weights: dgamma / dbeta wanted
};

template <typename T, int V, int G>
__global__ void __launch_bounds__(threads_of<G>()) k_layer_norm_bwd(const BwdArgs a) {
  constexpr int kRows = threads_of<G>() / G, kC = kElems / V;
  constexpr bool kShared = G == 1024;        // partials in shared memory
  extern __shared__ float acc[];             // kShared: [2][D]; else [kRows][2][D] for the final sum (kRows > 1)
  __shared__ float2 sm[64];
  fb::pdl_enter();
  int turn = 0;
  const int t = threadIdx.x % G, sub = threadIdx.x / G;
  float dg[kShared ? 1 : kC][V], db[kShared ? 1 : kC][V], gm[kC][V];
#pragma unroll
  for (int c = 0; c < kC; ++c) {
    const int i = (c * G + t) * V;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      gm[c][e] = i < a.D ? param<T>(a.gamma, a.wide, i + e) : 0.f;
      if (!kShared) dg[c][e] = db[c][e] = 0.f;
      else if (i < a.D) acc[i + e] = acc[a.D + i + e] = 0.f;
    }
  }
  const int64_t step = (int64_t)gridDim.x * kRows;
  // every thread of the CTA makes the same number of turns (shuffles, barriers)
  for (int64_t r0 = (int64_t)blockIdx.x * kRows; r0 < a.n; r0 += step) {
    const int64_t r = r0 + sub;
    const bool live = r < a.n;
    const float mean = live ? a.mean[r] : 0.f, rstd = live ? a.rstd[r] : 0.f;
    float xh[kC][V], dy[kC][V];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int c = 0; c < kC; ++c) {
      const int i = (c * G + t) * V;
      if (live && i < a.D) {
        load<T, V>(xh[c], static_cast<const T *>(a.x) + r * a.ldx + i);
        load<T, V>(dy[c], static_cast<const T *>(a.dy) + r * a.lddy + i);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) xh[c][e] = mean, dy[c][e] = 0.f;
      }
    }
#pragma unroll
    for (int c = 0; c < kC; ++c)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        xh[c][e] = (xh[c][e] - mean) * rstd;
        const float g = dy[c][e] * gm[c][e];
        s1 += g;
        s2 += g * xh[c][e];
        if (!kShared) {
          dg[c][e] += dy[c][e] * xh[c][e];
          db[c][e] += dy[c][e];
        } else {
          const int i = (c * G + t) * V + e;
          if (i < a.D && a.weights) {
            acc[i] += dy[c][e] * xh[c][e];
            acc[a.D + i] += dy[c][e];
          }
        }
      }
    const float2 s = row_sum<G>(s1, s2, sm, turn);
    const float m1 = s.x / (float)a.D, m2 = s.y / (float)a.D;
    if (!live) continue;
#pragma unroll
    for (int c = 0; c < kC; ++c) {
      const int i = (c * G + t) * V;
      if (i >= a.D) continue;
      float o[V];
#pragma unroll
      for (int e = 0; e < V; ++e) o[e] = rstd * (dy[c][e] * gm[c][e] - m1 - xh[c][e] * m2);
      if (a.ds) {
        float q[V];
        load<T, V>(q, static_cast<const T *>(a.ds) + r * a.ldds + i);
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] += q[e];
      }
      store<T, V>(static_cast<T *>(a.dx) + r * a.lddx + i, o);
    }
  }
  if (!a.weights) return;
  float *out = a.part + (int64_t)blockIdx.x * 2 * a.D;
  if (kShared) {
#pragma unroll
    for (int c = 0; c < kC; ++c)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int i = (c * G + t) * V + e;
        if (i < a.D) out[i] = acc[i], out[a.D + i] = acc[a.D + i];
      }
    return;
  }
  float *mine = kRows > 1 ? acc + (int64_t)sub * 2 * a.D : out;
#pragma unroll
  for (int c = 0; c < kC; ++c)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int i = (c * G + t) * V + e;
      if (i < a.D) mine[i] = dg[kShared ? 0 : c][e], mine[a.D + i] = db[kShared ? 0 : c][e];
    }
  if (kRows > 1) {
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * a.D; i += blockDim.x) {
      float v = 0.f;
#pragma unroll
      for (int q = 0; q < kRows; ++q) v += acc[q * 2 * a.D + i];
      out[i] = v;
    }
  }
}

// dgamma / dbeta from the CTA partials, in CTA order: 32 columns x 8 row
// lanes per CTA; each lane adds every eighth partial, the lanes meet in order.
__global__ void __launch_bounds__(256) k_layer_norm_reduce(const float *part, int parts, int D, void *dgamma,
                                                           void *dbeta, int wide, int accumulate) {
  __shared__ float sm[8][33];
  fb::pdl_enter();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int i = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (i < 2 * D)
    for (int p = w; p < parts; p += 8) s += part[(int64_t)p * 2 * D + i];
  sm[w][lane] = s;
  __syncthreads();
  if (w || i >= 2 * D) return;
#pragma unroll
  for (int q = 1; q < 8; ++q) s += sm[q][lane];
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
    return v;
  }
};

int group_of(int D) {
  for (int g : {8, 32, 128, 256, 512})
    if (D <= g * kElems) return g;
  return 1024;
}

template <template <typename, int, int> class K, typename T, int V, typename... A>
int by_group(int G, A &&...a) {
  switch (G) {
    case 8: return K<T, V, 8>::go(a...);
    case 32: return K<T, V, 32>::go(a...);
    case 128: return K<T, V, 128>::go(a...);
    case 256: return K<T, V, 256>::go(a...);
    case 512: return K<T, V, 512>::go(a...);
    default: return K<T, V, 1024>::go(a...);
  }
}
template <template <typename, int, int> class K, typename... A> int by_type(int type, int V, int G, A &&...a) {
  if (type == FB_F32) {
    if (V == 4) return by_group<K, float, 4>(G, a...);
    if (V == 2) return by_group<K, float, 2>(G, a...);
    return by_group<K, float, 1>(G, a...);
  }
  if (V == 8) return by_group<K, bf16, 8>(G, a...);
  if (V == 4) return by_group<K, bf16, 4>(G, a...);
  if (V == 2) return by_group<K, bf16, 2>(G, a...);
  return by_group<K, bf16, 1>(G, a...);
}

template <typename T, int V, int G> struct Fwd {
  static int go(const FwdArgs &a, cudaStream_t st) {
    constexpr int rows = threads_of<G>() / G;
    FB_TRY_CUDA(fb::launch(k_layer_norm_fwd<T, V, G>, (unsigned)((a.n + rows - 1) / rows), threads_of<G>(), 0, st, a));
    FB_LAUNCHED("k_layer_norm_fwd");
    return FB_OK;
  }
};

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

// CTAs of the backward grid (= partial rows): every SM busy, and enough rows
// per CTA that its one partial row is a small part of what it reads.
int bwd_ctas(int64_t n, int D, int sms) {
  const int G = group_of(D), rows = (G < 128 ? 128 : G) / G;
  const int per_sm = G >= 512 ? kBwdCtasPerSm : (G >= 256 ? 2 * kBwdCtasPerSm : 4 * kBwdCtasPerSm);
  return (int)std::max<int64_t>(1, std::min<int64_t>((n + rows - 1) / rows, (int64_t)sms * per_sm));
}

template <typename T, int V, int G> struct Bwd {
  static int go(const BwdArgs &a, int ctas, cudaStream_t st) {
    constexpr int rows = threads_of<G>() / G;
    const size_t smem = G == 1024 ? 2 * sizeof(float) * a.D : (rows > 1 ? rows * 2 * sizeof(float) * a.D : 0);
    if (smem > 48 * 1024)
      FB_TRY_CUDA(cudaFuncSetAttribute(k_layer_norm_bwd<T, V, G>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       (int)smem));
    FB_TRY_CUDA(fb::launch(k_layer_norm_bwd<T, V, G>, (unsigned)ctas, threads_of<G>(), smem, st, a));
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
  const FwdArgs a{x, res, gamma, beta, sum, y, mean, rstd, ldx, ldr, lds, ldy, n, D, param_type == FB_F32, eps};
  return by_type<Fwd>(type, al.vec(D), group_of(D), a, stream);
}

extern "C" size_t fb_layer_norm_bwd_ws_bytes(int64_t n, int D) {
  if (n < 1 || D < 1 || D > kMaxD) return 256;
  return (size_t)bwd_ctas(n, D, num_sms()) * 2 * D * sizeof(float) + 256;
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
  const int ctas = bwd_ctas(n, D, num_sms());
  float *part = static_cast<float *>(ws);
  const BwdArgs a{dy, x, gamma, ds, mean, rstd, dx, part, lddy, ldx, ldds, lddx, n, D, param_type == FB_F32, weights};
  const int rc = by_type<Bwd>(type, al.vec(D), group_of(D), a, ctas, stream);
  if (rc || !weights) return rc;
  FB_TRY_CUDA(fb::launch(k_layer_norm_reduce, (unsigned)((2 * D + 31) / 32), 256, 0, stream, (const float *)part, ctas,
                         D, dgamma, dbeta, (int)(param_type == FB_F32), accumulate));
  FB_LAUNCHED("k_layer_norm_reduce");
  return FB_OK;
}
