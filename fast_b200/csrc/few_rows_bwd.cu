// The backward of few rows (see few_rows.cuh): bound by the weights it reads
// and the weight gradients it writes.  Sums along the weights' rows (few_rows.cu:
// gate and up, or the logits), sums over them (k_few_columns: dh, dx), elementwise
// steps, and outer products written once (k_few_outer: the weights' gradients);
// everything between is fp32.
//
// Gated block of 2,048 x 8,192, one row, us: fp32 29 for gate and up (134 MB,
// 4.6 TB/s), 45 for dh and dx (201 MB, 4.5 TB/s), 33 for the gradients (201 MB,
// 6.1 TB/s), 5 elementwise.  Eight rows of x take 46, 76 and 56: three to eight
// multiply-adds for each byte then bind it, not the memory.
#include "few_rows.cuh"
#include <cuda_bf16.h>
#include <algorithm>
#include "act.cuh"
#include "tc_common.cuh"

namespace {

using namespace fbh;
using bf16 = __nv_bfloat16;

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(bf16 v) { return __bfloat162float(v); }

// P[split][m][n] = sum over the split's rows k of x_t[m, k] W_t[k, n]; a split is `chunk` rows of one term t.  A warp
// takes every eighth row, V columns a lane, kDeep rows asked for at once; x of the split waits in shared memory; the
// warps' sums meet there at the end, in warp order.
constexpr int kDeep = 8;
struct ColArgs {
  const float *x[2];
  const void *w[2];
  int64_t ldx, ldw[2];
  int per_term, n, N, chunk;                  // splits of a term, rows of a split
  int64_t K;
  float *P;
};
template <typename T, int V> struct Piece {
  using type = T;
};
template <> struct Piece<float, 4> {
  using type = float4;
};
template <> struct Piece<bf16, 4> {
  using type = uint2;
};
__device__ __forceinline__ void unpack(float4 u, float (&v)[4]) { v[0] = u.x, v[1] = u.y, v[2] = u.z, v[3] = u.w; }
__device__ __forceinline__ void unpack(uint2 u, float (&v)[4]) {
  v[0] = __uint_as_float(u.x << 16), v[1] = __uint_as_float(u.x & 0xFFFF0000u);
  v[2] = __uint_as_float(u.y << 16), v[3] = __uint_as_float(u.y & 0xFFFF0000u);
}
template <typename T> __device__ __forceinline__ void unpack(T u, float (&v)[1]) { v[0] = to_f(u); }

template <typename T, int V, int MT> __global__ void __launch_bounds__(256) k_few_columns(const __grid_constant__ ColArgs a) {
  using P = typename Piece<T, V>::type;
  extern __shared__ __align__(16) float sm[];  // [chunk][MT], then [8][MT][32 V]
  float *red = sm + MT * a.chunk;
  fb::pdl_enter();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, t = (int)blockIdx.y >= a.per_term;
  const int64_t k0 = (int64_t)((int)blockIdx.y - t * a.per_term) * a.chunk;
  const int kn = (int)min((int64_t)a.chunk, a.K - k0);
  const float *x = a.x[t];
#pragma unroll
  for (int m = 0; m < MT; ++m)
    for (int k = threadIdx.x; k < kn; k += 256) sm[k * MT + m] = m < a.n ? x[m * a.ldx + k0 + k] : 0.f;
  __syncthreads();
  const int64_t col = ((int64_t)blockIdx.x * 32 + lane) * V, ld = a.ldw[t];
  const T *w = static_cast<const T *>(a.w[t]) + k0 * ld + (col < a.N ? col : 0);   // columns past the end are not kept
  float acc[MT][V];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int e = 0; e < V; ++e) acc[m][e] = 0.f;
  auto row = [&](int k, P u) {
    float v[V];
    unpack(u, v);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const float q = sm[k * MT + m];
#pragma unroll
      for (int e = 0; e < V; ++e) acc[m][e] = fmaf(q, v[e], acc[m][e]);
    }
  };
  int k = warp;
  for (; k + 8 * (kDeep - 1) < kn; k += 8 * kDeep) {
    P u[kDeep];
#pragma unroll
    for (int d = 0; d < kDeep; ++d) u[d] = *reinterpret_cast<const P *>(w + (k + 8 * d) * ld);
#pragma unroll
    for (int d = 0; d < kDeep; ++d) row(k + 8 * d, u[d]);
  }
  for (; k < kn; k += 8) row(k, *reinterpret_cast<const P *>(w + k * ld));
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int e = 0; e < V; ++e) red[(warp * MT + m) * 32 * V + lane * V + e] = acc[m][e];
  __syncthreads();
  for (int i = threadIdx.x; i < MT * 32 * V; i += 256) {
    const int m = i / (32 * V), c = i - m * 32 * V;
    const int64_t at = (int64_t)blockIdx.x * 32 * V + c;
    if (m >= a.n || at >= a.N) continue;
    float s = 0.f;
#pragma unroll
    for (int q = 0; q < 8; ++q) s += red[q * MT * 32 * V + i];
    a.P[((int64_t)blockIdx.y * a.n + m) * a.N + at] = s;
  }
}

// (dg, du, h) [3][n][F] from gu [n][2 F] and dh's partials [splits][n][F].
__global__ void __launch_bounds__(256) k_few_act(const float *gu, const float *P, int splits, int act, float *o, int64_t n,
                                                 int F) {
  fb::pdl_enter();
  const int64_t total = n * F, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= total) return;
  float d = 0.f;
#pragma unroll 8
  for (int q = 0; q < splits; ++q) d += P[q * total + i];
  const int64_t m = i / F, f = i - m * F;
  const float g = gu[m * 2 * F + f], u = gu[m * 2 * F + F + f];
  const float2 v = act == fbact::kSilu ? fbact::act_exact<fbact::kSilu>(g)
                                       : (act == fbact::kGelu ? fbact::act_exact<fbact::kGelu>(g)
                                                              : fbact::act_exact<fbact::kRelu>(g));
  o[i] = d * u * v.y;
  o[total + i] = d * v.x;
  o[2 * total + i] = v.x * u;
}

// G from the logits [n, V], in their place; rows held out are zeros.
__global__ void __launch_bounds__(256) k_few_grad(float *l, int64_t V, const int64_t *target, const float *lse,
                                                  const float *dloss) {
  fb::pdl_enter();
  const int64_t r = blockIdx.y, c = (int64_t)blockIdx.x * 256 + threadIdx.x, t = target[r];
  if (c >= V) return;
  float v = 0.f;
  if (t >= 0 && t < V) v = dloss[r] * (expf(l[r * V + c] - lse[r]) - (t == c ? 1.f : 0.f));
  l[r * V + c] = v;
}

// n rows as fp32 [n, cols].
template <typename T> __global__ void __launch_bounds__(256) k_few_widen(const T *x, int64_t ldx, float *o, int64_t n, int cols) {
  fb::pdl_enter();
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < n * cols) o[i] = to_f(x[i / cols * ldx + i % cols]);
}

// kind 0, outer products: out[r, c] (+)= sum_m a[m, r] b[m, c] (weight gradients); a warp keeps b of its 128
// columns and walks 16 rows.  kind 1, the last sum of k_few_columns: out[m, c] = sum over splits of a.
struct OutJob {
  const void *a, *b;
  int64_t lda, ldb, ldo, rows;
  void *out;
  int cols, a_f32, b_f32, o_f32, accumulate, kind, splits, wide;   // wide: aligned groups of 4, written
  unsigned first, col_tiles;
  const int64_t *target;                     // given: rows m whose target is not one of V are left out
  int64_t V;
};
struct OutArgs {
  OutJob j[4];
  int n_jobs, n;
};
template <typename T> __device__ __forceinline__ float read_f(const void *p, int64_t i, int f32) {
  return f32 ? static_cast<const float *>(p)[i] : to_f(static_cast<const T *>(p)[i]);
}
__device__ __forceinline__ void write_f(const OutJob &j, int64_t at, float v) {
  if (j.o_f32) {
    float *o = static_cast<float *>(j.out) + at;
    *o = j.accumulate ? *o + v : v;
  } else {
    static_cast<bf16 *>(j.out)[at] = __float2bfloat16_rn(v);
  }
}
template <typename T, int MT> __global__ void __launch_bounds__(256) k_few_outer(const __grid_constant__ OutArgs a) {
  fb::pdl_enter();
  int job = 0;
  while (job + 1 < a.n_jobs && blockIdx.x >= a.j[job + 1].first) ++job;
  const OutJob &j = a.j[job];
  const unsigned blk = blockIdx.x - j.first;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (j.kind == 1) {
    const int64_t total = j.rows * j.cols, i = (int64_t)blk * 256 + threadIdx.x;
    if (i >= total) return;
    const float *P = static_cast<const float *>(j.a);
    float s = 0.f;
#pragma unroll 8
    for (int z = 0; z < j.splits; ++z) s += P[z * total + i];
    const int64_t m = i / j.cols;
    write_f(j, m * j.ldo + (i - m * j.cols), s);
    return;
  }
  __shared__ __align__(16) float as[128][MT];  // the CTA's rows of a
  // this lane's columns: c0 + e step, four side by side where they are written at once, else a warp's side by side
  const int c0 = (int)(blk % j.col_tiles) * 128 + (j.wide ? lane * 4 : lane), step = j.wide ? 1 : 32;
  const int64_t R0 = (int64_t)(blk / j.col_tiles) * 128;
  const int rows = (int)min((int64_t)128, j.rows - R0);
#pragma unroll
  for (int i = threadIdx.x; i < MT * 128; i += 256) {
    const int r = i & 127, m = i >> 7;
    as[r][m] = m < a.n && r < rows ? read_f<T>(j.a, m * j.lda + R0 + r, j.a_f32) : 0.f;
  }
  float b[MT][4];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const bool live = m < a.n && (!j.target || (j.target[m] >= 0 && j.target[m] < j.V));   // zeros against a's zeros
#pragma unroll
    for (int e = 0; e < 4; ++e)
      b[m][e] = live && c0 + e * step < j.cols ? read_f<T>(j.b, m * j.ldb + c0 + e * step, j.b_f32) : 0.f;
  }
  __syncthreads();
  for (int q = warp * 16; q < min(warp * 16 + 16, rows); ++q) {
    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const float x = as[q][m];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = fmaf(x, b[m][e], v[e]);
    }
    const int64_t at = (R0 + q) * j.ldo + c0;
    if (!j.wide) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (c0 + e * 32 < j.cols) write_f(j, at + e * 32, v[e]);
    } else if (c0 < j.cols) {
      if (j.o_f32) {
        *reinterpret_cast<float4 *>(static_cast<float *>(j.out) + at) = make_float4(v[0], v[1], v[2], v[3]);
      } else {
        const __nv_bfloat162 lo = __floats2bfloat162_rn(v[0], v[1]), hi = __floats2bfloat162_rn(v[2], v[3]);
        *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(j.out) + at) =
            make_uint2(*reinterpret_cast<const uint32_t *>(&lo), *reinterpret_cast<const uint32_t *>(&hi));
      }
    }
  }
}

// ---- host ----------------------------------------------------------------------------------------
constexpr int kMaxChunk = 512;

template <typename T, int V, int MT> int launch_columns(const ColArgs &a, unsigned splits, cudaStream_t st) {
  constexpr auto k = k_few_columns<T, V, MT>;
  const size_t smem = sizeof(float) * MT * (a.chunk + 8 * 32 * V);
  if (smem > 40 * 1024) {
    static bool set[64] = {false};
    int dev = 0;
    cudaGetDevice(&dev);
    if (!set[dev & 63]) {
      FB_TRY_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       (int)sizeof(float) * MT * (kMaxChunk + 8 * 32 * V)));
      set[dev & 63] = true;
    }
  }
  FB_TRY_CUDA(fb::launch(k, dim3((unsigned)((a.N + 32 * V - 1) / (32 * V)), splits), 256, smem, st, a));
  FB_LAUNCHED("k_few_columns");
  return FB_OK;
}
template <typename T, int V> int columns_by_rows(const ColArgs &a, unsigned splits, cudaStream_t st) {
  if (a.n == 1) return launch_columns<T, V, 1>(a, splits, st);
  if constexpr (sizeof(T) == 2) return launch_columns<T, V, 2>(a, splits, st);   // bf16: at most 2 rows
  else return a.n <= 4 ? launch_columns<T, V, 4>(a, splits, st) : launch_columns<T, V, 8>(a, splits, st);
}

struct Columns {
  float *P;
  int splits;
};
// The partials of sum_k sum_t x_t[m, k] W_t[k, n], x_t fp32 [n, K].
int columns(Call &c, int type, const float *const *x, int64_t ldx, const Mat *w, int terms, int64_t n, int64_t K, int N,
            Columns *out) {
  const int es = elem(type);
  uintptr_t m = 0;
  for (int t = 0; t < terms; ++t) m |= reinterpret_cast<uintptr_t>(w[t].p) | (uintptr_t)(w[t].ld * es);
  const bool wide = N % 4 == 0 && (m & (uintptr_t)(4 * es - 1)) == 0;
  // rows of a split: four CTAs for every SM, 64 to kMaxChunk
  const int64_t tiles = wide ? (N + 127) / 128 : (N + 31) / 32;
  int64_t chunk = round_up(std::max<int64_t>(1, K * terms * tiles / (4 * fbtc::num_sms())), 64);
  chunk = std::max<int64_t>(64, std::min<int64_t>(kMaxChunk, chunk));
  int64_t per = (K + chunk - 1) / chunk;
  if (per * terms > 65535) chunk = kMaxChunk, per = (K + chunk - 1) / chunk;   // fits: K is at most 2^24
  out->splits = (int)(per * terms);
  FBH_TAKE(P, c, float, (int64_t)out->splits * n * N);
  out->P = P;
  if (c.dry) return FB_OK;
  const int l = terms - 1;                    // a single term stands in both places
  const ColArgs a{{x[0], x[l]}, {w[0].p, w[l].p}, ldx, {w[0].ld, w[l].ld}, (int)per, (int)n, N, (int)chunk, K, P};
  if (type == FB_F32)
    return wide ? columns_by_rows<float, 4>(a, out->splits, c.stream) : columns_by_rows<float, 1>(a, out->splits, c.stream);
  return wide ? columns_by_rows<bf16, 4>(a, out->splits, c.stream) : columns_by_rows<bf16, 1>(a, out->splits, c.stream);
}

struct Outers {
  OutArgs a;
  unsigned ctas = 0;
  explicit Outers(int64_t n) { a.n_jobs = 0, a.n = (int)n; }
  void add(OutJob j, unsigned n_ctas) {
    j.first = ctas;
    a.j[a.n_jobs++] = j;
    ctas += n_ctas;
  }
  // out [rows, cols] (+)= a^T b
  void outer(const void *pa, int64_t lda, int a_f32, int64_t rows, const void *pb, int64_t ldb, int b_f32, int cols, void *out,
             int64_t ldo, int o_type, int accumulate, const int64_t *target = nullptr, int64_t V = 0) {
    if (!out) return;
    const int es = elem(o_type);
    const bool wide = !accumulate && cols % 4 == 0 &&
                      ((reinterpret_cast<uintptr_t>(out) | (uintptr_t)(ldo * es)) & (uintptr_t)(4 * es - 1)) == 0;
    const unsigned ct = (unsigned)((cols + 127) / 128);
    add(OutJob{pa, pb, lda, ldb, ldo, rows, out, cols, a_f32, b_f32, o_type == FB_F32, accumulate, 0, 0, wide, 0, ct, target,
               V},
        ct * (unsigned)((rows + 127) / 128));
  }
  void sum(const Columns &p, int64_t n, int cols, void *out, int64_t ldo, int o_type) {
    add(OutJob{p.P, nullptr, 0, 0, ldo, n, out, cols, 1, 1, o_type == FB_F32, 0, 1, p.splits, 0, 0, 1, nullptr, 0},
        (unsigned)((n * cols + 255) / 256));
  }
  template <typename T> int go(cudaStream_t st) {
    if (ctas == 0) return FB_OK;
    auto k = k_few_outer<T, 1>;
    if constexpr (sizeof(T) == 2) k = a.n == 1 ? k : k_few_outer<T, 2>;
    else k = a.n == 1 ? k : (a.n <= 4 ? k_few_outer<T, 4> : k_few_outer<T, 8>);
    FB_TRY_CUDA(fb::launch(k, ctas, 256, 0, st, a));
    FB_LAUNCHED("k_few_outer");
    return FB_OK;
  }
};

template <typename T> int widen(Call &c, const void *x, int64_t ldx, float *o, int64_t n, int cols) {
  FB_TRY_CUDA(fb::launch(k_few_widen<T>, (unsigned)((n * cols + 255) / 256), 256, 0, c.stream, static_cast<const T *>(x), ldx, o,
                         n, cols));
  FB_LAUNCHED("k_few_widen");
  return FB_OK;
}

}  // namespace

namespace fbh {

int few_rows_ffn_bwd(Call &c, const fb_gated_ffn &a) {
  const Mat x{a.x, a.ldx}, wg{a.w_gate, a.ld_gate}, wu{a.w_up, a.ld_up}, wd{a.w_down, a.ld_down};
  const int64_t n = a.n, nf = n * a.F;
  const int f32 = a.type == FB_F32;
  FBH_TAKE(gu, c, float, 2 * nf);
  FBH_TAKE(dyf, c, float, n * a.D);
  FBH_TAKE(o, c, float, 3 * nf);              // dg, du, h
  FBH_TRY(few_rows_gate_up(c, a.type, x, n, a.D, wg, wu, a.F, gu));
  if (!c.dry) FBH_TRY(f32 ? widen<float>(c, a.dy, a.lddy, dyf, n, a.D) : widen<bf16>(c, a.dy, a.lddy, dyf, n, a.D));
  Columns dh, dx;
  const float *xd[1] = {dyf};
  FBH_TRY(columns(c, a.type, xd, a.D, &wd, 1, n, a.D, a.F, &dh));
  if (!c.dry) {
    FB_TRY_CUDA(fb::launch(k_few_act, (unsigned)((nf + 255) / 256), 256, 0, c.stream, (const float *)gu, (const float *)dh.P,
                           dh.splits, a.act, o, n, a.F));
    FB_LAUNCHED("k_few_act");
  }
  if (a.dx) {
    const float *xg[2] = {o, o + nf};
    const Mat w[2] = {wg, wu};
    FBH_TRY(columns(c, a.type, xg, a.F, w, 2, n, a.F, a.D, &dx));
  }
  if (c.dry) return FB_OK;
  Outers out(n);
  out.outer(o, a.F, 1, a.F, a.x, a.ldx, f32, a.D, a.dw_gate, a.ldd_gate, a.grad_type, a.accumulate);
  out.outer(o + nf, a.F, 1, a.F, a.x, a.ldx, f32, a.D, a.dw_up, a.ldd_up, a.grad_type, a.accumulate);
  out.outer(a.dy, a.lddy, f32, a.D, o + 2 * nf, a.F, 1, a.F, a.dw_down, a.ldd_down, a.grad_type, a.accumulate);
  if (a.dx) out.sum(dx, n, a.D, a.dx, a.lddx, a.type);
  return f32 ? out.go<float>(c.stream) : out.go<bf16>(c.stream);
}

int few_rows_xent_bwd(Call &c, const fb_softmax_xent &a) {
  const Mat h{a.h, a.ldh}, w{a.w, a.ldw};
  const int64_t n = a.n;
  const int f32 = a.type == FB_F32;
  FBH_TAKE(l, c, float, n * a.V);
  FBH_TRY(few_rows_logits(c, a.type, h, n, a.D, w, a.V, l));
  if (!c.dry) {
    FB_TRY_CUDA(fb::launch(k_few_grad, dim3((unsigned)((a.V + 255) / 256), (unsigned)n), 256, 0, c.stream, l, a.V, a.target,
                           (const float *)a.lse, a.dloss));
    FB_LAUNCHED("k_few_grad");
  }
  Columns dh;
  const float *xl[1] = {l};
  if (a.dh) FBH_TRY(columns(c, a.type, xl, a.V, &w, 1, n, a.V, a.D, &dh));
  if (c.dry) return FB_OK;
  Outers out(n);
  out.outer(l, a.V, 1, a.V, a.h, a.ldh, f32, a.D, a.dw, a.lddw, a.grad_type, a.accumulate,
            a.target, a.V);
  if (a.dh) out.sum(dh, n, a.D, a.dh, a.lddh, a.type);
  return f32 ? out.go<float>(c.stream) : out.go<bf16>(c.stream);
}

}  // namespace fbh
