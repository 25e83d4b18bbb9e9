// Gated feed-forward block, forward and backward:
//   g = x Wg^T, u = x Wu^T, h = act(g) u, y = h Wd^T
//   dh = dy Wd, dg = dh u act'(g), du = dh act(g)
//   dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x, dWd = dy^T h
// Only x is kept between the two: the backward recomputes g and u.
#include <cuda_bf16.h>
#include <algorithm>
#include "head.cuh"

namespace {

using namespace fbh;

enum : int { kSilu = FB_ACT_SILU, kGelu = FB_ACT_GELU, kRelu = FB_ACT_RELU };

// act(g) and act'(g)
template <int ACT> __device__ __forceinline__ float2 act2(float g) {
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

__device__ __forceinline__ void put(float *p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }

// h = act(g) u over n elements (pitches alike, padding included).
template <int ACT, typename T> __global__ void k_glu_fwd(const float *g, const float *u, T *h, int64_t n) {
  fb::pdl_enter();
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x)
    put(h + i, act2<ACT>(g[i]).x * u[i]);
}

// (dg, du, h) from (g, u, dh); the outputs may be the inputs.
template <int ACT, typename T>
__global__ void k_glu_bwd(const float *g, const float *u, const float *dh, T *dg, T *du, T *h, int64_t n) {
  fb::pdl_enter();
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
    const float gv = g[i], uv = u[i], d = dh[i];
    const float2 a = act2<ACT>(gv);
    put(dg + i, d * uv * a.y);
    put(du + i, d * a.x);
    put(h + i, a.x * uv);
  }
}

unsigned blocks_for(int64_t n) { return (unsigned)std::max<int64_t>(1, std::min<int64_t>((n + 255) / 256, 148 * 16)); }

template <typename T> int glu_fwd(Call &c, int act, const float *g, const float *u, T *h, int64_t n) {
  if (c.dry) return FB_OK;
  auto k = act == kSilu ? k_glu_fwd<kSilu, T> : (act == kGelu ? k_glu_fwd<kGelu, T> : k_glu_fwd<kRelu, T>);
  FB_TRY_CUDA(fb::launch(k, blocks_for(n), 256, 0, c.stream, g, u, h, n));
  FB_LAUNCHED("k_glu_fwd");
  return FB_OK;
}

template <typename T>
int glu_bwd(Call &c, int act, const float *g, const float *u, const float *dh, T *dg, T *du, T *h, int64_t n) {
  if (c.dry) return FB_OK;
  auto k = act == kSilu ? k_glu_bwd<kSilu, T> : (act == kGelu ? k_glu_bwd<kGelu, T> : k_glu_bwd<kRelu, T>);
  FB_TRY_CUDA(fb::launch(k, blocks_for(n), 256, 0, c.stream, g, u, dh, dg, du, h, n));
  FB_LAUNCHED("k_glu_bwd");
  return FB_OK;
}

int check(const fb_gated_ffn *a, bool bwd) {
  if (!a) return fb::set_error(FB_ERR_ARG, "gated_ffn: null arguments");
  if ((a->type != FB_F32 && a->type != FB_BF16) || a->act < FB_ACT_SILU || a->act > FB_ACT_RELU)
    return fb::set_error(FB_ERR_ARG, "gated_ffn: rows are fp32 or bf16, act is FB_ACT_*");
  if (a->n < 0 || a->D < 1 || a->F < 1) return fb::set_error(FB_ERR_ARG, "gated_ffn: bad size");
  if (a->n > INT32_MAX / 2 || a->D > (1 << 20) || a->F > (1 << 20))
    return fb::set_error(FB_ERR_UNSUPPORTED, "gated_ffn: more than 2^30 rows or 2^20 columns");
  if ((a->n > 0 && !a->x) || !a->w_gate || !a->w_up || !a->w_down || a->ldx < a->D || a->ld_gate < a->D ||
      a->ld_up < a->D || a->ld_down < a->F)
    return fb::set_error(FB_ERR_ARG, "gated_ffn: bad pointer or leading dimension");
  if (!bwd) {
    if ((a->n > 0 && !a->y) || a->ldy < a->D) return fb::set_error(FB_ERR_ARG, "gated_ffn_fwd: bad output");
    return FB_OK;
  }
  if ((a->n > 0 && !a->dy) || a->lddy < a->D || (a->dx && a->lddx < a->D) || (a->dw_gate && a->ldd_gate < a->D) ||
      (a->dw_up && a->ldd_up < a->D) || (a->dw_down && a->ldd_down < a->F))
    return fb::set_error(FB_ERR_ARG, "gated_ffn_bwd: bad pointer or leading dimension");
  if (a->grad_type != FB_F32 && a->grad_type != a->type)
    return fb::set_error(FB_ERR_ARG, "gated_ffn_bwd: weight gradients are fp32 or of the rows' type");
  if (a->accumulate && a->grad_type != FB_F32)
    return fb::set_error(FB_ERR_UNSUPPORTED, "gated_ffn_bwd: only fp32 weight gradients accumulate");
  return FB_OK;
}

template <typename T> int forward(Call &c, const fb_gated_ffn &a) {
  const int64_t N = a.n, Fp = round_up(a.F, 8);
  Mat x, wg, wu, wd;
  FBH_TRY(aligned(c, a.type, Mat{a.x, a.ldx}, N, a.D, &x));
  FBH_TRY(aligned(c, a.type, Mat{a.w_gate, a.ld_gate}, a.F, a.D, &wg));
  FBH_TRY(aligned(c, a.type, Mat{a.w_up, a.ld_up}, a.F, a.D, &wu));
  FBH_TRY(aligned(c, a.type, Mat{a.w_down, a.ld_down}, a.D, a.F, &wd));
  FBH_TAKE(g, c, float, N * Fp);
  FBH_TAKE(u, c, float, N * Fp);
  T *h = reinterpret_cast<T *>(g);
  if (a.type != FB_F32) {
    FBH_TAKE(hb, c, T, N * Fp);
    h = hb;
  }
  FBH_TRY(product(c, a.type, FB_GEMM_NT, x, wg, g, Fp, N, a.F, a.D, 0));
  FBH_TRY(product(c, a.type, FB_GEMM_NT, x, wu, u, Fp, N, a.F, a.D, 0));
  FBH_TRY(glu_fwd<T>(c, a.act, g, u, h, N * Fp));
  if (a.type == FB_F32)
    return product(c, a.type, FB_GEMM_NT, Mat{h, Fp}, wd, static_cast<float *>(a.y), a.ldy, N, a.D, a.F, 0);
  FBH_TAKE(y, c, float, N * a.D);
  FBH_TRY(product(c, a.type, FB_GEMM_NT, Mat{h, Fp}, wd, y, a.D, N, a.D, a.F, 0));
  return store_rows(c, y, a.D, a.y, a.ldy, a.type, N, a.D, 0);
}

// A weight gradient G^T X ([rows_out, cols]) in grad_type.
int weight_grad(Call &c, const fb_gated_ffn &a, const Mat &G, const Mat &X, void *out, int64_t ldo, int rows_out,
                int cols) {
  if (!out) return FB_OK;
  if (a.grad_type == FB_F32)
    return product(c, a.type, FB_GEMM_TN, G, X, static_cast<float *>(out), ldo, a.n, rows_out, cols, a.accumulate);
  const size_t mark = c.off;
  FBH_TAKE(t, c, float, (int64_t)rows_out * cols);
  FBH_TRY(product(c, a.type, FB_GEMM_TN, G, X, t, cols, a.n, rows_out, cols, 0));
  FBH_TRY(store_rows(c, t, cols, out, ldo, a.grad_type, rows_out, cols, 0));
  c.off = mark;
  return FB_OK;
}

template <typename T> int backward(Call &c, const fb_gated_ffn &a) {
  const int64_t N = a.n, Fp = round_up(a.F, 8);
  Mat x, wg, wu, wd, dy;
  FBH_TRY(aligned(c, a.type, Mat{a.x, a.ldx}, N, a.D, &x));
  FBH_TRY(aligned(c, a.type, Mat{a.dy, a.lddy}, N, a.D, &dy));
  FBH_TRY(aligned(c, a.type, Mat{a.w_gate, a.ld_gate}, a.F, a.D, &wg));
  FBH_TRY(aligned(c, a.type, Mat{a.w_up, a.ld_up}, a.F, a.D, &wu));
  FBH_TRY(aligned(c, a.type, Mat{a.w_down, a.ld_down}, a.D, a.F, &wd));
  FBH_TAKE(g, c, float, N * Fp);
  FBH_TAKE(u, c, float, N * Fp);
  FBH_TAKE(dh, c, float, N * Fp);
  T *dg = reinterpret_cast<T *>(g), *du = reinterpret_cast<T *>(u), *h = reinterpret_cast<T *>(dh);
  if (a.type != FB_F32) {
    FBH_TAKE(b, c, T, 3 * N * Fp);
    dg = b, du = b + N * Fp, h = b + 2 * N * Fp;
  }
  FBH_TRY(product(c, a.type, FB_GEMM_NT, x, wg, g, Fp, N, a.F, a.D, 0));
  FBH_TRY(product(c, a.type, FB_GEMM_NT, x, wu, u, Fp, N, a.F, a.D, 0));
  FBH_TRY(product(c, a.type, FB_GEMM_NN, dy, wd, dh, Fp, N, a.F, a.D, 0));
  FBH_TRY(glu_bwd<T>(c, a.act, g, u, dh, dg, du, h, N * Fp));
  if (a.dx) {
    float *dx = static_cast<float *>(a.dx);
    int64_t ld = a.lddx;
    if (a.type != FB_F32) {
      FBH_TAKE(t, c, float, N * a.D);
      dx = t, ld = a.D;
    }
    FBH_TRY(product(c, a.type, FB_GEMM_NN, Mat{dg, Fp}, wg, dx, ld, N, a.D, a.F, 0));
    FBH_TRY(product(c, a.type, FB_GEMM_NN, Mat{du, Fp}, wu, dx, ld, N, a.D, a.F, 1));
    if (a.type != FB_F32) FBH_TRY(store_rows(c, dx, ld, a.dx, a.lddx, a.type, N, a.D, 0));
  }
  FBH_TRY(weight_grad(c, a, Mat{dg, Fp}, x, a.dw_gate, a.ldd_gate, a.F, a.D));
  FBH_TRY(weight_grad(c, a, Mat{du, Fp}, x, a.dw_up, a.ldd_up, a.F, a.D));
  return weight_grad(c, a, dy, Mat{h, Fp}, a.dw_down, a.ldd_down, a.D, a.F);
}

// Weight gradients of a call without rows: zeros.
int empty_grads(const fb_gated_ffn &a, cudaStream_t st) {
  if (a.accumulate) return FB_OK;
  const size_t es = elem(a.grad_type);
  if (a.dw_gate) FB_TRY_CUDA(cudaMemset2DAsync(a.dw_gate, a.ldd_gate * es, 0, a.D * es, a.F, st));
  if (a.dw_up) FB_TRY_CUDA(cudaMemset2DAsync(a.dw_up, a.ldd_up * es, 0, a.D * es, a.F, st));
  if (a.dw_down) FB_TRY_CUDA(cudaMemset2DAsync(a.dw_down, a.ldd_down * es, 0, a.F * es, a.D, st));
  return FB_OK;
}

int run(Call &c, const fb_gated_ffn &a, bool bwd) {
  if (a.type == FB_F32) return bwd ? backward<float>(c, a) : forward<float>(c, a);
  return bwd ? backward<__nv_bfloat16>(c, a) : forward<__nv_bfloat16>(c, a);
}

}  // namespace

extern "C" size_t fb_gated_ffn_ws_bytes(const fb_gated_ffn *a, int backward) {
  if (check(a, backward != 0) || a->n == 0) return 256;
  Call c;
  return run(c, *a, backward != 0) ? 0 : c.peak + 256;
}

extern "C" int fb_gated_ffn_fwd(const fb_gated_ffn *a, void *ws, size_t ws_bytes, cudaStream_t stream) {
  FBH_TRY(check(a, false));
  if (a->n == 0) return FB_OK;
  if (!ws) return fb::set_error(FB_ERR_ARG, "gated_ffn_fwd: no workspace");
  Call c(ws, ws_bytes, stream);
  return run(c, *a, false);
}

extern "C" int fb_gated_ffn_bwd(const fb_gated_ffn *a, void *ws, size_t ws_bytes, cudaStream_t stream) {
  FBH_TRY(check(a, true));
  if (a->n == 0) return empty_grads(*a, stream);
  if (!ws) return fb::set_error(FB_ERR_ARG, "gated_ffn_bwd: no workspace");
  Call c(ws, ws_bytes, stream);
  return run(c, *a, true);
}
