// Softmax cross entropy of rows h [n, D] against every row of a table w [V, D]:
//   l = h w^T,  lse_i = log sum_v exp(l_iv),  loss_i = lse_i - l_i,target
//   G = dloss_i (exp(l_iv - lse_i) - [v == target]),  dh = G w,  dw = G^T h
// The logits are never kept: both directions take the table in pieces of as
// many rows as make a logits piece of kPieceBytes (it stays in the L2), the
// forward carrying each row's running maximum and sum over the pieces.
#include <cuda_bf16.h>
#include <algorithm>
#include <cmath>
#include "head.cuh"

namespace {

using namespace fbh;

constexpr int64_t kPieceBytes = 48ll << 20;

struct MaxSum {
  float m, s;                                // sum of exp(l - m); m = -inf, s = 0: nothing yet
};
__device__ __forceinline__ MaxSum join(MaxSum a, MaxSum b) {
  const float m = fmaxf(a.m, b.m);
  if (m == -INFINITY) return MaxSum{m, a.s + b.s};     // a NaN sum stays one
  return MaxSum{m, a.s * expf(a.m - m) + b.s * expf(b.m - m)};
}

// One CTA per row: the piece's maximum and sum join the row's state; the
// target's logit is picked up when the piece holds it.  last: lse and loss.
__global__ void __launch_bounds__(256) k_xent_rows(const float *l, int64_t ldl, int v0, int cols, int64_t V,
                                                   const int64_t *target, float *state, float *tl, float *loss,
                                                   float *lse, int first, int last) {
  __shared__ MaxSum sm[8];
  fb::pdl_enter();
  const int64_t r = blockIdx.x;
  const float *p = l + r * ldl;
  float m = -INFINITY;
  bool nan = false;
  for (int c = threadIdx.x; c < cols; c += 256) {
    const float v = p[c];
    nan |= isnan(v);
    m = fmaxf(m, v);
  }
  MaxSum a{m, 0.f};
  if (m != -INFINITY)
    for (int c = threadIdx.x; c < cols; c += 256) a.s += expf(p[c] - m);
  if (nan) a.s = NAN;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    a = join(a, MaxSum{__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o)});
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = a;
  __syncthreads();
  if (threadIdx.x) return;
#pragma unroll
  for (int w = 1; w < 8; ++w) a = join(a, sm[w]);
  if (!first) a = join(a, MaxSum{state[2 * r], state[2 * r + 1]});
  const int64_t t = target[r];
  float lt = first ? 0.f : tl[r];
  if (t >= v0 && t < v0 + cols) lt = p[t - v0];
  if (!last) {
    state[2 * r] = a.m;
    state[2 * r + 1] = a.s;
    tl[r] = lt;
    return;
  }
  const float z = a.m + logf(a.s);
  lse[r] = z;
  loss[r] = t < 0 ? 0.f : (t >= V ? NAN : z - lt);
}

__device__ __forceinline__ void put(float *p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }

// G of one piece (G may be the logits themselves).  Rows held out of the loss
// are zeros whatever their logits are.
template <typename T>
__global__ void k_xent_grad(const float *l, int64_t ldl, int v0, int cols, int64_t V, const int64_t *target,
                            const float *lse, const float *dloss, T *G, int64_t ldg) {
  fb::pdl_enter();
  const int64_t r = blockIdx.x;
  const int64_t t = target[r];
  const bool live = t >= 0 && t < V;
  const float z = lse[r], d = dloss[r];
  for (int c = blockIdx.y * blockDim.x + threadIdx.x; c < cols; c += gridDim.y * blockDim.x) {
    float v = 0.f;
    if (live) v = d * (expf(l[r * ldl + c] - z) - (t == v0 + c ? 1.f : 0.f));
    put(G + r * ldg + c, v);
  }
}

// Table rows per piece: a multiple of 64, so that pieces start 16-byte aligned.
int64_t piece_rows(int64_t n, int64_t V) {
  const int64_t r = std::max<int64_t>(256, kPieceBytes / 4 / std::max<int64_t>(n, 1) / 64 * 64);
  return std::min<int64_t>(r, round_up(V, 64));
}

int check(const fb_softmax_xent *a, bool bwd) {
  if (!a) return fb::set_error(FB_ERR_ARG, "softmax_xent: null arguments");
  if (a->type != FB_F32 && a->type != FB_BF16) return fb::set_error(FB_ERR_ARG, "softmax_xent: rows are fp32 or bf16");
  if (a->n < 0 || a->D < 1 || a->V < 1) return fb::set_error(FB_ERR_ARG, "softmax_xent: bad size");
  if (a->n > INT32_MAX / 2 || a->D > (1 << 20) || a->V > INT32_MAX / 2)
    return fb::set_error(FB_ERR_UNSUPPORTED, "softmax_xent: more than 2^30 rows or 2^20 columns");
  if (!a->w || a->ldw < a->D || a->ldh < a->D || (a->n > 0 && (!a->h || !a->target || !a->lse)))
    return fb::set_error(FB_ERR_ARG, "softmax_xent: bad pointer or leading dimension");
  if (!bwd) {
    if (a->n > 0 && !a->loss) return fb::set_error(FB_ERR_ARG, "softmax_xent_fwd: bad output");
    return FB_OK;
  }
  if ((a->n > 0 && !a->dloss) || (a->dh && a->lddh < a->D) || (a->dw && a->lddw < a->D))
    return fb::set_error(FB_ERR_ARG, "softmax_xent_bwd: bad pointer or leading dimension");
  if (a->grad_type != FB_F32 && a->grad_type != a->type)
    return fb::set_error(FB_ERR_ARG, "softmax_xent_bwd: the table's gradient is fp32 or of the rows' type");
  if (a->accumulate && a->grad_type != FB_F32)
    return fb::set_error(FB_ERR_UNSUPPORTED, "softmax_xent_bwd: only an fp32 table gradient accumulates");
  return FB_OK;
}

Mat rows_from(const Mat &m, int type, int64_t r) {
  return Mat{static_cast<const uint8_t *>(m.p) + r * m.ld * elem(type), m.ld};
}

int forward(Call &c, const fb_softmax_xent &a) {
  Mat h, w;
  FBH_TRY(aligned(c, a.type, Mat{a.h, a.ldh}, a.n, a.D, &h));
  FBH_TRY(aligned(c, a.type, Mat{a.w, a.ldw}, a.V, a.D, &w));
  const int64_t pr = piece_rows(a.n, a.V);
  FBH_TAKE(l, c, float, a.n * pr);
  FBH_TAKE(state, c, float, 2 * a.n);
  FBH_TAKE(tl, c, float, a.n);
  for (int64_t v0 = 0; v0 < a.V; v0 += pr) {
    const int cols = (int)std::min<int64_t>(pr, a.V - v0);
    FBH_TRY(product(c, a.type, FB_GEMM_NT, h, rows_from(w, a.type, v0), l, pr, a.n, cols, a.D, 0));
    if (c.dry) break;                        // every piece takes the same workspace
    FB_TRY_CUDA(fb::launch(k_xent_rows, (unsigned)a.n, 256, 0, c.stream, (const float *)l, pr, (int)v0, cols, a.V,
                           a.target, state, tl, a.loss, a.lse, (int)(v0 == 0), (int)(v0 + pr >= a.V)));
    FB_LAUNCHED("k_xent_rows");
  }
  return FB_OK;
}

template <typename T> int backward(Call &c, const fb_softmax_xent &a) {
  Mat h, w;
  FBH_TRY(aligned(c, a.type, Mat{a.h, a.ldh}, a.n, a.D, &h));
  FBH_TRY(aligned(c, a.type, Mat{a.w, a.ldw}, a.V, a.D, &w));
  const int64_t pr = piece_rows(a.n, a.V);
  FBH_TAKE(l, c, float, a.n * pr);
  T *G = reinterpret_cast<T *>(l);
  float *dh = static_cast<float *>(a.dh), *dwt = nullptr;
  int64_t lddh = a.lddh;
  if (a.type != FB_F32) {
    FBH_TAKE(gb, c, T, a.n * pr);
    G = gb;
    if (a.dh) {
      FBH_TAKE(t, c, float, a.n * a.D);
      dh = t, lddh = a.D;
    }
  }
  if (a.dw && a.grad_type != FB_F32) {
    FBH_TAKE(t, c, float, pr * a.D);
    dwt = t;
  }
  for (int64_t v0 = 0; v0 < a.V; v0 += pr) {
    const int cols = (int)std::min<int64_t>(pr, a.V - v0);
    const Mat wp = rows_from(w, a.type, v0), Gm{G, pr};
    FBH_TRY(product(c, a.type, FB_GEMM_NT, h, wp, l, pr, a.n, cols, a.D, 0));
    if (!c.dry) {
      FB_TRY_CUDA(fb::launch(k_xent_grad<T>, dim3((unsigned)a.n, (unsigned)std::min(64, (cols + 255) / 256)), 256, 0,
                             c.stream, (const float *)l, pr, (int)v0, cols, a.V, a.target, (const float *)a.lse,
                             a.dloss, G, pr));
      FB_LAUNCHED("k_xent_grad");
    }
    if (a.dh) FBH_TRY(product(c, a.type, FB_GEMM_NN, Gm, wp, dh, lddh, a.n, a.D, cols, v0 > 0));
    if (a.dw) {
      if (dwt) {
        FBH_TRY(product(c, a.type, FB_GEMM_TN, Gm, h, dwt, a.D, a.n, cols, a.D, 0));
        FBH_TRY(store_rows(c, dwt, a.D, static_cast<uint8_t *>(a.dw) + v0 * a.lddw * elem(a.grad_type), a.lddw,
                           a.grad_type, cols, a.D, 0));
      } else {
        FBH_TRY(product(c, a.type, FB_GEMM_TN, Gm, h, static_cast<float *>(a.dw) + v0 * a.lddw, a.lddw, a.n, cols,
                        a.D, a.accumulate));
      }
    }
    if (c.dry) break;
  }
  if (a.dh && a.type != FB_F32) FBH_TRY(store_rows(c, dh, lddh, a.dh, a.lddh, a.type, a.n, a.D, 0));
  return FB_OK;
}

int run(Call &c, const fb_softmax_xent &a, bool bwd) {
  if (!bwd) return forward(c, a);
  return a.type == FB_F32 ? backward<float>(c, a) : backward<__nv_bfloat16>(c, a);
}

}  // namespace

extern "C" size_t fb_softmax_xent_ws_bytes(const fb_softmax_xent *a, int backward) {
  if (check(a, backward != 0) || a->n == 0) return 256;
  Call c;
  return run(c, *a, backward != 0) ? 0 : c.peak + 256;
}

extern "C" int fb_softmax_xent_fwd(const fb_softmax_xent *a, void *ws, size_t ws_bytes, cudaStream_t stream) {
  FBH_TRY(check(a, false));
  if (a->n == 0) return FB_OK;
  if (!ws) return fb::set_error(FB_ERR_ARG, "softmax_xent_fwd: no workspace");
  Call c(ws, ws_bytes, stream);
  return run(c, *a, false);
}

extern "C" int fb_softmax_xent_bwd(const fb_softmax_xent *a, void *ws, size_t ws_bytes, cudaStream_t stream) {
  FBH_TRY(check(a, true));
  if (a->n == 0) {                           // an empty sum is zero
    if (a->dw && !a->accumulate)
      FB_TRY_CUDA(cudaMemset2DAsync(a->dw, a->lddw * elem(a->grad_type), 0, (size_t)a->D * elem(a->grad_type), a->V,
                                    stream));
    return FB_OK;
  }
  if (!ws) return fb::set_error(FB_ERR_ARG, "softmax_xent_bwd: no workspace");
  Call c(ws, ws_bytes, stream);
  return run(c, *a, true);
}
