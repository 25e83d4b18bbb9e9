// Gated feed-forward block, forward and backward:
//   g = x Wg^T, u = x Wu^T, h = act(g) u, y = h Wd^T
//   dh = dy Wd, dg = dh u act'(g), du = dh act(g)
//   dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x, dWd = dy^T h
// Only x is kept between the two: the backward recomputes g and u.
//
// bf16: two launches forward, four backward (plus the sums of split
// reductions), each a product on SM pairs (pair_gemm.cuh).  The first of each
// direction computes g and u side by side in one tile -- one CTA of the pair
// stages Wg, the other Wu -- and for the backward dh beside them, and applies
// the activation to the fp32 accumulators: h, dg, du are rounded once, and g,
// u, dh never reach memory.  fp32: the grouped 3xTF32 products with the
// activation between them.
#include "pair_gemm.cuh"

namespace {

using namespace fbh;

constexpr int kSilu = FB_ACT_SILU, kGelu = FB_ACT_GELU;

// act(g) and act'(g)
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

// h = act(g) u over n elements (pitches alike, padding included), in g's place.
template <int ACT> __global__ void k_glu_fwd(float *g, const float *u, int64_t n) {
  fb::pdl_enter();
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x)
    g[i] = act_exact<ACT>(g[i]).x * u[i];
}

// (dg, du, h) in the places of (g, u, dh).
template <int ACT> __global__ void k_glu_bwd(float *g, float *u, float *dh, int64_t n) {
  fb::pdl_enter();
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
    const float uv = u[i], d = dh[i];
    const float2 a = act_exact<ACT>(g[i]);
    g[i] = d * uv * a.y;
    u[i] = d * a.x;
    dh[i] = a.x * uv;
  }
}

unsigned blocks_for(int64_t n) { return (unsigned)std::max<int64_t>(1, std::min<int64_t>((n + 255) / 256, 148 * 16)); }

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

int forward_f32(Call &c, const fb_gated_ffn &a, const Mat &x, const Mat &wg, const Mat &wu, const Mat &wd) {
  const int64_t N = a.n, Fp = round_up(a.F, 4);
  FBH_TAKE(g, c, float, N * Fp);
  FBH_TAKE(u, c, float, N * Fp);
  FBH_TRY(product(c, FB_GEMM_NT, x, wg, g, Fp, N, a.F, a.D, 0));
  FBH_TRY(product(c, FB_GEMM_NT, x, wu, u, Fp, N, a.F, a.D, 0));
  if (!c.dry) {
    auto k = a.act == kSilu ? k_glu_fwd<FB_ACT_SILU> : (a.act == kGelu ? k_glu_fwd<FB_ACT_GELU> : k_glu_fwd<FB_ACT_RELU>);
    FB_TRY_CUDA(fb::launch(k, blocks_for(N * Fp), 256, 0, c.stream, g, (const float *)u, N * Fp));
    FB_LAUNCHED("k_glu_fwd");
  }
  return product(c, FB_GEMM_NT, Mat{g, Fp}, wd, static_cast<float *>(a.y), a.ldy, N, a.D, a.F, 0);
}

int backward_f32(Call &c, const fb_gated_ffn &a, const Mat &x, const Mat &dy, const Mat &wg, const Mat &wu,
                 const Mat &wd) {
  const int64_t N = a.n, Fp = round_up(a.F, 4);
  FBH_TAKE(g, c, float, N * Fp);             // then dg
  FBH_TAKE(u, c, float, N * Fp);             // then du
  FBH_TAKE(d, c, float, N * Fp);             // dh, then h
  FBH_TRY(product(c, FB_GEMM_NT, x, wg, g, Fp, N, a.F, a.D, 0));
  FBH_TRY(product(c, FB_GEMM_NT, x, wu, u, Fp, N, a.F, a.D, 0));
  FBH_TRY(product(c, FB_GEMM_NN, dy, wd, d, Fp, N, a.F, a.D, 0));
  if (!c.dry) {
    auto k = a.act == kSilu ? k_glu_bwd<FB_ACT_SILU> : (a.act == kGelu ? k_glu_bwd<FB_ACT_GELU> : k_glu_bwd<FB_ACT_RELU>);
    FB_TRY_CUDA(fb::launch(k, blocks_for(N * Fp), 256, 0, c.stream, g, u, d, N * Fp));
    FB_LAUNCHED("k_glu_bwd");
  }
  if (a.dx) {
    float *dx = static_cast<float *>(a.dx);
    FBH_TRY(product(c, FB_GEMM_NN, Mat{g, Fp}, wg, dx, a.lddx, N, a.D, a.F, 0));
    FBH_TRY(product(c, FB_GEMM_NN, Mat{u, Fp}, wu, dx, a.lddx, N, a.D, a.F, 1));
  }
  auto grad = [&](const Mat &G, const Mat &X, void *o, int64_t ld, int rows, int cols) {
    return o ? product(c, FB_GEMM_TN, G, X, static_cast<float *>(o), ld, N, rows, cols, a.accumulate) : FB_OK;
  };
  FBH_TRY(grad(Mat{g, Fp}, x, a.dw_gate, a.ldd_gate, a.F, a.D));
  FBH_TRY(grad(Mat{u, Fp}, x, a.dw_up, a.ldd_up, a.F, a.D));
  return grad(dy, Mat{d, Fp}, a.dw_down, a.ldd_down, a.D, a.F);
}

// g and u (and dh) of every tile, the activation in the epilogue: h [N, Fp],
// and for the backward dgu [N, 2 Fp] = [dg | du].  Fp = F rounded up to 64;
// the padding columns are zeros (weight rows past F read as zeros).
template <int EPI>
int glu(Call &c, const fb_gated_ffn &a, const Mat &x, const Mat &dy, const Mat &wg, const Mat &wu, const Mat &wd,
        __nv_bfloat16 *h, __nv_bfloat16 *dgu, int64_t Fp) {
  using namespace fbpair;
  if (c.dry) return FB_OK;
  PairArgs p;
  std::memset(&p, 0, sizeof(p));
  p.phases = EPI == kGluBwd ? 2 : 1;
  p.probs = p.splits = 1;
  p.kb[0] = p.kb[1] = p.kper = tiles_of(a.D, BK);
  p.mt = tiles_of(a.n, 256);
  p.nt = tiles_of(Fp, 128);
  p.M = (int)a.n;
  p.N = (int)Fp;
  p.act = a.act;
  p.has_tc = 1;
  p.err = err_word();
  FBH_TRY(make_map(&p.ta[0], x.p, a.n, a.D, x.ld, kHalfM));
  FBH_TRY(make_map(&p.tb[0], wg.p, a.F, a.D, wg.ld, 128));
  FBH_TRY(make_map(&p.tb[1], wu.p, a.F, a.D, wu.ld, 128));
  FBH_TRY(make_map(&p.tc[0], h, a.n, Fp, Fp, 32, false, true));
  if (EPI == kGluBwd) {
    FBH_TRY(make_map(&p.ta[1], dy.p, a.n, a.D, dy.ld, kHalfM));
    FBH_TRY(make_map(&p.tw, wd.p, a.D, a.F, wd.ld, BK));
    FBH_TRY(make_map(&p.tc[1], dgu, a.n, Fp, 2 * Fp, 32, false, true));
    FBH_TRY(make_map(&p.tc[2], dgu + Fp, a.n, Fp, 2 * Fp, 32, false, true));
  }
  return launch_pair<EPI, false, false, 256>(p, c.stream);
}

int forward_bf16(Call &c, const fb_gated_ffn &a, const Mat &x, const Mat &wg, const Mat &wu, const Mat &wd) {
  const int64_t Fp = round_up(a.F, 64);
  FBH_TAKE(h, c, __nv_bfloat16, a.n * Fp);
  FBH_TRY(glu<fbpair::kGluFwd>(c, a, x, Mat{}, wg, wu, wd, h, nullptr, Fp));
  const Term t{wd, 0, a.F};
  return pair_rows(c, Mat{h, Fp}, a.n, a.F, &t, 1, false, a.D, Out{a.y, a.ldy, FB_BF16, 0});
}

int backward_bf16(Call &c, const fb_gated_ffn &a, const Mat &x, const Mat &dy, const Mat &wg, const Mat &wu,
                  const Mat &wd) {
  const int64_t Fp = round_up(a.F, 64);
  FBH_TAKE(h, c, __nv_bfloat16, a.n * Fp);
  FBH_TAKE(dgu, c, __nv_bfloat16, a.n * 2 * Fp);
  FBH_TRY(glu<fbpair::kGluBwd>(c, a, x, dy, wg, wu, wd, h, dgu, Fp));
  if (a.dx) {
    const Term t[2] = {{wg, 0, a.F}, {wu, (int)Fp, a.F}};
    FBH_TRY(pair_rows(c, Mat{dgu, 2 * Fp}, a.n, (int)(2 * Fp), t, 2, true, a.D, Out{a.dx, a.lddx, FB_BF16, 0}));
  }
  const Out og{a.dw_gate, a.ldd_gate, a.grad_type, a.accumulate}, ou{a.dw_up, a.ldd_up, a.grad_type, a.accumulate};
  const Out both[2] = {og, ou};
  if (a.dw_gate && a.dw_up) {
    FBH_TRY(pair_columns(c, Mat{dgu, 2 * Fp}, a.n, (int)(2 * Fp), (int)Fp, 2, a.F, x, a.D, both));
  } else if (a.dw_gate) {
    FBH_TRY(pair_columns(c, Mat{dgu, 2 * Fp}, a.n, a.F, 0, 1, a.F, x, a.D, &og));
  } else if (a.dw_up) {
    FBH_TRY(pair_columns(c, Mat{dgu + Fp, 2 * Fp}, a.n, a.F, 0, 1, a.F, x, a.D, &ou));
  }
  const Out od{a.dw_down, a.ldd_down, a.grad_type, a.accumulate};
  if (a.dw_down) FBH_TRY(pair_columns(c, dy, a.n, a.D, 0, 1, a.D, Mat{h, Fp}, a.F, &od));
  return FB_OK;
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
  Mat x, wg, wu, wd, dy{};
  FBH_TRY(aligned(c, a.type, Mat{a.x, a.ldx}, a.n, a.D, &x));
  FBH_TRY(aligned(c, a.type, Mat{a.w_gate, a.ld_gate}, a.F, a.D, &wg));
  FBH_TRY(aligned(c, a.type, Mat{a.w_up, a.ld_up}, a.F, a.D, &wu));
  FBH_TRY(aligned(c, a.type, Mat{a.w_down, a.ld_down}, a.D, a.F, &wd));
  if (!bwd) return a.type == FB_F32 ? forward_f32(c, a, x, wg, wu, wd) : forward_bf16(c, a, x, wg, wu, wd);
  FBH_TRY(aligned(c, a.type, Mat{a.dy, a.lddy}, a.n, a.D, &dy));
  return a.type == FB_F32 ? backward_f32(c, a, x, dy, wg, wu, wd) : backward_bf16(c, a, x, dy, wg, wu, wd);
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
