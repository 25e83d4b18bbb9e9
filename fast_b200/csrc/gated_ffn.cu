// Gated feed-forward block, forward and backward:
//   g = x Wg^T, u = x Wu^T, h = act(g) u, y = h Wd^T
//   dh = dy Wd, dg = dh u act'(g), du = dh act(g)
//   dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x, dWd = dy^T h
// Only x is kept between the two: the backward recomputes g and u.
//
// bf16: two launches forward, two backward (plus the sums of split
// reductions), each of products on SM pairs (pair_gemm.cuh).  The first of each
// direction computes g and u side by side in one tile -- one CTA of the pair
// stages Wg, the other Wu -- and for the backward dh beside them, and applies
// the activation to the fp32 accumulators: h, dg, du are rounded once, and g,
// u, dh never reach memory.  fp32: the same products over planes, with the
// activation between them in a kernel of its own.
#include "few_rows.cuh"
#include "pair_gemm.cuh"
#include "planes.cuh"

namespace {

using namespace fbh;

constexpr int kSilu = FB_ACT_SILU, kGelu = FB_ACT_GELU;

// fp32: h = act(g) u over rows x Fp elements, as planes; gu rows are [g | u].
template <int ACT> __global__ void __launch_bounds__(256) k_glu_fwd(const float *gu, uint16_t *h, int64_t rows, int Fp) {
  fb::pdl_enter();
  const int64_t n = rows * Fp;
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < n; i += (int64_t)gridDim.x * 1024) {
    const float *p = gu + i / Fp * 2 * Fp + i % Fp;
    const float4 g = *reinterpret_cast<const float4 *>(p), u = *reinterpret_cast<const float4 *>(p + Fp);
    fbplanes::put4(h + i, n, fbact::act_exact<ACT>(g.x).x * u.x, fbact::act_exact<ACT>(g.y).x * u.y,
                   fbact::act_exact<ACT>(g.z).x * u.z, fbact::act_exact<ACT>(g.w).x * u.w);
  }
}

// fp32: h, and dgu rows [dg | du], as planes, from gu rows [g | u] and dh.
template <int ACT>
__global__ void __launch_bounds__(256) k_glu_bwd(const float *gu, const float *dh, uint16_t *h, uint16_t *dgu, int64_t rows,
                                                 int Fp) {
  fb::pdl_enter();
  const int64_t n = rows * Fp;
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < n; i += (int64_t)gridDim.x * 1024) {
    const int64_t at = i / Fp * 2 * Fp + i % Fp;
    float g[4], u[4], d[4];
    *reinterpret_cast<float4 *>(g) = *reinterpret_cast<const float4 *>(gu + at);
    *reinterpret_cast<float4 *>(u) = *reinterpret_cast<const float4 *>(gu + at + Fp);
    *reinterpret_cast<float4 *>(d) = *reinterpret_cast<const float4 *>(dh + i);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 a = fbact::act_exact<ACT>(g[k]);
      g[k] = d[k] * u[k] * a.y;
      d[k] *= a.x;
      u[k] *= a.x;
    }
    fbplanes::put4(dgu + at, 2 * n, g[0], g[1], g[2], g[3]);
    fbplanes::put4(dgu + at + Fp, 2 * n, d[0], d[1], d[2], d[3]);
    fbplanes::put4(h + i, n, u[0], u[1], u[2], u[3]);
  }
}

unsigned blocks_for(int64_t n) { return (unsigned)std::max<int64_t>(1, std::min<int64_t>((n + 1023) / 1024, 148 * 8)); }

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

// fp32: g | u [N, 2 Fp] (and dh [N, Fp], from dy), then the activation; the
// padding columns up to Fp are zeros (weight rows past F read as zeros).
int gate_up_f32(Call &c, const fb_gated_ffn &a, const Mat &x, const Mat &wg, const Mat &wu, float *gu, int64_t Fp,
                const Mat *dy = nullptr, const Mat *wd = nullptr, float *dh = nullptr) {
  Product p[3] = {rows_product(x, a.n, a.D, wg, false, (int)Fp, Out{gu, 2 * Fp, FB_F32, 0}),
                  rows_product(x, a.n, a.D, wu, false, (int)Fp, Out{gu + Fp, 2 * Fp, FB_F32, 0})};
  if (dh) p[2] = rows_product(*dy, a.n, a.D, *wd, true, (int)Fp, Out{dh, Fp, FB_F32, 0});
  p[0].b_n = p[1].b_n = p[2].b_n = a.F;
  return products(c, p, dh ? 3 : 2);
}

int forward_f32(Call &c, const fb_gated_ffn &a, const Mat &x, const Mat &wg, const Mat &wu, const Mat &wd) {
  const int64_t Fp = round_up(a.F, 64);
  FBH_TAKE(gu, c, float, a.n * 2 * Fp);
  FBH_TAKE(h, c, uint16_t, 3 * a.n * Fp);
  FBH_TRY(gate_up_f32(c, a, x, wg, wu, gu, Fp));
  if (!c.dry) {
    auto k = a.act == kSilu ? k_glu_fwd<FB_ACT_SILU> : (a.act == kGelu ? k_glu_fwd<FB_ACT_GELU> : k_glu_fwd<FB_ACT_RELU>);
    FB_TRY_CUDA(fb::launch(k, blocks_for(a.n * Fp), 256, 0, c.stream, (const float *)gu, h, a.n, (int)Fp));
    FB_LAUNCHED("k_glu_fwd");
  }
  const Product p = rows_product(Mat{h, Fp, a.n * Fp}, a.n, a.F, wd, false, a.D, Out{a.y, a.ldy, FB_F32, 0});
  return products(c, &p, 1);
}

// g and u (and dh) of every tile, the activation in the epilogue: h [N, Fp],
// and for the backward dgu [N, 2 Fp] = [dg | du].  Fp = F rounded up to 64;
// the padding columns are zeros (weight rows past F read as zeros).
//
// ReLU's backward turns with the sign of g, and the tensor cores' accumulation truncates: it sums g and u in slabs of
// kGluSlab stages (kGluBwdLong) where D is longer than one.  The other activations' derivatives are smooth, and an error
// of g of some 2^-18 is lost in the rounding to bf16.  us of the whole backward, with slabs / without: 8,192 x 2,048 x
// 8,192 1,624 / 1,594; 1,500 x 1,024 x 2,000 64 / 64; 12,000 x 300 x 1,200 115 / 120.
template <int EPI>
int glu(Call &c, const fb_gated_ffn &a, const Mat &x, const Mat &dy, const Mat &wg, const Mat &wu, const Mat &wd,
        __nv_bfloat16 *h, __nv_bfloat16 *dgu, int64_t Fp) {
  using namespace fbpair;
  constexpr bool bwd = EPI == kGluBwd || EPI == kGluBwdLong;
  constexpr int dh = EPI == kGluBwd ? 0 : 1;   // the term of dh
  if (c.dry) return FB_OK;
  PairArgs p;
  one_product(p, a.n, Fp, 128, tiles_of(a.D, BK), bwd ? 2 : 1);
  p.act = a.act;
  PairProb &b = p.p[0];
  FBH_TRY(make_map(&b.ta[1 - dh], x.p, a.n, a.D, x.ld, kHalfM));
  FBH_TRY(make_map(&b.tb[0], wg.p, a.F, a.D, wg.ld, 128));
  FBH_TRY(make_map(&b.tb[1], wu.p, a.F, a.D, wu.ld, 128));
  FBH_TRY(make_map(&b.tc, h, a.n, Fp, Fp, 32));
  if (bwd) {
    FBH_TRY(make_map(&b.ta[dh], dy.p, a.n, a.D, dy.ld, kHalfM));
    FBH_TRY(make_map(&p.tw, wd.p, a.D, a.F, wd.ld, BK));
    FBH_TRY(make_map(&p.tc2[0], dgu, a.n, Fp, 2 * Fp, 32));
    FBH_TRY(make_map(&p.tc2[1], dgu + Fp, a.n, Fp, 2 * Fp, 32));
  }
  return launch_pair<EPI>(p, c.stream);
}

int forward_bf16(Call &c, const fb_gated_ffn &a, const Mat &x, const Mat &wg, const Mat &wu, const Mat &wd) {
  const int64_t Fp = round_up(a.F, 64);
  FBH_TAKE(h, c, __nv_bfloat16, a.n * Fp);
  FBH_TRY(glu<fbpair::kGluFwd>(c, a, x, Mat{}, wg, wu, wd, h, nullptr, Fp));
  const Product p = rows_product(Mat{h, Fp}, a.n, a.F, wd, false, a.D, Out{a.y, a.ldy, FB_BF16, 0});
  return products(c, &p, 1);
}

// dx and the weight gradients from h [n, Fp] and dgu [n, 2 Fp].
int gradients(Call &c, const fb_gated_ffn &a, const Mat &x, const Mat &dy, const Mat &wg, const Mat &wu, const Mat &h,
              const Mat &dgu, int64_t Fp) {
  const Mat du{static_cast<const uint16_t *>(dgu.p) + Fp, dgu.ld, dgu.plane};
  auto grad = [&](void *p, int64_t ld) { return Out{p, ld, a.grad_type, a.accumulate}; };
  Product dx = rows_product(dgu, a.n, a.F, wg, true, a.D, Out{a.dx, a.lddx, a.type, 0});
  dx.acols = (int)(2 * Fp);
  dx.term[1] = Term{wu, (int)Fp, a.F};
  dx.terms = 2;
  const Product p[4] = {dx, columns_product(dgu, a.n, a.F, x, a.D, grad(a.dw_gate, a.ldd_gate)),
                        columns_product(du, a.n, a.F, x, a.D, grad(a.dw_up, a.ldd_up)),
                        columns_product(dy, a.n, a.D, h, a.F, grad(a.dw_down, a.ldd_down))};
  return products(c, p, 4);
}

int backward_f32(Call &c, const fb_gated_ffn &a, const Mat &x, const Mat &dy, const Mat &wg, const Mat &wu,
                 const Mat &wd) {
  const int64_t Fp = round_up(a.F, 64), n = a.n * Fp;
  FBH_TAKE(gu, c, float, 2 * n);
  FBH_TAKE(dh, c, float, n);
  FBH_TAKE(h, c, uint16_t, 3 * n);
  FBH_TAKE(dgu, c, uint16_t, 6 * n);
  FBH_TRY(gate_up_f32(c, a, x, wg, wu, gu, Fp, &dy, &wd, dh));
  if (!c.dry) {
    auto k = a.act == kSilu ? k_glu_bwd<FB_ACT_SILU> : (a.act == kGelu ? k_glu_bwd<FB_ACT_GELU> : k_glu_bwd<FB_ACT_RELU>);
    FB_TRY_CUDA(fb::launch(k, blocks_for(n), 256, 0, c.stream, (const float *)gu, (const float *)dh, h, dgu, a.n,
                           (int)Fp));
    FB_LAUNCHED("k_glu_bwd");
  }
  return gradients(c, a, x, dy, wg, wu, Mat{h, Fp, n}, Mat{dgu, 2 * Fp, 2 * n}, Fp);
}

int backward_bf16(Call &c, const fb_gated_ffn &a, const Mat &x, const Mat &dy, const Mat &wg, const Mat &wu,
                  const Mat &wd) {
  const int64_t Fp = round_up(a.F, 64);
  FBH_TAKE(h, c, __nv_bfloat16, a.n * Fp);
  FBH_TAKE(dgu, c, __nv_bfloat16, a.n * 2 * Fp);
  const bool slabs = a.act == FB_ACT_RELU && a.D > fbpair::kGluSlab * fbpair::BK;
  FBH_TRY(slabs ? glu<fbpair::kGluBwdLong>(c, a, x, dy, wg, wu, wd, h, dgu, Fp)
                : glu<fbpair::kGluBwd>(c, a, x, dy, wg, wu, wd, h, dgu, Fp));
  return gradients(c, a, x, dy, wg, wu, Mat{h, Fp}, Mat{dgu, 2 * Fp}, Fp);
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
  if (bwd && few_rows_ok(a.type, bwd, a.n, a.D, (int64_t)a.D * a.F) && a.F <= kFewRowsTable)
    return few_rows_ffn_bwd(c, a);
  if (!bwd && few_rows_ok(a.type, bwd, a.n, std::max(a.D, a.F), (int64_t)a.D * a.F)) {
    FBH_TAKE(h, c, float, a.n * a.F);
    FBH_TRY(few_rows_glu(c, a.type, a.act, Mat{a.x, a.ldx}, a.n, a.D, Mat{a.w_gate, a.ld_gate}, Mat{a.w_up, a.ld_up}, a.F,
                         h));
    return few_rows_product(c, a.type, h, a.n, a.F, Mat{a.w_down, a.ld_down}, a.D, a.y, a.ldy);
  }
  Mat x, wg, wu, wd, dy{};
  const Operand ops[5] = {{Mat{a.x, a.ldx}, a.n, a.D, &x}, {Mat{a.w_gate, a.ld_gate}, a.F, a.D, &wg},
                          {Mat{a.w_up, a.ld_up}, a.F, a.D, &wu}, {Mat{a.w_down, a.ld_down}, a.D, a.F, &wd},
                          {Mat{a.dy, a.lddy}, a.n, a.D, &dy}};
  FBH_TRY(operands(c, a.type, ops, bwd ? 5 : 4));
  if (!bwd) return a.type == FB_F32 ? forward_f32(c, a, x, wg, wu, wd) : forward_bf16(c, a, x, wg, wu, wd);
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
  FBH_TRY(check_ws(ws, "gated_ffn_fwd"));
  Call c(ws, ws_bytes, stream);
  return run(c, *a, false);
}

extern "C" int fb_gated_ffn_bwd(const fb_gated_ffn *a, void *ws, size_t ws_bytes, cudaStream_t stream) {
  FBH_TRY(check(a, true));
  if (a->n == 0) return empty_grads(*a, stream);
  FBH_TRY(check_ws(ws, "gated_ffn_bwd"));
  Call c(ws, ws_bytes, stream);
  return run(c, *a, true);
}
