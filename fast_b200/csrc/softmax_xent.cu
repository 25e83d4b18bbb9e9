// Softmax cross entropy of rows h [n, D] against every row of a table w [V, D]:
//   l = h w^T,  lse_i = log sum_v exp(l_iv),  loss_i = lse_i - l_i,target
//   G = dloss_i (exp(l_iv - lse_i) - [v == target]),  dh = G w,  dw = G^T h
// The logits are not kept (but see few_tiles()).  The products run on SM pairs (pair_gemm.cuh), fp32
// rows as three bf16 planes: the forward reduces every tile of logits to a
// maximum and a sum per row in its epilogue, one launch over the whole table,
// and a second kernel joins them; the backward takes the table in pieces of as
// many rows as make a G piece of kPieceBytes, computes G from the logits in the
// epilogue that would have stored them, then adds G w to dh and writes G^T h.
#include <cmath>
#include "few_rows.cuh"
#include "pair_gemm.cuh"

namespace {

using namespace fbh;

// Memory of a piece of G (bf16: 2 bytes an element, fp32: its planes' 6).  A
// piece that stays in the 126 MB L2 was expected to pay, but its products are
// short: 48 / 160 / 512 MB a piece took 160 / 110 / 110 us for 4,000 rows x
// 16,700 nodes x 104 and 2.45 / 2.22 / 2.13 ms for 8,192 x 50,000 x 1,024 (bf16);
// beyond that little changes and memory is not given back.
constexpr int64_t kPieceBytes = 512ll << 20;
constexpr int64_t kPartBytes = 256ll << 20;   // of the forward's partials

__device__ __forceinline__ float value(const float *p) { return *p; }
__device__ __forceinline__ float value(const uint16_t *p) { return __uint_as_float((uint32_t)*p << 16); }   // bf16

// TH threads (a warp, or a CTA of 256 where rows are few and latency counts)
// join a row's partial (max, sum of exp2) pairs, take the target's logit as an
// fp32 dot product of its own, and write lse and loss.
template <typename U, int TH>
__global__ void __launch_bounds__(TH == 32 ? 128 : TH) k_xent_finish(const float2 *part, int np, const U *h, int64_t ldh,
                                                                     const U *w, int64_t ldw, int D, int64_t V,
                                                                     const int64_t *target, float *loss, float *lse,
                                                                     int64_t n) {
  __shared__ float3 sm[TH / 32];
  fb::pdl_enter();
  const int64_t r = TH == 32 ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x;
  const int t = threadIdx.x % TH;
  if (r >= n) return;
  const int64_t tg = target[r];
  const float2 *p = part + r * np;
  float m = -INFINITY, s = 0.f, l = 0.f;
#pragma unroll 2
  for (int i = t; i < np; i += TH) {
    const float2 q = p[i];
    const float nm = fmaxf(m, q.x), base = nm == -INFINITY ? 0.f : nm;
    s = s * exp2f(m - base) + q.y * exp2f(q.x - base);
    m = nm;
  }
  if (tg >= 0 && tg < V)
#pragma unroll 4
    for (int i = t; i < D; i += TH) l = fmaf(value(h + r * ldh + i), value(w + tg * ldw + i), l);
  auto fold = [&](float m2, float s2) {
    const float nm = fmaxf(m, m2), base = nm == -INFINITY ? 0.f : nm;
    s = s * exp2f(m - base) + s2 * exp2f(m2 - base);
    m = nm;
  };
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
    fold(m2, s2);
  }
  l = fb::warp_sum(l);
  if (TH > 32) {
    if ((t & 31) == 0) sm[t / 32] = make_float3(m, s, l);
    __syncthreads();
    if (t) return;
#pragma unroll
    for (int q = 1; q < TH / 32; ++q) {
      fold(sm[q].x, sm[q].y);
      l += sm[q].z;
    }
  }
  if (t) return;
  const float z = (m + log2f(s)) * 0.69314718055994530942f;
  lse[r] = z;
  loss[r] = tg < 0 ? 0.f : (tg >= V ? NAN : z - l);
}

// fp32 rows of few tiles (few_tiles()): from stored logits [n, ldl], ldl a multiple of 4.  A warp reduces an eighth of
// a row to its partial (max, sum of exp2), as the products' epilogue would have.
__global__ void __launch_bounds__(256) k_logit_parts(const float *l, int64_t ldl, int V, float2 *part) {
  constexpr float kLog2e = 1.44269504088896340736f;
  fb::pdl_enter();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float *p = l + blockIdx.x * ldl;
  float m = -INFINITY, s = 0.f;
  auto fold = [&](float m2, float s2) {
    const float nm = fmaxf(m, m2), base = nm == -INFINITY ? 0.f : nm;    // nothing but -inf: zeros, and NaN stays NaN
    s = s * exp2f(m - base) + s2 * exp2f(m2 - base);
    m = nm;
  };
  for (int c = warp * 32 + lane; c < V; c += 256) {
    const float v = p[c];
    const float nm = fmaxf(m, v * kLog2e), base = nm == -INFINITY ? 0.f : nm;
    s = s * exp2f(m - base) + exp2f(fmaf(v, kLog2e, -base));
    m = nm;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
    fold(m2, s2);
  }
  if (lane == 0) part[(int64_t)blockIdx.x * 8 + warp] = make_float2(m, s);
}

// The planes of G, pitch ldl as the logits'; columns past V are never read.
__global__ void __launch_bounds__(256) k_logit_grad(const float *l, int64_t ldl, int V, const int64_t *target,
                                                    const float *lse, const float *dloss, uint16_t *G, int64_t plane) {
  fb::pdl_enter();
  const int64_t r = blockIdx.x, t = target[r];
  const bool live = t >= 0 && t < V;          // a held-out row is zeros whatever its logits are
  const float z = lse[r], d = dloss[r];
  const int c = (blockIdx.y * 256 + threadIdx.x) * 4;
  if (c >= V) return;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  if (live) {
    *reinterpret_cast<float4 *>(v) = *reinterpret_cast<const float4 *>(l + r * ldl + c);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = d * (expf(v[k] - z) - (t == c + k ? 1.f : 0.f));
  }
  fbplanes::put4(G + r * ldl + c, plane, v[0], v[1], v[2], v[3]);
}

// bf16 rows: dst = src rounded.
__global__ void k_round_rows(const float *src, int64_t lds, __nv_bfloat16 *dst, int64_t ldd, int64_t rows, int cols) {
  fb::pdl_enter();
  const int64_t total = rows * cols;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / cols;
    const int c = (int)(i - r * cols);
    dst[r * ldd + c] = __float2bfloat16_rn(src[r * lds + c]);
  }
}

// Table rows per piece: a multiple of 64, so that pieces start 16-byte aligned.
int64_t piece_rows(int64_t n, int64_t V, int bytes) {
  const int64_t r = std::max<int64_t>(256, kPieceBytes / bytes / std::max<int64_t>(n, 1) / 64 * 64);
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

Mat rows_from(const Mat &m, int64_t r) { return Mat{static_cast<const uint16_t *>(m.p) + r * m.ld, m.ld, m.plane}; }

// The common fields of a launch over the logits of rows h against table rows w.
int logits_args(fbpair::PairArgs &p, const fb_softmax_xent &a, const Mat &h, int64_t n, const Mat &w, int cols) {
  using namespace fbpair;
  const bool planes = h.plane > 0;
  one_product(p, n, cols, planes ? 128 : 256, tiles_of(a.D, BK), 1);
  FBH_TRY(operand_map(&p.p[0].ta[0], h, n, a.D, kHalfM));
  return operand_map(&p.p[0].tb[0], w, cols, a.D, planes ? 64 : 128);
}

// fp32 rows whose logits make too few tiles for the SM pairs, of sums long enough to be split: the launches that keep
// no logits do not split them, so here the logits are stored (a few MB) and read again.
// us, stored / not, forward and backward together, rows x width, nodes: 548 x 3,942, 657 (18 tiles) 118 / 180;
// 100 x 2,048, 1,000 (8) 52 / 89; 200 x 600, 1,000 (8) 45 / 48; with 36 tiles, at 200 rows and 4,600 nodes, 255 / 274 for
// 4,096 columns but 162 / 159 for 2,048 and 92 / 87 for 1,024.
bool few_tiles(const fb_softmax_xent &a) {
  return a.type == FB_F32 && a.D > 8 * fbpair::BK &&
         ((a.n + 255) / 256) * ((a.V + 127) / 128) * 4 <= fbtc::num_sms() / 2;
}
// bf16 gradients of few rows hang on few elements of G (the targets', near -1), whose rounding to bf16 would not average
// out: 3 rows against 895 nodes of width 257 were 0.0033 off in the 2-norm, 0.0017 of it the gradients' own rounding.
// While twice the rows still make one 256-row tile, G is kept as two bf16 parts, the second below the first, against h
// laid out twice (dw) and with the halves of dh added at the end.
// us, forward and backward, two parts / one, 16 rows: 100 x 10,000 32.9 / 30.4, 1,024 x 50,000 107 / 105; 128 rows:
// 35.6 / 32.5, 122 / 112.  For more rows the products would cost twice, and the rounding of their more elements averages.
bool two_parts(const fb_softmax_xent &a) { return a.type == FB_BF16 && a.n <= fbpair::kHalfM; }
int stored_logits(Call &c, const fb_softmax_xent &a, const Mat &h, const Mat &w, float *l, int64_t ldl) {
  const Product p = rows_product(h, a.n, a.D, w, false, (int)a.V, Out{l, ldl, FB_F32, 0});
  return products(c, &p, 1);
}

// lse and loss of rows r0 .. r0 + n - 1 (h: those rows) from their partials.
template <typename U>
int finish(Call &c, const fb_softmax_xent &a, const float2 *part, int np, const Mat &h, const Mat &w, int64_t r0,
           int64_t n) {
  const bool wide = n <= 1024;
  FB_TRY_CUDA(fb::launch(wide ? k_xent_finish<U, 256> : k_xent_finish<U, 32>, (unsigned)(wide ? n : (n + 3) / 4),
                         wide ? 256 : 128, 0, c.stream, part, np, static_cast<const U *>(h.p), h.ld,
                         static_cast<const U *>(w.p), w.ld, a.D, a.V, a.target + r0, a.loss + r0, a.lse + r0, n));
  FB_LAUNCHED("k_xent_finish");
  return FB_OK;
}

int forward_few(Call &c, const fb_softmax_xent &a) {
  const Mat h{a.h, a.ldh}, w{a.w, a.ldw};
  const int np = few_rows_parts();
  FBH_TAKE(part, c, float2, a.n * np);
  FBH_TRY(few_rows_lse(c, a.type, h, a.n, a.D, w, a.V, part));
  if (c.dry) return FB_OK;
  return a.type == FB_F32 ? finish<float>(c, a, part, np, h, w, 0, a.n) : finish<uint16_t>(c, a, part, np, h, w, 0, a.n);
}

int forward(Call &c, const fb_softmax_xent &a, const Mat &h, const Mat &w) {
  using namespace fbpair;
  if (few_tiles(a)) {
    const int64_t ldl = round_up(a.V, 64);
    FBH_TAKE(l, c, float, a.n * ldl);
    FBH_TAKE(part, c, float2, a.n * 8);
    FBH_TRY(stored_logits(c, a, h, w, l, ldl));
    if (c.dry) return FB_OK;
    FB_TRY_CUDA(fb::launch(k_logit_parts, (unsigned)a.n, 256, 0, c.stream, (const float *)l, ldl, (int)a.V, part));
    FB_LAUNCHED("k_logit_parts");
    return finish<float>(c, a, part, 8, Mat{a.h, a.ldh}, Mat{a.w, a.ldw}, 0, a.n);
  }
  const bool f32 = a.type == FB_F32, longer = !f32 && tiles_of(a.D, BK) > kLseSlab;
  const int64_t np = (int64_t)tiles_of(a.V, f32 ? 128 : 256) * (longer ? 4 : 2);   // partials of a row
  // rows per launch: the partials of one stay within kPartBytes
  const int64_t rows = std::min<int64_t>(a.n, std::max<int64_t>(256, kPartBytes / (8 * np) / 256 * 256));
  FBH_TAKE(part, c, float2, rows * np);
  if (c.dry) return FB_OK;
  for (int64_t r0 = 0; r0 < a.n; r0 += rows) {
    const int64_t n = std::min(rows, a.n - r0);
    const Mat hp = rows_from(h, r0);
    PairArgs p;
    FBH_TRY(logits_args(p, a, hp, n, w, (int)a.V));
    p.part = part;
    if (f32) {
      FBH_TRY((launch_pair<kLsePlanes, 3>(p, c.stream)));
      FBH_TRY(finish<float>(c, a, part, (int)np, Mat{static_cast<const float *>(a.h) + r0 * a.ldh, a.ldh}, Mat{a.w, a.ldw},
                            r0, n));
    } else {
      FBH_TRY(longer ? launch_pair<kLseLong>(p, c.stream) : launch_pair<kLse>(p, c.stream));
      FBH_TRY(finish<uint16_t>(c, a, part, (int)np, hp, w, r0, n));
    }
  }
  return FB_OK;
}

int backward(Call &c, const fb_softmax_xent &a, const Mat &h, const Mat &w) {
  using namespace fbpair;
  const bool f32 = a.type == FB_F32, two = two_parts(a);
  const int np = f32 ? 3 : (two ? 2 : 1);     // planes of G; two: its parts one below the other
  const int64_t gn = two ? 2 * a.n : a.n;     // rows of G (and of h) to the products
  const int64_t pr = piece_rows(a.n, a.V, 2 * np);
  const bool sum = !f32 && a.dh && pr < a.V;  // bf16 dh adds up over the pieces in fp32
  FBH_TAKE(G, c, uint16_t, np * a.n * pr);
  const bool few = few_tiles(a);
  float *l = nullptr;                         // few: the logits
  if (few) {
    FBH_TAKE(t, c, float, a.n * pr);
    l = t;
  }
  const int64_t lds = round_up(a.D, 4);
  float *acc = nullptr;
  if (sum) {
    FBH_TAKE(t, c, float, a.n * lds);
    acc = t;
  }
  for (int64_t v0 = 0; v0 < a.V; v0 += pr) {
    const int cols = (int)std::min<int64_t>(pr, a.V - v0);
    const Mat wp = rows_from(w, v0), Gm{G, pr, f32 ? a.n * pr : 0};
    if (few) {                                // one piece
      FBH_TRY(stored_logits(c, a, h, w, l, pr));
      if (!c.dry) {
        FB_TRY_CUDA(fb::launch(k_logit_grad, dim3((unsigned)a.n, (unsigned)((a.V + 1023) / 1024)), 256, 0, c.stream,
                               (const float *)l, pr, (int)a.V, a.target, (const float *)a.lse, a.dloss, G, a.n * pr));
        FB_LAUNCHED("k_logit_grad");
      }
    } else if (!c.dry) {
      PairArgs p;
      FBH_TRY(logits_args(p, a, h, a.n, wp, cols));
      p.target = a.target;
      p.lse = a.lse;
      p.dloss = a.dloss;
      p.V = a.V;
      p.v0 = v0;
      for (int k = 0; k < np; ++k)
        FBH_TRY(make_map(k == 0 ? &p.p[0].tc : &p.tc2[k - 1], G + k * a.n * pr, a.n, cols, pr, 32));
      FBH_TRY(f32 ? (launch_pair<kProbPlanes, 3>(p, c.stream))
                  : (two ? launch_pair<kProbTwo>(p, c.stream) : launch_pair<kProb>(p, c.stream)));
    }
    void *dw = a.dw ? static_cast<uint8_t *>(a.dw) + v0 * a.lddw * elem(a.grad_type) : nullptr;
    const Out dh = sum ? Out{acc, lds, FB_F32, v0 > 0} : Out{a.dh, a.lddh, a.type, f32 && v0 > 0};
    Product p[2] = {rows_product(Gm, gn, cols, wp, true, a.D, dh),
                    columns_product(Gm, gn, cols, h, a.D, Out{dw, a.lddw, a.grad_type, a.accumulate})};
    p[0].fold = two;
    FBH_TRY(products(c, p, 2));
    // dry: every piece takes the first one's workspace but the last, shorter one, which may split its sums differently
    if (c.dry && v0 == 0) v0 = std::max<int64_t>(0, (a.V - 1) / pr * pr - pr);
  }
  if (sum && !c.dry) {
    const unsigned blocks = (unsigned)std::max<int64_t>(1, std::min<int64_t>((a.n * a.D + 255) / 256, 148 * 16));
    FB_TRY_CUDA(fb::launch(k_round_rows, blocks, 256, 0, c.stream, (const float *)acc, lds,
                           static_cast<__nv_bfloat16 *>(a.dh), a.lddh, a.n, a.D));
    FB_LAUNCHED("k_round_rows");
  }
  return FB_OK;
}

int run(Call &c, const fb_softmax_xent &a, bool bwd) {
  if (few_rows_ok(a.type, bwd, a.n, a.D, a.D * a.V) && (!bwd || a.V <= kFewRowsTable))
    return bwd ? few_rows_xent_bwd(c, a) : forward_few(c, a);
  Mat h, w;
  // dw sums over the rows, so rows held out are zeros to it (bf16 rows that could be read where they lie are copied for
  // that: 4,000 x 100 against 16,700 nodes, training, 141 us before that copy and 139 with it; 8,192 x 1,024 against
  // 50,000, 2.73 and 2.71 ms)
  Operand ops[2] = {{Mat{a.h, a.ldh}, a.n, a.D, &h}, {Mat{a.w, a.ldw}, a.V, a.D, &w}};
  if (bwd && a.dw) ops[0].target = a.target, ops[0].V = a.V, ops[0].twice = two_parts(a);
  FBH_TRY(operands(c, a.type, ops, 2));
  return bwd ? backward(c, a, h, w) : forward(c, a, h, w);
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
  FBH_TRY(check_ws(ws, "softmax_xent_fwd"));
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
  FBH_TRY(check_ws(ws, "softmax_xent_bwd"));
  Call c(ws, ws_bytes, stream);
  return run(c, *a, true);
}
