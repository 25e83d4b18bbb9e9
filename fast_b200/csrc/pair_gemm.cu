// Plain products of the node-ranking head on pairs of SMs (pair_gemm.cuh), and
// the sum of their partial results when the reduction is split.
#include "pair_gemm.cuh"

namespace {

using namespace fbpair;
using namespace fbh;

// out (+)= sum over splits of P[s], in split order; P rows have pitch ldp.
// blockIdx.y: the problem.
struct SumArgs {
  const float *P[2];
  void *out[2];
  int64_t ldo[2];
  int64_t split_stride, ldp, rows;
  int splits, cols, accumulate;
};
template <bool kBf16> __global__ void __launch_bounds__(256) k_sum_splits(const __grid_constant__ SumArgs a) {
  fb::pdl_enter();
  const float *const P = a.P[blockIdx.y];
  void *const out = a.out[blockIdx.y];
  const int64_t ldo = a.ldo[blockIdx.y], ldp = a.ldp, split_stride = a.split_stride, rows = a.rows;
  const int splits = a.splits, cols = a.cols, accumulate = a.accumulate;
  const int64_t total = rows * cols;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / cols;
    const int c = (int)(i - r * cols);
    const float *p = P + r * ldp + c;
    float s = 0.f;
    int z = 0;
    for (; z + 8 <= splits; z += 8) {
      float v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = p[(z + u) * split_stride];
#pragma unroll
      for (int u = 0; u < 8; ++u) s += v[u];
    }
    for (; z < splits; ++z) s += p[z * split_stride];
    if (kBf16) {
      static_cast<__nv_bfloat16 *>(out)[r * ldo + c] = __float2bfloat16_rn(s);
    } else {
      float *o = static_cast<float *>(out) + r * ldo + c;
      *o = accumulate ? *o + s : s;
    }
  }
}

int sum_splits(Call &c, SumArgs a, int probs, int type) {
  const dim3 grid((unsigned)std::max<int64_t>(1, std::min<int64_t>((a.rows * a.cols + 255) / 256, 148 * 16)), probs);
  if (type == FB_BF16) FB_TRY_CUDA(fb::launch(k_sum_splits<true>, grid, 256, 0, c.stream, a));
  else FB_TRY_CUDA(fb::launch(k_sum_splits<false>, grid, 256, 0, c.stream, a));
  FB_LAUNCHED("k_sum_splits");
  return FB_OK;
}

// Tile width and splits for results of M x N over kb stages.  256 columns keep
// the tensor cores fed; a grid that would leave half the SM pairs idle takes
// 128-column tiles, then splits the reduction, at least min_stages a split (a
// stage of planes is six products).
constexpr int min_stages(bool planes) { return planes ? 2 : 4; }
struct Plan {
  int bn, splits, kper;
};
Plan plan_of(int64_t M, int N, int probs, int kb, bool planes) {
  const int slots = num_sms() / 2;
  Plan p{N > 128 && !planes ? 256 : 128, 1, kb};
  const int64_t mt = tiles_of(M, 256);
  if (p.bn == 256 && mt * tiles_of(N, 256) * probs * 2 <= slots) p.bn = 128;
  const int64_t tiles = mt * tiles_of(N, p.bn) * probs;
  if (tiles * 2 <= slots) {
    const int s = (int)std::min<int64_t>(slots / tiles, kb / min_stages(planes));
    if (s > 1) {
      p.kper = (kb + s - 1) / s;
      p.splits = tiles_of(kb, p.kper);
    }
  }
  return p;
}

template <bool A_MN, bool B_MN> int dispatch(const PairArgs &a, int bn, bool f32, bool planes, cudaStream_t st) {
  if (planes) return launch_pair<kStoreF32, A_MN, B_MN, 128, 3>(a, st);
  if (f32)
    return bn == 256 ? launch_pair<kStoreF32, A_MN, B_MN, 256>(a, st) : launch_pair<kStoreF32, A_MN, B_MN, 128>(a, st);
  return bn == 256 ? launch_pair<kStoreBf16, A_MN, B_MN, 256>(a, st) : launch_pair<kStoreBf16, A_MN, B_MN, 128>(a, st);
}

// Fills the tiling and the outputs (or the partial results') of `a`, launches, sums the splits.
template <bool A_MN, bool B_MN> int finish(Call &c, PairArgs &a, const Plan &p, bool planes, int64_t M, int N, const Out *out) {
  a.mt = tiles_of(M, 256);
  a.nt = tiles_of(N, p.bn);
  a.splits = p.splits;
  a.kper = p.kper;
  a.M = (int)M;
  a.N = N;
  a.err = c.dry ? nullptr : err_word();
  const int64_t prow = (int64_t)a.mt * 256, pld = round_up(N, 4);
  float *P[2] = {nullptr, nullptr};
  const size_t mark = c.off;
  if (p.splits > 1)
    for (int i = 0; i < a.probs; ++i) {
      P[i] = static_cast<float *>(c.take((size_t)(p.splits * prow * pld) * 4));
      if (!P[i]) return fb::set_error(FB_ERR_ARG, "workspace too small");
    }
  c.off = mark;
  if (c.dry) return FB_OK;
  const bool f32 = p.splits > 1 || out[0].type == FB_F32;
  a.has_tc = 1;
  a.accumulate = p.splits > 1 ? 0 : out[0].accumulate;
  a.split_rows = prow;
  for (int i = 0; i < a.probs; ++i) {
    if (p.splits > 1) {
      FBH_TRY(make_map(&a.tc[i], P[i], p.splits * prow, N, pld, 32, true));
    } else {
      a.C[i] = out[i].p;
      a.ldc = out[i].ld;
      if (out[i].ld != out[0].ld || !map_ok(out[i].p, out[i].ld, f32 ? 4 : 2)) a.has_tc = 0;
    }
  }
  if (p.splits == 1 && a.has_tc)
    for (int i = 0; i < a.probs; ++i) FBH_TRY(make_map(&a.tc[i], out[i].p, M, N, out[i].ld, 32, f32));
  FBH_TRY((dispatch<A_MN, B_MN>(a, p.bn, f32, planes, c.stream)));
  if (p.splits == 1) return FB_OK;
  SumArgs sa{{P[0], P[1]}, {out[0].p, nullptr}, {out[0].ld, 0}, prow * pld, pld, M, p.splits, N, out[0].accumulate};
  if (a.probs > 1) sa.out[1] = out[1].p, sa.ldo[1] = out[1].ld;
  return sum_splits(c, sa, a.probs, out[0].type);
}

int operand_map(CUtensorMap *m, const Mat &x, int64_t rows, int64_t cols, int box_rows) {
  return x.plane ? make_map3(m, x.p, rows, cols, x.ld, x.plane, box_rows) : make_map(m, x.p, rows, cols, x.ld, box_rows);
}

}  // namespace

namespace fbh {

int pair_rows(Call &c, const Mat &A, int64_t M, int acols, const Term *terms, int n_terms, bool b_mn, int N,
              const Out &out, int b_n) {
  if (M == 0) return FB_OK;
  if (!b_n) b_n = N;
  PairArgs a;
  std::memset(&a, 0, sizeof(a));
  a.phases = n_terms;
  a.probs = 1;
  for (int t = 0; t < n_terms; ++t) {
    a.kb[t] = tiles_of(terms[t].K, BK);
    a.ax[t] = terms[t].ax;
  }
  const Plan p = plan_of(M, N, 1, a.kb[0] + a.kb[1], A.plane > 0);
  if (!c.dry)
    for (int t = 0; t < n_terms; ++t) {
      FBH_TRY(operand_map(&a.ta[t], A, M, acols, kHalfM));
      if (b_mn) FBH_TRY(operand_map(&a.tb[t], terms[t].B, terms[t].K, b_n, BK));
      else FBH_TRY(operand_map(&a.tb[t], terms[t].B, b_n, terms[t].K, p.bn / 2));
    }
  return b_mn ? finish<false, true>(c, a, p, A.plane > 0, M, N, &out) : finish<false, false>(c, a, p, A.plane > 0, M, N, &out);
}

int pair_rows2(Call &c, const Mat &A, int64_t M, const Mat *B, int K, int N, const Out *out, int b_n) {
  if (M == 0) return FB_OK;
  PairArgs a;
  std::memset(&a, 0, sizeof(a));
  a.phases = 1;
  a.probs = 2;
  a.bprob = 1;
  a.kb[0] = tiles_of(K, BK);
  const Plan p = plan_of(M, N, 2, a.kb[0], A.plane > 0);
  if (!c.dry) {
    FBH_TRY(operand_map(&a.ta[0], A, M, K, kHalfM));
    for (int i = 0; i < 2; ++i) FBH_TRY(operand_map(&a.tb[i], B[i], b_n, K, p.bn / 2));
  }
  return finish<false, false>(c, a, p, A.plane > 0, M, N, out);
}

int pair_columns(Call &c, const Mat &A, int64_t rows, int acols, int aprob, int probs, int M, const Mat &B, int N,
                 const Out *out) {
  PairArgs a;
  std::memset(&a, 0, sizeof(a));
  a.phases = 1;
  a.probs = probs;
  a.aprob = aprob;
  a.kb[0] = tiles_of(rows, BK);
  const Plan p = plan_of(M, N, probs, a.kb[0], A.plane > 0);
  if (!c.dry) {
    FBH_TRY(operand_map(&a.ta[0], A, rows, acols, BK));
    FBH_TRY(operand_map(&a.tb[0], B, rows, N, BK));
  }
  return finish<true, true>(c, a, p, A.plane > 0, M, N, out);
}

}  // namespace fbh
