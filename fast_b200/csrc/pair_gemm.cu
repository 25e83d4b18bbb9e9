// Plain products of the node-ranking head on pairs of SMs (pair_gemm.cuh), and
// the sum of their partial results where the reduction is split.
#include "pair_gemm.cuh"

namespace {

using namespace fbpair;
using namespace fbh;

// out (+)= sum over splits of P[s], in split order; P rows have pitch ldp.  fold > 0: and of the values `fold`
// elements further on, a sum of its own.
struct SumJob {
  const float *P;
  void *out;
  int64_t ldo, ldp, split_stride, rows, fold;
  int splits, cols, accumulate, bf16;
  unsigned first;                              // first CTA of the job
};
struct SumArgs {
  SumJob j[kMaxProbs];
  int n;
};
constexpr int kSumPerCta = 256;

__global__ void __launch_bounds__(kSumPerCta) k_sum_splits(const __grid_constant__ SumArgs a) {
  fb::pdl_enter();
  int q = 0;
  while (q + 1 < a.n && blockIdx.x >= a.j[q + 1].first) ++q;
  const SumJob &j = a.j[q];
  const int64_t i = (int64_t)(blockIdx.x - j.first) * kSumPerCta + threadIdx.x, stride = j.split_stride;
  if (i >= j.rows * j.cols) return;
  const int64_t r = i < ((int64_t)1 << 31) ? (int64_t)((uint32_t)i / (uint32_t)j.cols) : i / j.cols;
  const int c = (int)(i - r * j.cols);
  const float *p = j.P + r * j.ldp + c;
  auto total = [&](const float *p) {
    float s = 0.f;
    int z = 0;
    for (; z + 8 <= j.splits; z += 8) {
      float v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = p[(z + u) * stride];
#pragma unroll
      for (int u = 0; u < 8; ++u) s += v[u];
    }
    if (z < j.splits) {                        // the last few at once too
      float v[7];
#pragma unroll
      for (int u = 0; u < 7; ++u) v[u] = z + u < j.splits ? p[(z + u) * stride] : 0.f;
#pragma unroll
      for (int u = 0; u < 7; ++u) s += v[u];
    }
    return s;
  };
  float s = total(p);
  if (j.fold) s += total(p + j.fold);
  if (j.bf16) {
    static_cast<__nv_bfloat16 *>(j.out)[r * j.ldo + c] = __float2bfloat16_rn(s);
  } else {
    float *o = static_cast<float *>(j.out) + r * j.ldo + c;
    *o = j.accumulate ? *o + s : s;
  }
}

// Tile widths and splits of a launch's products.  256 columns keep the tensor
// cores fed; where that leaves half the SM pairs idle, 128.  Reductions are
// split into parts of about `part` stages, at least min_stages (a stage of
// planes is six products); of a few part sizes around the launch's mean work
// per pair the one whose busiest pair is done first is taken, by a model in SM
// cycles: a stage and a tile as measured, the partial results written and read
// at 2.6 KB a cycle, and a second launch for their sum.
constexpr int min_stages(bool planes) { return planes ? 2 : 4; }
constexpr int kStage256 = 515, kStage128 = 390, kStagePlanes = 1600, kTileCycles = 1500, kSumCycles = 6000;

int split_of(int kb, int part, bool planes) {
  const int s = std::max(1, std::min(kb / min_stages(planes), (kb + part / 2) / part));
  const int per = (kb + s - 1) / s;
  return (kb + per - 1) / per;
}

void plan(PairArgs &a, bool planes) {
  const int slots = num_sms() / 2;
  int64_t tiles = 0, work = 0;
  int longest = 1;
  for (int i = 0; i < a.n; ++i) {
    PairProb &b = a.p[i];
    b.bn = b.N > 128 && !planes ? 256 : 128;
    b.mt = tiles_of(b.M, 256);
    tiles += (int64_t)b.mt * tiles_of(b.N, b.bn);
  }
  for (int i = 0; i < a.n; ++i) {
    PairProb &b = a.p[i];
    if (tiles * 2 <= slots) b.bn = 128;
    b.nt = tiles_of(b.N, b.bn);
    work += (int64_t)b.mt * b.nt * (b.kb[0] + b.kb[1]);
    longest = std::max(longest, b.kb[0] + b.kb[1]);
  }
  const int mean = (int)std::max<int64_t>(1, (work + slots - 1) / slots);
  int best = longest;
  if (longest >= 2 * min_stages(planes)) {
    double least = 0;
    for (int part : {longest, 2 * mean, mean, (mean + 1) / 2, (mean + 2) / 3}) {
      if (part > longest || part < 1) continue;
      // the busiest pair is among those that get a product's first tile
      int64_t at = 0, starts[kMaxProbs];
      for (int i = 0; i < a.n; ++i) {
        const PairProb &b = a.p[i];
        starts[i] = at % slots;
        at += (int64_t)b.mt * b.nt * split_of(b.kb[0] + b.kb[1], part, planes);
      }
      at = 0;
      double load[kMaxProbs] = {0}, sum = 0;
      for (int i = 0; i < a.n; ++i) {
        const PairProb &b = a.p[i];
        const int kb = b.kb[0] + b.kb[1], s = split_of(kb, part, planes);
        const int64_t t = (int64_t)b.mt * b.nt * s;
        const double cost = (double)((kb + s - 1) / s) * (planes ? kStagePlanes : (b.bn == 256 ? kStage256 : kStage128)) +
                            kTileCycles;
        for (int k = 0; k < a.n; ++k) {
          const int64_t c = slots - 1 - starts[k];
          load[k] += cost * (double)((at + t + c) / slots - (at + c) / slots);
        }
        at += t;
        if (s > 1) sum += 8.0 * s * b.M * b.N / 2600;
      }
      double busiest = 0;
      for (int k = 0; k < a.n; ++k) busiest = std::max(busiest, load[k]);
      const double cycles = busiest + (sum > 0 ? sum + kSumCycles : 0);
      if (least == 0 || cycles < least) least = cycles, best = part;
    }
  }
  a.tile0[0] = 0;
  for (int i = 0; i < a.n; ++i) {
    PairProb &b = a.p[i];
    const int kb = b.kb[0] + b.kb[1];
    b.splits = split_of(kb, best, planes);
    b.kper = (kb + b.splits - 1) / b.splits;
    a.tile0[i + 1] = a.tile0[i] + b.mt * b.nt * b.splits;
  }
}

}  // namespace

namespace fbh {

int products(Call &c, const Product *all, int n_all) {
  const Product *ps[kMaxProbs];
  PairArgs a;
  std::memset(&a, 0, sizeof(a));
  // longest reductions first: tiles go to the SM pairs in turn
  for (int i = 0; i < n_all; ++i) {
    const Product &p = all[i];
    if (p.M == 0 || !p.out.p) continue;
    int at = a.n++;
    auto len = [](const Product &q) { return q.columns ? q.rows : (int64_t)q.term[0].K + (q.terms > 1 ? q.term[1].K : 0); };
    for (; at > 0 && len(*ps[at - 1]) < len(p); --at) ps[at] = ps[at - 1];
    ps[at] = &p;
  }
  if (a.n == 0) return FB_OK;
  const bool planes = ps[0]->A.plane > 0;
  for (int i = 0; i < a.n; ++i) {
    const Product &p = *ps[i];
    PairProb &b = a.p[i];
    b.M = (int)p.M;
    b.N = p.N;
    b.a_mn = p.columns;
    b.b_mn = p.b_mn;
    for (int t = 0; t < p.terms; ++t) {
      b.kb[t] = tiles_of(p.columns ? p.rows : p.term[t].K, BK);
      b.ax[t] = p.term[t].ax;
    }
  }
  plan(a, planes);
  const size_t mark = c.off;
  SumArgs sums;
  sums.n = 0;
  unsigned ctas = 0;
  for (int i = 0; i < a.n; ++i) {
    const Product &p = *ps[i];
    PairProb &b = a.p[i];
    const int64_t prow = (int64_t)b.mt * 256, pld = round_up(p.N, 4);
    b.split_rows = (int)prow;
    b.f32 = b.splits > 1 || p.fold || p.out.type == FB_F32;
    if (b.splits > 1 || p.fold) {
      const int64_t rows = p.fold ? p.M / 2 : p.M;
      float *P = static_cast<float *>(c.take((size_t)(b.splits * prow * pld) * 4));
      if (!P) return fb::set_error(FB_ERR_ARG, "workspace too small");
      sums.j[sums.n++] = SumJob{P, p.out.p, p.out.ld, pld, prow * pld, rows, p.fold ? rows * pld : 0, b.splits, p.N,
                                p.out.accumulate, p.out.type == FB_BF16, ctas};
      ctas += (unsigned)((rows * p.N + kSumPerCta - 1) / kSumPerCta);
      b.has_tc = 1;
      if (!c.dry) FBH_TRY(make_map(&b.tc, P, b.splits * prow, p.N, pld, 32, true));
    } else if (!c.dry) {
      b.C = p.out.p;
      b.ldc = p.out.ld;
      b.accumulate = p.out.accumulate;
      b.has_tc = map_ok(p.out.p, p.out.ld, b.f32 ? 4 : 2);
      if (b.has_tc) FBH_TRY(make_map(&b.tc, p.out.p, p.M, p.N, p.out.ld, 32, b.f32));
    }
    if (c.dry) continue;
    for (int t = 0; t < p.terms; ++t) {
      const Term &tm = p.term[t];
      if (p.columns) {
        FBH_TRY(operand_map(&b.ta[t], p.A, p.rows, p.acols, BK));
        FBH_TRY(operand_map(&b.tb[t], tm.B, p.rows, p.N, BK));
      } else {
        FBH_TRY(operand_map(&b.ta[t], p.A, p.M, p.acols, kHalfM));
        FBH_TRY(p.b_mn ? operand_map(&b.tb[t], tm.B, tm.K, p.b_n, BK) : operand_map(&b.tb[t], tm.B, p.b_n, tm.K, b.bn / 2));
      }
    }
  }
  c.off = mark;
  if (c.dry) return FB_OK;
  a.err = err_word();
  FBH_TRY((planes ? launch_pair<kStore, 3>(a, c.stream) : launch_pair<kStore, 1>(a, c.stream)));
  if (sums.n == 0) return FB_OK;
  FB_TRY_CUDA(fb::launch(k_sum_splits, ctas, 256, 0, c.stream, sums));
  FB_LAUNCHED("k_sum_splits");
  return FB_OK;
}

}  // namespace fbh
