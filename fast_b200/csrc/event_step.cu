// Single events against per-node state tables, in place: the short causal
// convolution and the selective scan, one row of each event.
//
//   conv: window = [state[i] | x],  y = act(bias + sum_k w[k] window[k]),  state[i] = the window without its oldest
//   scan: dt = softplus(delta + bias),  h = exp(dt A) state[i] + dt u B,  y = (<C, h> + D u) silu(z),  state[i] = h
//
// Bound by the state's bytes, read once and written once.  Row r works on state
// index[r].  Events of one node take their turns in the rows' order, as a
// chronological batch means them: k_links finds each row's successor of the
// same node, the first row of a node walks the chain with the state in
// registers, the others do nothing.
#include <algorithm>
#include "head.cuh"
#include "history.cuh"

namespace {
using namespace fbq;

constexpr int64_t kSms = 148;
constexpr int kMaxTaps = 8, kMaxStates = 64;
constexpr int kFollows = -2;               // link of a row that another row of its node comes before
constexpr int kLast = -1;                  // end of a chain

struct Rows {
  const int64_t *index;                    // null: row r is state r
  int64_t states;
  int rows;
  const int2 *link;                        // x: the next row of the node, or kLast; y: kFollows where it is not the first
  // The state of a row, -1: none.
  __device__ __forceinline__ int64_t at(int r) const {
    if (!index) return r;
    const int64_t i = index[r];
    return i >= 0 && i < states ? i : -1;
  }
};

// One warp a row: all other rows of the same node, 32 a step.
__global__ void __launch_bounds__(256) k_links(const int64_t *index, int rows, int2 *link) {
  fb::pdl_enter();
  const int r = (int)((blockIdx.x * 256 + threadIdx.x) >> 5), lane = threadIdx.x & 31;
  if (r >= rows) return;
  const int64_t me = index[r];
  int next = INT32_MAX;
  bool before = false;
#pragma unroll 4
  for (int j = lane; j < rows; j += 32) {
    const bool same = index[j] == me;
    before |= same && j < r;
    if (same && j > r) next = min(next, j);
  }
  next = __reduce_min_sync(0xffffffffu, next);
  before = __any_sync(0xffffffffu, before);
  if (lane == 0) link[r] = make_int2(next == INT32_MAX ? kLast : next, before ? kFollows : 0);
}

// ---- convolution -----------------------------------------------------------------------------------
struct ConvStep {
  int D, K, silu;
  const void *x; int64_t ldx;
  void *y; int64_t ldy;
  void *state;                             // [states, K - 1, D]
  const float *w, *bias;
  Rows r;
};

template <typename T, int V, int KT> __global__ void __launch_bounds__(256) k_conv_step(ConvStep a) {
  fb::pdl_enter();
  const int groups = a.D / V;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (int64_t)groups * a.r.rows) return;
  int r = (int)(i / groups);
  const int col = (int)(i % groups) * V;
  const int64_t at = a.r.at(r);
  const int skip = KT - a.K;
  if (at < 0) {                            // held out: nothing is touched
    Vec<T, V> y;
#pragma unroll
    for (int v = 0; v < V; ++v) y.e[v] = from_f<T>(a.r.index[r] < 0 ? 0.f : __int_as_float(0x7fffffff));
    *reinterpret_cast<Vec<T, V> *>(static_cast<T *>(a.y) + r * a.ldy + col) = y;
    return;
  }
  if (a.r.link && a.r.link[r].y == kFollows) return;
  T *const state = static_cast<T *>(a.state) + at * (a.K - 1) * a.D + col;
  Vec<T, V> win[KT];
#pragma unroll
  for (int k = 0; k < KT - 1; ++k)
    if (k >= skip) win[k] = *reinterpret_cast<const Vec<T, V> *>(state + (int64_t)(k - skip) * a.D);
  float w[KT][V], bias[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    bias[v] = a.bias ? a.bias[col + v] : 0.f;
#pragma unroll
    for (int k = 0; k < KT; ++k) w[k][v] = k >= skip ? a.w[(int64_t)(col + v) * a.K + k - skip] : 0.f;
  }
  for (;;) {
    win[KT - 1] = *reinterpret_cast<const Vec<T, V> *>(static_cast<const T *>(a.x) + r * a.ldx + col);
    Vec<T, V> y;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float p = bias[v];
#pragma unroll
      for (int k = 0; k < KT; ++k)
        if (k >= skip) p = fmaf(w[k][v], to_f(win[k].e[v]), p);
      y.e[v] = from_f<T>(a.silu ? p * sigmoid(p) : p);
    }
    *reinterpret_cast<Vec<T, V> *>(static_cast<T *>(a.y) + r * a.ldy + col) = y;
#pragma unroll
    for (int k = 0; k < KT - 1; ++k) win[k] = win[k + 1];
    const int next = a.r.link ? a.r.link[r].x : kLast;
    if (next < 0) break;
    r = next;
  }
#pragma unroll
  for (int k = 0; k < KT - 1; ++k)
    if (k >= skip) *reinterpret_cast<Vec<T, V> *>(state + (int64_t)(k - skip) * a.D) = win[k];
}

// ---- scan ------------------------------------------------------------------------------------------
struct ScanStep {
  int D, N, per, softplus, vec;
  const void *u, *delta, *B, *C, *z;
  int64_t ldu, ldd, ldb, gsb, ldc, gsc, ldz, ldy;
  void *y;
  const float *A, *Ds, *bias;
  float *state;                            // [states, D, N]
  Rows r;
  int across;                              // warps along the channels
};

// A warp holds 32 / NL channels, NL = NP / 4 lanes a channel with 4 states each,
// and takes every (warps / across)-th row, so A stays in registers.
template <typename T, int NP> __global__ void __launch_bounds__(256) k_scan_step(ScanStep a) {
  fb::pdl_enter();
  constexpr int NL = NP / 4, CL = 32 / NL;
  const int lane = threadIdx.x & 31, nl = lane % NL, n0 = nl * 4;
  const int64_t wid = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 5, warps = (int64_t)gridDim.x * 8;
  const int d = (int)(wid % a.across) * CL + lane / NL;
  const bool has = d < a.D;
  const int grp = has ? d / a.per : 0;
  const auto load = [&](const float *p, float (&v)[4]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = 0.f;
    if (!has || n0 >= a.N) return;
    if (a.vec) {
      const float4 f = *reinterpret_cast<const float4 *>(p + n0);
      v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (n0 + k < a.N) v[k] = p[n0 + k];
    }
  };
  float A2[4];
  load(a.A + (int64_t)(has ? d : 0) * a.N, A2);
#pragma unroll
  for (int k = 0; k < 4; ++k) A2[k] *= kLog2e;
  const float bias = has && a.bias ? a.bias[d] : 0.f, skip = has && a.Ds ? a.Ds[d] : 0.f;
  const int64_t step = warps / a.across;
  if (wid / a.across >= step) return;
  for (int64_t head = wid / a.across; head < a.r.rows; head += step) {
    int r = (int)head;
    const int64_t at = a.r.at(r);
    if (at < 0) {
      if (has && nl == 0)
        static_cast<T *>(a.y)[r * a.ldy + d] = from_f<T>(a.r.index[r] < 0 ? 0.f : __int_as_float(0x7fffffff));
      continue;
    }
    if (a.r.link && a.r.link[r].y == kFollows) continue;
    float *const state = a.state + (at * a.D + (has ? d : 0)) * a.N;
    float h[4];
    load(state, h);
    for (;;) {
      const float u = has ? to_f(static_cast<const T *>(a.u)[r * a.ldu + d]) : 0.f;
      float dt = has ? to_f(static_cast<const T *>(a.delta)[r * a.ldd + d]) + bias : 0.f;
      if (a.softplus) dt = softplus(dt);
      const T *b = static_cast<const T *>(a.B) + r * a.ldb + grp * a.gsb, *c = static_cast<const T *>(a.C) + r * a.ldc + grp * a.gsc;
      float v = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const bool in = n0 + k < a.N;
        const float Bn = in ? to_f(b[n0 + k]) : 0.f, Cn = in ? to_f(c[n0 + k]) : 0.f;
        h[k] = fmaf(ex2(dt * A2[k]), h[k], dt * u * Bn);
        v = fmaf(Cn, h[k], v);
      }
#pragma unroll
      for (int o = NL / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      if (has && nl == 0) {
        v = fmaf(skip, u, v);
        if (a.z) {
          const float z = to_f(static_cast<const T *>(a.z)[r * a.ldz + d]);
          v *= z * sigmoid(z);
        }
        static_cast<T *>(a.y)[r * a.ldy + d] = from_f<T>(v);
      }
      const int next = a.r.link ? a.r.link[r].x : kLast;
      if (next < 0) break;
      r = next;
    }
    if (has && n0 < a.N) {
      if (a.vec) {
        *reinterpret_cast<float4 *>(state + n0) = make_float4(h[0], h[1], h[2], h[3]);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (n0 + k < a.N) state[n0 + k] = h[k];
      }
    }
  }
}

// ---- host ------------------------------------------------------------------------------------------
int rows_of(const char *who, int64_t n, int64_t states, const int64_t *index, void *ws, size_t ws_bytes, cudaStream_t st, Rows &r) {
  if (!index && n > states) return fb::set_error(FB_ERR_ARG, std::string(who) + ": more rows than states");
  r = Rows{index, states, (int)n, nullptr};
  if (!index || n < 2) return FB_OK;
  FBH_TRY(fbh::check_ws(ws, who));
  if (ws_bytes < (size_t)n * sizeof(int2)) return fb::set_error(FB_ERR_ARG, std::string(who) + ": workspace too small");
  FB_TRY_CUDA(fb::launch(k_links, dim3((unsigned)((n + 7) / 8)), 256, 0, st, index, (int)n, static_cast<int2 *>(ws)));
  r.link = static_cast<const int2 *>(ws);
  return FB_OK;
}

template <typename T, int V> int conv_step(const ConvStep &a, cudaStream_t st) {
  const int64_t threads = (int64_t)(a.D / V) * a.r.rows;
  const dim3 grid((unsigned)((threads + 255) / 256));
  if (a.K <= 4) FB_TRY_CUDA(fb::launch(k_conv_step<T, V, 4>, grid, 256, 0, st, a));
  else FB_TRY_CUDA(fb::launch(k_conv_step<T, V, 8>, grid, 256, 0, st, a));
  return FB_OK;
}

template <typename T> int scan_step(ScanStep &a, cudaStream_t st) {
  const int np = a.N <= 8 ? 8 : (a.N <= 16 ? 16 : (a.N <= 32 ? 32 : 64)), cl = 32 / (np / 4);
  a.across = (a.D + cl - 1) / cl;
  // one resident wave of warps (8 CTAs of 8 an SM), each with as many rows as it takes; at least a warp for each channel
  const int64_t wave = kSms * 64, need = (int64_t)a.across * a.r.rows;
  int64_t warps = std::max<int64_t>(std::min(need, wave) / a.across * a.across, a.across);
  const dim3 grid((unsigned)((warps + 7) / 8));
  switch (np) {
    case 8: FB_TRY_CUDA(fb::launch(k_scan_step<T, 8>, grid, 256, 0, st, a)); break;
    case 16: FB_TRY_CUDA(fb::launch(k_scan_step<T, 16>, grid, 256, 0, st, a)); break;
    case 32: FB_TRY_CUDA(fb::launch(k_scan_step<T, 32>, grid, 256, 0, st, a)); break;
    default: FB_TRY_CUDA(fb::launch(k_scan_step<T, 64>, grid, 256, 0, st, a));
  }
  return FB_OK;
}

}  // namespace

extern "C" size_t fb_event_step_ws_bytes(int64_t n) { return n > 1 ? (size_t)n * sizeof(int2) : 0; }

extern "C" int fb_short_conv_step(int type, int act, const void *x, int64_t ldx, const float *w, const float *bias, void *state,
                                  int64_t states, const int64_t *index, void *y, int64_t ldy, int64_t n, int D, int K,
                                  void *ws, size_t ws_bytes, cudaStream_t stream) {
  const auto bad = [&](const char *what) { return fb::set_error(FB_ERR_ARG, std::string("short_conv_step: ") + what); };
  if (type != FB_F32 && type != FB_BF16) return bad("unknown element type");
  if (act != FB_ACT_NONE && act != FB_ACT_SILU) return bad("unknown activation");
  if (n < 0 || states < 0 || D < 1 || K < 1) return bad("bad sizes");
  if (K > kMaxTaps) return fb::set_error(FB_ERR_UNSUPPORTED, "short_conv_step: at most 8 taps");
  if (n > (1 << 24) || D > (1 << 20)) return fb::set_error(FB_ERR_UNSUPPORTED, "short_conv_step: too many rows or columns");
  if (!w || (n && (!x || !y || (K > 1 && !state)))) return bad("missing operand");
  if (n > 1 && (ldx < D || ldy < D)) return bad("leading dimension below the width");
  if (!n) return FB_OK;
  ConvStep a{D, K, act == FB_ACT_SILU, x, ldx, y, ldy, state, w, bias, {}};
  const int es = type == FB_F32 ? 4 : 2;
  const uint64_t at = (uint64_t)(uintptr_t)x | (uint64_t)(uintptr_t)y | (K > 1 ? (uint64_t)(uintptr_t)state : 0);
  if (at % es) return bad("rows that are not aligned to their elements");
  FBH_TRY(rows_of("short_conv_step", n, states, index, ws, ws_bytes, stream, a.r));
  uint64_t bits = at / es | (uint64_t)D;
  if (n > 1) bits |= (uint64_t)ldx | (uint64_t)ldy;
  const int V = bits % 4 == 0 ? 4 : (bits % 2 == 0 ? 2 : 1);
  if (type == FB_F32) return V == 4 ? conv_step<float, 4>(a, stream) : V == 2 ? conv_step<float, 2>(a, stream) : conv_step<float, 1>(a, stream);
  return V == 4 ? conv_step<bf16, 4>(a, stream) : V == 2 ? conv_step<bf16, 2>(a, stream) : conv_step<bf16, 1>(a, stream);
}

extern "C" int fb_selective_scan_step(const fb_selective_scan_event *s, void *ws, size_t ws_bytes, cudaStream_t stream) {
  const auto bad = [&](const char *what) { return fb::set_error(FB_ERR_ARG, std::string("selective_scan_step: ") + what); };
  if (!s) return bad("no arguments");
  if (s->type != FB_F32 && s->type != FB_BF16) return bad("unknown element type");
  if (s->n < 0 || s->states < 0 || s->D < 1 || s->N < 1 || s->G < 1 || s->D % s->G) return bad("bad sizes");
  if (s->N > kMaxStates) return fb::set_error(FB_ERR_UNSUPPORTED, "selective_scan_step: at most 64 states");
  if (s->n > (1 << 24) || s->D > (1 << 20)) return fb::set_error(FB_ERR_UNSUPPORTED, "selective_scan_step: too many rows or columns");
  if (!s->A || (s->n && (!s->u || !s->delta || !s->B || !s->C || !s->state || !s->y))) return bad("missing operand");
  if (s->n > 1 && (s->ldu < s->D || s->ld_delta < s->D || s->ldy < s->D || (s->z && s->ldz < s->D)))
    return bad("leading dimension below the width");
  if (!s->n) return FB_OK;
  ScanStep a{};
  a.D = s->D, a.N = s->N, a.per = s->D / s->G, a.softplus = s->softplus;
  a.vec = s->N % 4 == 0 && ((uintptr_t)s->state | (uintptr_t)s->A) % 16 == 0;
  a.u = s->u, a.ldu = s->ldu, a.delta = s->delta, a.ldd = s->ld_delta, a.B = s->B, a.ldb = s->ldb, a.gsb = s->ldb_group;
  a.C = s->C, a.ldc = s->ldc, a.gsc = s->ldc_group, a.z = s->z, a.ldz = s->ldz, a.y = s->y, a.ldy = s->ldy;
  a.A = s->A, a.Ds = s->skip, a.bias = s->delta_bias, a.state = s->state;
  FBH_TRY(rows_of("selective_scan_step", s->n, s->states, s->index, ws, ws_bytes, stream, a.r));
  return s->type == FB_F32 ? scan_step<float>(a, stream) : scan_step<bf16>(a, stream);
}
