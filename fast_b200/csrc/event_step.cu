// Single events against per-node state tables, in place: the short causal
// convolution and the selective scan, one row of each event.
//
//   conv: window = [state[i] | x],  y = act(bias + sum_k w[k] window[k]),  state[i] = the window without its oldest
//   scan: dt = softplus(delta + bias),  h = exp(dt A) state[i] + dt u B,  y = (<C, h> + D u) silu(z),  state[i] = h
//
// with the operations of the packed histories (history.cuh), so that events decay as
// histories do.
//
// Bound by the state's bytes, read once and written once.  Row r works on state
// index[r].  Events of one node take their turns in the rows' order, as a
// chronological batch means them: the first row of a node walks its rows with the
// state in registers, the others do nothing.  Which row is first and which comes
// next is looked up by comparing indices: by the warps themselves in calls of few
// rows, in calls of many by k_links before (a lane a row, the other indices from
// shared memory, four a branch: 4.5 us for 4,000 rows, 7.4 with one a branch; it
// grows with the square of the rows, about 35 us for 16,384 and 425 for 65,536).
// Warps stay on their columns and take rows one after the other, so that weights
// stay in registers; the convolution loads two nodes' windows at once.  (States
// copied two nodes ahead by asynchronous copies, or two or four nodes' loaded at
// once, were no faster: 4,000 events of width 200, 46 to 55 us against 45 with
// the indices' comparison of then, 40 with today's; the states are 102 MB from and
// to memory.)
#include <algorithm>
#include "head.cuh"
#include "history.cuh"

namespace {
using namespace fbq;

constexpr int64_t kSms = 148;
constexpr int kMaxTaps = 8, kMaxStates = 64;
constexpr int kAlone = 64;                 // rows up to which the warps compare indices themselves
constexpr int kMaxRows = 1 << 24;
constexpr int kMaxIndexed = 1 << 16;       // comparing grows with the square of the rows
constexpr int kLast = -1;                  // end of a node's rows

struct Rows {
  const int64_t *index;                    // null: row r is state r
  int64_t states;
  int rows;
  const int2 *link;                        // x: the next row of the node, or kLast; y: 1 where another row comes before
  // The state of a row, -1: none.
  __device__ __forceinline__ int at(int r) const {
    if (!index) return r;
    const int64_t i = index[r];
    return i >= 0 && i < states ? (int)i : -1;
  }
  // What a row that has no state receives.
  __device__ __forceinline__ float held(int r) const { return index[r] < 0 ? 0.f : __int_as_float(0x7fffffff); }
  // Whether a row of the same node comes before r; each lane for a row of its own.
  __device__ __forceinline__ bool follows(int r) const {
    if (!index || rows == 1 || r >= rows) return false;
    if (link) return link[r].y != 0;
    const int64_t me = index[r];
    bool yes = false;
    for (int j = 0; j < rows; ++j) yes |= j < r && index[j] == me;
    return yes;
  }
  // The next row of the node, kLast: none.
  __device__ __forceinline__ int next(int r) const {
    if (!index || rows == 1) return kLast;
    if (link) return link[r].x;
    const int64_t me = index[r];
    for (int j = r + 1; j < rows; ++j)
      if (index[j] == me) return j;
    return kLast;
  }
};

// A lane a row, the 32 warps of a CTA a 32nd of the other rows each.
constexpr int kPart = 4096;
__global__ void __launch_bounds__(1024) k_links(const int64_t *index, int rows, int64_t states, int2 *link) {
  fb::pdl_enter();
  __shared__ __align__(16) int some[kPart];
  __shared__ int2 found[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = blockIdx.x * 32 + lane;
  const auto id = [&](int j) {             // rows without a state are of no node
    const int64_t i = j < rows ? index[j] : -1;
    return i >= 0 && i < states ? (int)i : -1;
  };
  const int mine = r < rows ? id(r) : -1, me = mine < 0 ? -2 : mine;       // -2: meets nothing
  int next = INT32_MAX, before = 0;
  for (int base = 0; base < rows; base += kPart) {
    if (base) __syncthreads();
#pragma unroll
    for (int i = 0; i < kPart / 1024; ++i) some[i * 1024 + threadIdx.x] = id(base + i * 1024 + threadIdx.x);
    __syncthreads();
    const int from = warp * (kPart / 32), end = min(from + kPart / 32, rows - base);
#pragma unroll 4
    for (int i = from; i < end; i += 4) {
      const int4 v = *reinterpret_cast<const int4 *>(&some[i]);
      if (v.x == me || v.y == me || v.z == me || v.w == me) {     // seldom
        const int o[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int j = base + i + k;
          if (o[k] == me && j < r) before = 1;
          if (o[k] == me && j > r) next = min(next, j);
        }
      }
    }
  }
  found[lane][warp] = make_int2(next, before);
  __syncthreads();
  const int2 f = found[warp][lane];        // warp w: row w of the 32
  next = __reduce_min_sync(0xffffffffu, f.x), before = __reduce_or_sync(0xffffffffu, (unsigned)f.y);
  const int out = blockIdx.x * 32 + warp;
  if (lane == 0 && out < rows) link[out] = make_int2(next == INT32_MAX ? kLast : next, before);
}

// The V K taps of V columns, in one go where they are aligned.
template <int V, int KT> __device__ __forceinline__ void taps(const float *w, int K, bool wide, float (&out)[KT][V]) {
  constexpr int N = V * KT, A = N % 4 == 0 ? 4 : (N % 2 == 0 ? 2 : 1);
  if (KT < 8 && wide) {
    alignas(16) float flat[N];
#pragma unroll
    for (int i = 0; i < N; i += A) *reinterpret_cast<Vec<float, A> *>(&flat[i]) = *reinterpret_cast<const Vec<float, A> *>(w + i);
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int k = 0; k < KT; ++k) out[k][v] = flat[v * KT + k];
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int k = 0; k < KT; ++k) out[k][v] = k >= KT - K ? w[v * K + k - (KT - K)] : 0.f;
  }
}

// ---- convolution -----------------------------------------------------------------------------------
struct ConvStep {
  int D, K, silu;
  const void *x; int64_t ldx;
  void *y; int64_t ldy;
  void *state;                             // [states, K - 1, D]
  const float *w, *bias;
  Rows r;
  int across, each;                        // warps along the columns; rows of a warp, at most 32
  bool wide;                               // w is 16-byte aligned
};

// KT taps in registers; KT 2, 3, 4: exactly K, KT 8: the first 8 - K of them do not exist.
template <typename T, int V, int KT> __global__ void __launch_bounds__(256) k_conv_step(ConvStep a) {
  fb::pdl_enter();
  using E = Vec<T, V>;
  const int lane = threadIdx.x & 31, skip = KT < 8 ? 0 : KT - a.K;
  const int wid = (int)(((int64_t)blockIdx.x * 256 + threadIdx.x) >> 5);
  const int col = (wid % a.across * 32 + lane) * V, base = wid / a.across * a.each;
  if (base >= a.r.rows) return;
  const bool has = col < a.D;
  const int count = min(a.each, a.r.rows - base);
  // what the lanes know of the warp's rows
  const int at_ = lane < count ? a.r.at(base + lane) : -1;
  const bool follows = lane < count && a.r.follows(base + lane);
  float w[KT][V], bias[V];
  taps<V, KT>(a.w + (int64_t)(has ? col : 0) * a.K, a.K, a.wide, w);
#pragma unroll
  for (int v = 0; v < V; ++v) bias[v] = has && a.bias ? a.bias[col + v] : 0.f;
  const auto state_of = [&](int at) { return static_cast<T *>(a.state) + (int64_t)at * (a.K - 1) * a.D + col; };
  const auto input = [&](int r) { return *reinterpret_cast<const E *>(static_cast<const T *>(a.x) + r * a.ldx + col); };
  const auto put = [&](int r, const E &y) { *reinterpret_cast<E *>(static_cast<T *>(a.y) + r * a.ldy + col) = y; };
  const auto window = [&](int at, E (&win)[KT]) {
#pragma unroll
    for (int k = 0; k < KT - 1; ++k)
      if (k >= skip) win[k] = *reinterpret_cast<const E *>(state_of(at) + (int64_t)(k - skip) * a.D);
  };
  unsigned held = __ballot_sync(0xffffffffu, lane < count && at_ < 0);
  unsigned heads = __ballot_sync(0xffffffffu, lane < count && at_ >= 0 && !follows);
  for (; held; held &= held - 1) {
    const int r = base + __ffs(held) - 1;
    E y;
#pragma unroll
    for (int v = 0; v < V; ++v) y.e[v] = from_f<T>(a.r.held(r));
    if (has) put(r, y);
  }
  if (!heads) return;
  // kBatch nodes' windows are loaded together, then worked on one by one
  constexpr int kBatch = 2;
  while (heads) {
    E win[kBatch][KT];
    int row[kBatch], at[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      row[i] = heads ? base + __ffs(heads) - 1 : -1;
      at[i] = __shfl_sync(0xffffffffu, at_, max(row[i] - base, 0));
      heads &= heads - 1;
      if (row[i] >= 0 && has) window(at[i], win[i]), win[i][KT - 1] = input(row[i]);
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      int r = row[i];
      if (r < 0) break;
      int next = a.r.next(r);
      for (;;) {
        E y;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          float p = bias[v];
#pragma unroll
          for (int k = 0; k < KT; ++k)
            if (k >= skip) p = fmaf(w[k][v], to_f(win[i][k].e[v]), p);
          y.e[v] = from_f<T>(a.silu ? p * sigmoid<T>(p) : p);
        }
        if (has) put(r, y);
#pragma unroll
        for (int k = 0; k < KT - 1; ++k) win[i][k] = win[i][k + 1];
        if (next < 0) break;
        r = next;
        if (has) win[i][KT - 1] = input(r);
        next = a.r.next(r);
      }
      if (has)
#pragma unroll
        for (int k = 0; k < KT - 1; ++k)
          if (k >= skip) *reinterpret_cast<E *>(state_of(at[i]) + (int64_t)(k - skip) * a.D) = win[i][k];
    }
  }
}

// ---- scan ------------------------------------------------------------------------------------------
struct ScanStep {
  int D, N, per, tiles, softplus, vec, vec_bc;   // per: channels of a group; tiles: warps across a group
  const void *u, *delta, *B, *C, *z;
  int64_t ldu, ldd, ldb, gsb, ldc, gsc, ldz, ldy;
  void *y;
  const float *A, *Ds, *bias;
  float *state;                            // [states, D, N]
  Rows r;
  int across, each;                        // warps along the channels; rows of a warp, at most 32
};

// Sums V values over V lanes, each lane keeping the sum of its own number.
template <int V> __device__ __forceinline__ float spread_sum(float *v) {
  if constexpr (V == 1) {
    return v[0];
  } else {
    constexpr int H = V / 2;
    const bool up = (threadIdx.x & H) != 0;
#pragma unroll
    for (int k = 0; k < H; ++k) {
      const float send = up ? v[k] : v[k + H], stay = up ? v[k + H] : v[k];
      v[k] = stay + __shfl_xor_sync(0xffffffffu, send, H);
    }
    return spread_sum<H>(v);
  }
}

// A warp holds 32 channels.  NL = NP / 4 lanes side by side share NL of them and
// hold 4 of their states each; what a channel has once (dt, the gate, y) is one
// lane's, so it is loaded and computed once, 32 channels in a row.
template <typename T, int NP> __global__ void __launch_bounds__(256, NP <= 16 ? 3 : 1) k_scan_step(ScanStep a) {
  fb::pdl_enter();
  constexpr int NL = NP / 4, P = NL / 2;
  const int lane = threadIdx.x & 31, nl = lane % NL, n0 = nl * 4;
  const int wid = (int)(((int64_t)blockIdx.x * 256 + threadIdx.x) >> 5);
  const int tile = wid % a.across, grp = tile / a.tiles, in = tile % a.tiles * 32;
  const int base = wid / a.across * a.each;
  if (base >= a.r.rows) return;
  const bool own = in + lane < a.per;
  const int d = grp * a.per + in + lane;                         // the lane's own channel
  const int shared = grp * a.per + in + lane - nl;               // the first of those it shares
  const int has = n0 < a.N ? a.per - (in + lane - nl) : 0;       // how many of them exist (for its states)
  const int count = min(a.each, a.r.rows - base);
  const int at_ = lane < count ? a.r.at(base + lane) : -1;
  const bool follows = lane < count && a.r.follows(base + lane);
  const auto load = [&](const float *p, F2 (&v)[P][4]) {
#pragma unroll
    for (int q = 0; q < P; ++q) {
      float x[2][4] = {};
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (2 * q + j < has) {
          const float *s = p + (2 * q + j) * a.N + n0;
          if (a.vec) {
            const float4 f = *reinterpret_cast<const float4 *>(s);
            x[j][0] = f.x, x[j][1] = f.y, x[j][2] = f.z, x[j][3] = f.w;
          } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (n0 + k < a.N) x[j][k] = s[k];
          }
        }
#pragma unroll
      for (int k = 0; k < 4; ++k) v[q][k] = pack(x[0][k], x[1][k]);
    }
  };
  F2 A2[P][4];
  load(a.A + (int64_t)shared * a.N, A2);
#pragma unroll
  for (int q = 0; q < P; ++q)
#pragma unroll
    for (int k = 0; k < 4; ++k) A2[q][k] = pack(scaled(unpack(A2[q][k]).x), scaled(unpack(A2[q][k]).y));
  const float bias = own && a.bias ? a.bias[d] : 0.f, skip = own && a.Ds ? a.Ds[d] : 0.f;

  struct Event {
    T u, delta, z;
    Vec<T, 4> b, c;
  };
  const T none = from_f<T>(0.f);
  const auto four = [&](const void *p, int64_t at, Vec<T, 4> &v) {
    const T *q = static_cast<const T *>(p) + at + n0;
#pragma unroll
    for (int k = 0; k < 4; ++k) v.e[k] = none;
    if (a.vec_bc) {
      if (n0 < a.N) v = *reinterpret_cast<const Vec<T, 4> *>(q);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (n0 + k < a.N) v.e[k] = q[k];
    }
  };
  const auto event = [&](int r, Event &e) {
    e.u = own ? static_cast<const T *>(a.u)[r * a.ldu + d] : none;
    e.delta = own ? static_cast<const T *>(a.delta)[r * a.ldd + d] : none;
    e.z = own && a.z ? static_cast<const T *>(a.z)[r * a.ldz + d] : none;
    four(a.B, r * a.ldb + grp * a.gsb, e.b), four(a.C, r * a.ldc + grp * a.gsc, e.c);
  };
  unsigned held = __ballot_sync(0xffffffffu, lane < count && at_ < 0);
  unsigned heads = __ballot_sync(0xffffffffu, lane < count && at_ >= 0 && !follows);
  for (; held; held &= held - 1) {
    const int r = base + __ffs(held) - 1;
    if (own) static_cast<T *>(a.y)[r * a.ldy + d] = from_f<T>(a.r.held(r));
  }
  for (; heads; heads &= heads - 1) {
    const int first = __ffs(heads) - 1;
    int r = base + first;
    float *const state = a.state + ((int64_t)__shfl_sync(0xffffffffu, at_, first) * a.D + shared) * a.N;
    Event e;
    F2 h[P][4];
    load(state, h);
    event(r, e);
    int next = a.r.next(r);
    for (;;) {
      const float u = to_f(e.u);
      float dt = to_f(e.delta) + bias;
      if (a.softplus) dt = softplus(dt);
      const float dtu = dt * u;
      F2 B[4], C[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) B[k] = both(to_f(e.b.e[k])), C[k] = both(to_f(e.c.e[k]));
      float y[NL];
#pragma unroll
      for (int q = 0; q < P; ++q) {
        const auto of = [&](float v) {
          return pack(__shfl_sync(0xffffffffu, v, lane - nl + 2 * q), __shfl_sync(0xffffffffu, v, lane - nl + 2 * q + 1));
        };
        const F2 dt2 = of(dt), dtu2 = of(dtu);
        F2 v;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          h[q][k] = fma2(decays(dt2, A2[q][k]), h[q][k], mul2(dtu2, B[k]));
          v = k == 0 ? mul2(C[k], h[q][k]) : fma2(C[k], h[q][k], v);
        }
        const float2 f = unpack(v);
        y[2 * q] = f.x, y[2 * q + 1] = f.y;
      }
      float v = fmaf(skip, u, spread_sum<NL>(y));
      if (a.z) {
        const float z = to_f(e.z);
        v *= z * sigmoid<T>(z);
      }
      if (own) static_cast<T *>(a.y)[r * a.ldy + d] = from_f<T>(v);
      if (next < 0) break;
      r = next;
      event(r, e);
      next = a.r.next(r);
    }
#pragma unroll
    for (int q = 0; q < P; ++q)
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (2 * q + j < has) {
          float x[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) x[k] = j ? unpack(h[q][k]).y : unpack(h[q][k]).x;
          float *const s = state + (2 * q + j) * a.N + n0;
          if (a.vec) {
            *reinterpret_cast<float4 *>(s) = make_float4(x[0], x[1], x[2], x[3]);
          } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (n0 + k < a.N) s[k] = x[k];
          }
        }
  }
}

// ---- host ------------------------------------------------------------------------------------------
int rows_of(const char *who, int64_t n, int64_t states, const int64_t *index, void *ws, size_t ws_bytes, cudaStream_t st, Rows &r) {
  if (!index && n > states) return fb::set_error(FB_ERR_ARG, std::string(who) + ": more rows than states");
  if (states > INT32_MAX) return fb::set_error(FB_ERR_UNSUPPORTED, std::string(who) + ": too many states");
  if (index && n > kMaxIndexed) return fb::set_error(FB_ERR_UNSUPPORTED, std::string(who) + ": at most 65,536 rows with an index");
  r = Rows{index, states, (int)n, nullptr};
  if (!index || n <= kAlone) return FB_OK;
  FBH_TRY(fbh::check_ws(ws, who));
  if (ws_bytes < (size_t)n * sizeof(int2)) return fb::set_error(FB_ERR_ARG, std::string(who) + ": workspace too small");
  FB_TRY_CUDA(fb::launch(k_links, dim3((unsigned)((n + 31) / 32)), 1024, 0, st, index, (int)n, states, static_cast<int2 *>(ws)));
  r.link = static_cast<const int2 *>(ws);
  return FB_OK;
}

// Rows of a warp: as few as make `resident` warps, at most 32.
int rows_each(int64_t rows, int64_t across, int64_t resident) {
  return (int)std::min<int64_t>(32, std::max<int64_t>(1, (rows * across + resident - 1) / resident));
}
dim3 warps_grid(int64_t rows, int each, int64_t across) { return dim3((unsigned)(((rows + each - 1) / each * across + 7) / 8)); }

template <typename T, int V> int conv_step(ConvStep &a, cudaStream_t st) {
  a.across = (a.D + 32 * V - 1) / (32 * V);
  a.wide = (uintptr_t)a.w % 16 == 0;
  a.each = rows_each(a.r.rows, a.across, kSms * 32);
  const dim3 grid = warps_grid(a.r.rows, a.each, a.across);
  switch (a.K) {
    case 2: FB_TRY_CUDA(fb::launch(k_conv_step<T, V, 2>, grid, 256, 0, st, a)); break;
    case 3: FB_TRY_CUDA(fb::launch(k_conv_step<T, V, 3>, grid, 256, 0, st, a)); break;
    case 4: FB_TRY_CUDA(fb::launch(k_conv_step<T, V, 4>, grid, 256, 0, st, a)); break;
    default: FB_TRY_CUDA(fb::launch(k_conv_step<T, V, 8>, grid, 256, 0, st, a));
  }
  return FB_OK;
}

template <typename T> int scan_step(ScanStep &a, cudaStream_t st) {
  const int np = a.N <= 8 ? 8 : (a.N <= 16 ? 16 : (a.N <= 32 ? 32 : 64)), ch = 32;
  a.tiles = (a.per + ch - 1) / ch, a.across = a.D / a.per * a.tiles;
  a.each = rows_each(a.r.rows, a.across, kSms * 96);
  const dim3 grid = warps_grid(a.r.rows, a.each, a.across);
  switch (np) {
    case 8: FB_TRY_CUDA(fb::launch(k_scan_step<T, 8>, grid, 256, 0, st, a)); break;
    case 16: FB_TRY_CUDA(fb::launch(k_scan_step<T, 16>, grid, 256, 0, st, a)); break;
    case 32: FB_TRY_CUDA(fb::launch(k_scan_step<T, 32>, grid, 256, 0, st, a)); break;
    default: FB_TRY_CUDA(fb::launch(k_scan_step<T, 64>, grid, 256, 0, st, a));
  }
  return FB_OK;
}

}  // namespace

extern "C" size_t fb_event_step_ws_bytes(int64_t n) { return n > kAlone ? (size_t)n * sizeof(int2) : 0; }

extern "C" int fb_short_conv_step(int type, int act, const void *x, int64_t ldx, const float *w, const float *bias, void *state,
                                  int64_t states, const int64_t *index, void *y, int64_t ldy, int64_t n, int D, int K,
                                  void *ws, size_t ws_bytes, cudaStream_t stream) {
  const auto bad = [&](const char *what) { return fb::set_error(FB_ERR_ARG, std::string("short_conv_step: ") + what); };
  if (type != FB_F32 && type != FB_BF16) return bad("unknown element type");
  if (act != FB_ACT_NONE && act != FB_ACT_SILU) return bad("unknown activation");
  if (n < 0 || states < 0 || D < 1 || K < 1) return bad("bad sizes");
  if (K > kMaxTaps) return fb::set_error(FB_ERR_UNSUPPORTED, "short_conv_step: at most 8 taps");
  if (n > kMaxRows || D > (1 << 20)) return fb::set_error(FB_ERR_UNSUPPORTED, "short_conv_step: too many rows or columns");
  if (!w || (n && (!x || !y || (K > 1 && states && !state)))) return bad("missing operand");
  if (n > 1 && (ldx < D || ldy < D)) return bad("leading dimension below the width");
  if (!n) return FB_OK;
  ConvStep a{D, K, act == FB_ACT_SILU, x, ldx, y, ldy, state, w, bias, {}};
  const int es = type == FB_F32 ? 4 : 2;
  const uint64_t at = (uint64_t)(uintptr_t)x | (uint64_t)(uintptr_t)y | (K > 1 ? (uint64_t)(uintptr_t)state : 0);
  if (at % es) return bad("rows that are not aligned to their elements");
  if (!aligned(4, w, bias) || !aligned(8, index)) return bad("parameters or indices that are not aligned to their elements");
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
  if (s->n > kMaxRows || s->D > (1 << 20)) return fb::set_error(FB_ERR_UNSUPPORTED, "selective_scan_step: too many rows or columns");
  if (!s->A || (s->n && (!s->u || !s->delta || !s->B || !s->C || (s->states && !s->state) || !s->y))) return bad("missing operand");
  if (s->n > 1 && (s->ldu < s->D || s->ld_delta < s->D || s->ldy < s->D || (s->z && s->ldz < s->D)))
    return bad("leading dimension below the width");
  if (s->ldb < 0 || s->ldb_group < 0 || s->ldc < 0 || s->ldc_group < 0) return bad("negative pitch");
  if (!s->n) return FB_OK;
  const uintptr_t es = s->type == FB_F32 ? 4 : 2;
  if (!aligned(es, s->u, s->delta, s->B, s->C, s->z, s->y)) return bad("rows that are not aligned to their elements");
  if (!aligned(4, s->A, s->skip, s->delta_bias, s->state) || !aligned(8, s->index))
    return bad("parameters, states or indices that are not aligned to their elements");
  ScanStep a{};
  a.D = s->D, a.N = s->N, a.per = s->D / s->G, a.softplus = s->softplus;
  a.vec = s->N % 4 == 0 && ((uintptr_t)s->state | (uintptr_t)s->A) % 16 == 0;
  a.u = s->u, a.ldu = s->ldu, a.delta = s->delta, a.ldd = s->ld_delta, a.B = s->B, a.ldb = s->ldb, a.gsb = s->ldb_group;
  a.C = s->C, a.ldc = s->ldc, a.gsc = s->ldc_group, a.z = s->z, a.ldz = s->ldz, a.y = s->y, a.ldy = s->ldy;
  a.A = s->A, a.Ds = s->skip, a.bias = s->delta_bias, a.state = s->state;
  const uint64_t bc = (uint64_t)s->ldb | (uint64_t)s->ldb_group | (uint64_t)s->ldc | (uint64_t)s->ldc_group;
  a.vec_bc = s->N % 4 == 0 && bc % 4 == 0 && ((uintptr_t)s->B | (uintptr_t)s->C) % (4 * es) == 0;
  FBH_TRY(rows_of("selective_scan_step", s->n, s->states, s->index, ws, ws_bytes, stream, a.r));
  return s->type == FB_F32 ? scan_step<float>(a, stream) : scan_step<bf16>(a, stream);
}
