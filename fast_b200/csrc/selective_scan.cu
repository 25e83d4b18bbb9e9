// Selective state space scan over packed histories, forward and backward.
//
//   dt = softplus(delta + delta_bias)   (or delta + delta_bias as it is)
//   h[t] = exp(dt A) h[t-1] + dt u B[t]      per channel d and state n
//   v = sum_n C[t] h[t] + D u,   y = v silu(z)
//
//   gv = dy silu(z),  dz = dy v silu'(z)
//   g[t] = C gv + r[t],  r[t-1] = exp(dt A) g[t]      (r = dfinal behind a sequence)
//   dC = sum_d gv h,  dB = sum_d g dt u,  du = dt <g, B> + D gv
//   q = g exp(dt A) h[t-1] = r[t-1] h[t-1]
//   ddelta = (<q, A> + u <g, B>) softplus',  dA = sum_t q dt,  dD = sum_t gv u
//
// What bounds it: instructions.  The special function units give 16 exponentials
// a clock and SM, so at 16 states one clock for each (row, channel) and pass; the
// bytes (8 a (row, channel) in bf16, gate included) take 0.36 of that, and the
// packed fp32 arithmetic about as much as the exponentials.  So the layout saves
// what surrounds them:
//
// - A warp owns a tile of channels and walks down the rows.  A thread holds 4
//   channels x 4 states (2 x 4 in the backward): what is read from shared memory
//   per row (dt, dt u of its channels, B, C of its states) serves several of
//   them.  Channels sit in pairs, which the packed instructions take two at a
//   time.  Sums over states and over channels go through shared memory: each lane
//   stores its parts, whoever needs a sum adds them (with shuffles, in which
//   every lane ended up with one sum, the backward took 485 us instead of 444 at
//   16,384 x 1,024, 16 states, bf16).
// - Rows come in tiles of 8.  Their softplus, dt u and the gate are computed
//   once for each (row, channel) with the lanes along the channels; the next
//   tile's loads are in flight meanwhile.  Any pitch and alignment is the same.
//   Tiles in which no sequence begins run without a branch.
// - The packed rows are cut into chunks of a fixed number of rows wherever the
//   sequences begin, so the grid needs nothing from the device.  A first pass
//   reduces each chunk to its last state, from the last beginning of a sequence
//   on (decay over the chunk: exp(A sum dt)), a second joins the chunks in
//   order, the third computes the rows.  Sequences begin by assignment, never by
//   a factor of 0: an infinity stays in its own sequence.  One chunk needs one
//   launch.
// - For a backward pass the forward keeps the state in front of every 8th row,
//   N / 2 bytes a (row, channel): written beside arithmetic that leaves the memory
//   idle, and cheaper than another pass of exponentials.  The backward recomputes
//   4 rows of states and decays into registers and walks them back: 8 rows at
//   once take the registers of the third CTA an SM (906 us against 866, both
//   passes).
// - Sums over rows and channels end in per-CTA partials that one more launch
//   adds in a fixed order: results repeat bit for bit.
//
// 16,384 x 1,024, 64 ragged sequences, bf16, 16 states: both passes 832 us; under a
// profiler, with cold caches, forward 89 (last states) + 14 + 170, backward 95 (first
// gradients) + 12 + 464 + 18; at 148 SMs and 1.9 GHz the exponentials alone take 60 us
// a pass.
//
// Everything between the loads and the stores is fp32.
#include <algorithm>
#include <type_traits>
#include "head.cuh"
#include "history.cuh"

namespace {
using namespace fbq;

constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kMaxStates = 64;
constexpr int kHalf = kTile / 2;          // rows whose states the backward holds at once
// CTAs an SM that the registers are shared among.  A fourth in the forward takes
// what keeps a row's instructions apart: both passes of 12,000 x 200 fp32 224 us,
// 242 with four, of 5,003 x 413 162 and 177, of 16,384 x 1,024 bf16 825 and 821; five
// and six spill (957, 1,094).
constexpr int kFwdCtas = 3, kBwdCtas = 3;
constexpr int kKept = 1;                  // pairs of a thread whose decays it holds, too

struct ScanArgs {
  int D, N, G, per, tiles, softplus;      // per: channels of a group; tiles: a group's tiles of channels
  const void *u, *delta, *B, *C, *z, *dy;
  int64_t ldu, ldd, ldb, gsb, ldc, gsc, ldz, lddy;
  const float *A, *Ds, *bias, *init, *dfin;
  float *fin, *dinit;
  void *y, *du, *ddelta, *dz, *dB, *dC;
  int64_t ldy;
  float *keep;                            // [ceil(rows / 8), D, N] states in front of every 8th row
  float *edge;                            // [nc - 1, D, N] what crosses the chunks' borders
  float *sumdt;                           // [nc - 1, D]
  int *cut;                               // [nc - 1] nothing passes through the chunk
  float *pA, *pD, *pBC;                   // partial sums: [nc, D, N], [nc, 2, D], [G ctas, rows, 2 NP]
  float *dA, *dD, *dbias;
  Starts st;
  int64_t chunk;                          // rows, a multiple of kTile
  int nc, ctas;                           // chunks; CTAs side by side on a group (backward)
  int vec;                                // states move four at a time
};

// Four states from n0 on of one channel.
__device__ __forceinline__ void load4(const float *p, int n0, int N, int vec, float (&v)[4]) {
  if (vec) {
    const float4 f = *reinterpret_cast<const float4 *>(p + n0);
    v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
    return;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) v[k] = n0 + k < N ? p[n0 + k] : 0.f;
}
__device__ __forceinline__ void store4(float *p, int n0, int N, int vec, const float (&v)[4]) {
  if (vec) {
    *reinterpret_cast<float4 *>(p + n0) = make_float4(v[0], v[1], v[2], v[3]);
    return;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (n0 + k < N) p[n0 + k] = v[k];
}

// The states of a thread: P pairs of channels x 4 states.
template <int P> struct States {
  F2 v[P][4];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int k = 0; k < 4; ++k) v[p][k] = pack(0.f, 0.f);
  }
  // From / to [D, N] rows at `base`; c: channel (in the tensor) of the thread's first, `has` of them exist.
  __device__ __forceinline__ void load(const float *base, int c, int has, int n0, const ScanArgs &a) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      float x[2][4] = {};
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (2 * p + j < has && n0 < a.N) load4(base + (c + 2 * p + j) * a.N, n0, a.N, a.vec, x[j]);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[p][k] = pack(x[0][k], x[1][k]);
    }
  }
  __device__ __forceinline__ void store(float *base, int c, int has, int n0, const ScanArgs &a) const {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      float x[2][4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 f = unpack(v[p][k]);
        x[0][k] = f.x, x[1][k] = f.y;
      }
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (2 * p + j < has && n0 < a.N) store4(base + (c + 2 * p + j) * a.N, n0, a.N, a.vec, x[j]);
    }
  }
};

// The sum of the values that L neighbouring lanes left at p.
template <int L> __device__ __forceinline__ float lanes_sum(const float *p) {
  float v = 0.f;
  if constexpr (L == 2) {
    const float2 f = *reinterpret_cast<const float2 *>(p);
    v = f.x + f.y;
  } else {
#pragma unroll
    for (int i = 0; i < L; i += 4) {
      const float4 f = *reinterpret_cast<const float4 *>(p + i);
      v += (f.x + f.y) + (f.z + f.w);
    }
  }
  return v;
}

// A warp's tile: kTile rows x CH channels, or x NP states.  The lanes lie along the
// columns; element i of a lane is row(i), col(i).
template <int COLS> struct Tile {
  static constexpr int E = kTile * COLS / 32;                            // elements a lane
  static constexpr int W = COLS > 32 ? COLS / 32 : 1;                    // columns a lane meets
  static constexpr int RS = COLS > 32 ? 1 : 32 / COLS;                   // rows between a column's elements
  static __device__ __forceinline__ int col(int i) { return (threadIdx.x & 31) % COLS + 32 * (i % W); }
  static __device__ __forceinline__ int row(int i) { return COLS > 32 ? i / W : (threadIdx.x & 31) / COLS + RS * i; }
  // Loads the rows [a, b) of the tile whose first row, first column is at p.
  template <typename T> static __device__ __forceinline__ void fetch(T (&x)[E], const void *base, int64_t at, int64_t ld, int cols, int a,
                                                                     int b) {
    const T *p = static_cast<const T *>(base) + at + row(0) * ld + col(0);
    const T none = from_f<T>(0.f);
    const int64_t step = RS * ld;
    if (a == 0 && b == kTile) {
#pragma unroll
      for (int i = 0; i < E; i += W, p += step)
#pragma unroll
        for (int w = 0; w < W; ++w) x[i + w] = col(w) < cols ? p[32 * w] : none;
    } else {
#pragma unroll
      for (int i = 0; i < E; i += W, p += step)
#pragma unroll
        for (int w = 0; w < W; ++w) x[i + w] = col(w) < cols && row(i) >= a && row(i) < b ? p[32 * w] : none;
    }
  }
};

// A thread's place: NP states (padded to 8, 16, 32 or 64) of P pairs of channels a thread.
template <int NP, int P> struct Lay {
  static constexpr int NL = NP / 4, CL = 32 / NL, CH = 2 * P * CL;       // lanes along states, channels; channels a warp
  using X = Tile<CH>;
  using S = Tile<NP>;
  // Where a channel's lanes lie in their row of parts: moved by whole groups, so that the groups of neighbouring
  // channels, read together, meet different banks.
  static __device__ __forceinline__ int turn(int by) { return by & ~(NL - 1); }
};

// v with the elements of the rows outside [a, b) at zero.
template <typename X> __device__ __forceinline__ float only(float v, int i, int a, int b) {
  return X::row(i) >= a && X::row(i) < b ? v : 0.f;
}

// dt of a lane's elements (pairs of them) and, with SLOPE, the derivative by delta.
template <bool SLOPE, typename X, typename T> __device__ __forceinline__ void steps(const T (&raw)[X::E], const float (&bias)[X::W], int sp,
                                                                                   float (&dt)[X::E], float (&slope)[X::E]) {
#pragma unroll
  for (int i = 0; i < X::E; i += 2) {
    const int j = i + 1 < X::E ? i + 1 : i;
    const F2 x = add2(pack(to_f(raw[i]), to_f(raw[j])), pack(bias[i % X::W], bias[j % X::W]));
    F2 sl = both(1.f);
    const float2 v = unpack(sp ? softplus2<SLOPE>(x, sl) : x), k = unpack(sl);
    dt[i] = v.x, dt[j] = X::E > 1 ? v.y : v.x;
    if (SLOPE) slope[i] = k.x, slope[j] = X::E > 1 ? k.y : k.x;
  }
}

template <int NP> struct FwdSmem {
  static constexpr int CH = Lay<NP, 2>::CH;
  float dt[kTile][CH], dtu[kTile][CH];
  float y[kTile][4][32];                                                 // each lane's part of its 4 channels' y
  float2 B[kTile][NP], C[kTile][NP];                                     // each value twice: a pair's factor
};

__device__ __forceinline__ int rows_in(int64_t v) { return (int)max((int64_t)0, min((int64_t)kTile, v)); }

// Forward.  LOCAL: the chunk's last state alone, from the last beginning of a
// sequence on, for all chunks but the last.
template <typename T, int NP, bool LOCAL> __global__ void __launch_bounds__(kThreads, kFwdCtas) k_scan_fwd(ScanArgs a) {
  using L = Lay<NP, 2>;
  using X = typename L::X;
  using S = typename L::S;
  fb::pdl_enter();
  extern __shared__ __align__(16) unsigned char dyn[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  FwdSmem<NP> &sm = reinterpret_cast<FwdSmem<NP> *>(dyn)[warp];
  const int nct = a.G * a.tiles;
  const int64_t wid = (int64_t)blockIdx.x * kWarps + warp;
  const int64_t chunk = wid / nct;
  const int ct = (int)(wid % nct);
  if (chunk >= a.nc - (LOCAL ? 1 : 0)) return;
  const int grp = ct / a.tiles, ch0 = (ct % a.tiles) * L::CH, left = a.per - ch0;   // channels the tile has
  const int cb = grp * a.per + ch0, size = a.D * a.N;
  const int nl = lane % L::NL, cl = lane / L::NL, n0 = nl * 4;
  const int mine = cb + cl * 4;
  const int has = left - cl * 4;
  const int64_t rows = a.st.rows, c0 = chunk * a.chunk, c1 = min(c0 + a.chunk, rows);

  States<2> A2, h;
  A2.load(a.A, mine, has, n0, a);
#pragma unroll
  for (int p = 0; p < 2; ++p)
#pragma unroll
    for (int k = 0; k < 4; ++k) A2.v[p][k] = pack(scaled(unpack(A2.v[p][k]).x), scaled(unpack(A2.v[p][k]).y));
  h.zero();

  int64_t lo, hi;                                 // rows that count
  Walk walk;
  if constexpr (LOCAL) {
    const int s = owner(a.st, c1 - 1);
    const bool in = s >= 0 && s < a.st.seqs;
    const int64_t b = in ? a.st[s] : 0;
    const bool ends = !in || a.st[s + 1] <= c1;   // nothing goes on into the next chunk
    if (ct == 0 && lane == 0) a.cut[chunk] = ends || b >= c0;
    lo = ends ? c1 : max(b, c0), hi = c1;
    if (!ends && b >= c0 && a.init) h.load(a.init + (int64_t)s * size, mine, has, n0, a);
  } else {
    walk.begin(a.st, c0);
    lo = a.st[0], hi = min(a.st[a.st.seqs], c1);
    if (chunk > 0) h.load(a.edge + (chunk - 1) * (int64_t)size, mine, has, n0, a);
  }

  float bias[X::W], skip[X::W];
#pragma unroll
  for (int w = 0; w < X::W; ++w) {
    const int c = X::col(w);
    bias[w] = a.bias && c < left ? a.bias[cb + c] : 0.f;
    skip[w] = !LOCAL && a.Ds && c < left ? a.Ds[cb + c] : 0.f;
  }
  T xu[X::E], xd[X::E], xb[S::E], xc[LOCAL ? 1 : S::E];
  const auto fetch = [&](int64_t r0) {
    const int ra = rows_in(lo - r0), rb = rows_in(hi - r0);
    X::fetch(xu, a.u, r0 * a.ldu + cb, a.ldu, left, ra, rb);
    X::fetch(xd, a.delta, r0 * a.ldd + cb, a.ldd, left, ra, rb);
    S::fetch(xb, a.B, r0 * a.ldb + grp * a.gsb, a.ldb, a.N, ra, rb);
    if constexpr (!LOCAL) S::fetch(xc, a.C, r0 * a.ldc + grp * a.gsc, a.ldc, a.N, ra, rb);
  };

  F2 total[2] = {both(0.f), both(0.f)};
  const auto row = [&](int i) {
    F2 dt[2], dtu[2], B[4], C[4], y[2];
    const ulonglong2 t = *reinterpret_cast<const ulonglong2 *>(&sm.dt[i][cl * 4]);
    const ulonglong2 x = *reinterpret_cast<const ulonglong2 *>(&sm.dtu[i][cl * 4]);
    const ulonglong2 *b = reinterpret_cast<const ulonglong2 *>(&sm.B[i][n0]);
    dt[0].v = t.x, dt[1].v = t.y, dtu[0].v = x.x, dtu[1].v = x.y;
    B[0].v = b[0].x, B[1].v = b[0].y, B[2].v = b[1].x, B[3].v = b[1].y;
    if constexpr (!LOCAL) {
      const ulonglong2 *c = reinterpret_cast<const ulonglong2 *>(&sm.C[i][n0]);
      C[0].v = c[0].x, C[1].v = c[0].y, C[2].v = c[1].x, C[3].v = c[1].y;
    }
#pragma unroll
    for (int p = 0; p < 2; ++p) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const F2 decay = decays(dt[p], A2.v[p][k]);
        h.v[p][k] = fma2(decay, h.v[p][k], mul2(dtu[p], B[k]));
        if constexpr (!LOCAL) y[p] = k == 0 ? mul2(C[k], h.v[p][k]) : fma2(C[k], h.v[p][k], y[p]);
      }
      if constexpr (LOCAL) total[p] = add2(total[p], dt[p]);
    }
    if constexpr (!LOCAL) {
      const float2 ya = unpack(y[0]), yb = unpack(y[1]);
      const float v[4] = {ya.x, ya.y, yb.x, yb.y};
#pragma unroll
      for (int j = 0; j < 4; ++j) sm.y[i][j][lane ^ L::turn(j * 8)] = v[j];
    }
  };

  int64_t r0 = LOCAL ? c0 + (lo - c0) / kTile * kTile : c0;
  if (r0 < c1) fetch(r0);
  for (; r0 < c1; r0 += kTile) {
    const int ra = rows_in(lo - r0), rb = rows_in(hi - r0);
    float dt[X::E], slope[X::E];
    T ku[X::E], kz[X::E];
    steps<false, X>(xd, bias, a.softplus, dt, slope);
#pragma unroll
    for (int i = 0; i < X::E; ++i) {
      const float v = only<X>(dt[i], i, ra, rb);
      sm.dt[X::row(i)][X::col(i)] = v;
      sm.dtu[X::row(i)][X::col(i)] = v * to_f(xu[i]);
      ku[i] = xu[i];
    }
#pragma unroll
    for (int i = 0; i < S::E; ++i) {
      const float b = to_f(xb[i]);
      sm.B[S::row(i)][S::col(i)] = make_float2(b, b);
      if constexpr (!LOCAL) {
        const float c = to_f(xc[i]);
        sm.C[S::row(i)][S::col(i)] = make_float2(c, c);
      }
    }
    unsigned begins = 0;
    if constexpr (!LOCAL) {
      begins = walk.tile(a.st, r0);
      if (c1 - r0 < kTile) begins &= (1u << (int)(c1 - r0)) - 1u;
      if (a.z) X::fetch(kz, a.z, r0 * a.ldz + cb, a.ldz, left, ra, rb);
    }
    if (r0 + kTile < c1) fetch(r0 + kTile);
    __syncwarp();
    if (!LOCAL && a.keep) h.store(a.keep + r0 / kTile * size, mine, has, n0, a);
    if (LOCAL || begins == 0) {
#pragma unroll
      for (int i = 0; i < kTile; ++i) row(i);
    } else {
#pragma unroll 1
      for (int i = 0; i < kTile; ++i) {
        if (begins >> i & 1u) {
          const int64_t at = r0 + i;
          if (a.fin && at > c0) {                 // the sequence in front leaves its last state
            const int s = walk.sequence(a.st, at - 1);
            if (s >= 0 && s < a.st.seqs) h.store(a.fin + (int64_t)s * size, mine, has, n0, a);
          }
          h.zero();
          if (a.init) {
            const int s = walk.sequence(a.st, at);
            if (s >= 0 && s < a.st.seqs) h.load(a.init + (int64_t)s * size, mine, has, n0, a);
          }
        }
        row(i);
      }
    }
    __syncwarp();
    if constexpr (!LOCAL) {
      T *py = static_cast<T *>(a.y) + (r0 + X::row(0)) * a.ldy + cb + X::col(0);
      const int end = rows_in(c1 - r0);
#pragma unroll
      for (int i = 0; i < X::E; ++i) {
        const int c = X::col(i);
        float v = fmaf(skip[i % X::W], to_f(ku[i]), lanes_sum<L::NL>(&sm.y[X::row(i)][c & 3][((c >> 2) * L::NL) ^ L::turn((c & 3) * 8)]));
        if (a.z) {
          const float z = to_f(kz[i]);
          v *= z * sigmoid<T>(z);
        }
        if (X::row(i) < end && X::col(i) < left) py[i / X::W * X::RS * a.ldy + 32 * (i % X::W)] = from_f<T>(only<X>(v, i, ra, rb));
      }
    }
  }
  if constexpr (LOCAL) {
    __syncwarp();
    h.store(a.edge + chunk * (int64_t)size, mine, has, n0, a);
    if (nl == 0) {
      const float2 x = unpack(total[0]), y = unpack(total[1]);
      const float t[4] = {x.x, x.y, y.x, y.y};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < has) a.sumdt[chunk * a.D + mine + j] = t[j];
    }
  } else if (a.fin) {
    const int s = owner(a.st, c1 - 1);
    if (s >= 0 && s < a.st.seqs && a.st[s + 1] <= c1) h.store(a.fin + (int64_t)s * size, mine, has, n0, a);
    for (int q = (int)chunk; q < a.st.seqs; q += 32 * a.nc) {          // empty sequences end as they began
      const int e = q + lane * a.nc;
      unsigned m = __ballot_sync(0xffffffffu, e < a.st.seqs && a.st[e] >= a.st[e + 1]);
      for (; m; m &= m - 1) {
        const int64_t s0 = q + (__ffs(m) - 1) * a.nc;
        States<2> x;
        x.zero();
        if (a.init) x.load(a.init + s0 * size, mine, has, n0, a);
        x.store(a.fin + s0 * size, mine, has, n0, a);
      }
    }
  }
}

// Joins the chunks: edge[c], what chunk c alone leaves, becomes what arrives
// behind it (REV: in front of chunk c + 1, from the rows behind).
// A chunk's factor is applied as its root, twice: where states grow (A > 0) it can
// lie beyond fp32 and what it makes of a small state inside; of a 0 it makes 0.
// Bound by the latency of its loads, so 32 chunks' are in flight (188 chunks of
// width 200: 20 us with 8).
template <bool REV> __global__ void __launch_bounds__(128) k_scan_join(ScanArgs a) {
  fb::pdl_enter();
  const int64_t i = (int64_t)blockIdx.x * 128 + threadIdx.x, size = (int64_t)a.D * a.N;
  if (i >= size) return;
  const int c = (int)(i / a.N);
  const float A2 = scaled(a.A[i]);
  constexpr int kAhead = 32;
  const int n = a.nc - 1;
  float x = 0.f;
  for (int at = 0; at < n; at += kAhead) {
    float local[kAhead], sum[kAhead];
    int cut[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int j = at + k < n ? (REV ? n - 1 - (at + k) : at + k) : 0;
      local[k] = a.edge[j * size + i], sum[k] = a.sumdt[(int64_t)j * a.D + c], cut[k] = a.cut[j];
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (at + k < n) {
        const float root = ex2(A2 * sum[k] * 0.5f);
        x = cut[k] || x == 0.f ? local[k] : fmaf(root, root * x, local[k]);
        a.edge[(REV ? n - 1 - (at + k) : at + k) * size + i] = x;
      }
  }
}

// ---- backward ------------------------------------------------------------------------------------
template <int NP> struct RevSmem {
  static constexpr int CH = Lay<NP, 2>::CH;
  float dt[kTile][CH], gv[kTile][CH];
  float2 C[kTile][NP];
};

// What chunk c (all but the first) sends up to the chunk in front of it: r in
// front of its first row, from the rows of the sequence that comes in.
template <typename T, int NP> __global__ void __launch_bounds__(kThreads, kFwdCtas) k_scan_rev(ScanArgs a) {
  using L = Lay<NP, 2>;
  using X = typename L::X;
  using S = typename L::S;
  fb::pdl_enter();
  __shared__ __align__(16) RevSmem<NP> smem[kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  RevSmem<NP> &sm = smem[warp];
  const int nct = a.G * a.tiles;
  const int64_t wid = (int64_t)blockIdx.x * kWarps + warp;
  const int64_t chunk = wid / nct + 1;
  const int ct = (int)(wid % nct);
  if (chunk >= a.nc) return;
  const int grp = ct / a.tiles, ch0 = (ct % a.tiles) * L::CH, left = a.per - ch0;
  const int cb = grp * a.per + ch0, size = a.D * a.N;
  const int nl = lane % L::NL, cl = lane / L::NL, n0 = nl * 4;
  const int mine = cb + cl * 4;
  const int has = left - cl * 4;
  const int64_t rows = a.st.rows, c0 = chunk * a.chunk, c1 = min(c0 + a.chunk, rows);

  States<2> A2, r;
  A2.load(a.A, mine, has, n0, a);
#pragma unroll
  for (int p = 0; p < 2; ++p)
#pragma unroll
    for (int k = 0; k < 4; ++k) A2.v[p][k] = pack(scaled(unpack(A2.v[p][k]).x), scaled(unpack(A2.v[p][k]).y));
  r.zero();
  const int s = owner(a.st, c0);
  const bool in = s >= 0 && s < a.st.seqs && a.st[s] < c0;      // a sequence comes in
  const int64_t end = in ? a.st[s + 1] : c0, e = min(end, c1);
  if (ct == 0 && lane == 0) a.cut[chunk - 1] = !in || end <= c1;
  if (in && end <= c1 && a.dfin) r.load(a.dfin + (int64_t)s * size, mine, has, n0, a);

  float bias[X::W];
#pragma unroll
  for (int w = 0; w < X::W; ++w) bias[w] = a.bias && X::col(w) < left ? a.bias[cb + X::col(w)] : 0.f;
  T xd[X::E], xy[X::E], xz[X::E], xc[S::E];
  const auto fetch = [&](int64_t r0) {
    const int rb = rows_in(e - r0);
    X::fetch(xd, a.delta, r0 * a.ldd + cb, a.ldd, left, 0, rb);
    X::fetch(xy, a.dy, r0 * a.lddy + cb, a.lddy, left, 0, rb);
    if (a.z) X::fetch(xz, a.z, r0 * a.ldz + cb, a.ldz, left, 0, rb);
    S::fetch(xc, a.C, r0 * a.ldc + grp * a.gsc, a.ldc, a.N, 0, rb);
  };
  F2 total[2] = {both(0.f), both(0.f)};
  int64_t r0 = e > c0 ? c0 + (e - 1 - c0) / kTile * kTile : c0 - kTile;
  if (r0 >= c0) fetch(r0);
  for (; r0 >= c0; r0 -= kTile) {
    const int rb = rows_in(e - r0);
    float dt[X::E], slope[X::E];
    steps<false, X>(xd, bias, a.softplus, dt, slope);
#pragma unroll
    for (int i = 0; i < X::E; ++i) {
      float gv = to_f(xy[i]);
      if (a.z) {
        const float z = to_f(xz[i]);
        gv *= z * sigmoid<T>(z);
      }
      sm.dt[X::row(i)][X::col(i)] = only<X>(dt[i], i, 0, rb);
      sm.gv[X::row(i)][X::col(i)] = only<X>(gv, i, 0, rb);
    }
#pragma unroll
    for (int i = 0; i < S::E; ++i) {
      const float c = to_f(xc[i]);
      sm.C[S::row(i)][S::col(i)] = make_float2(c, c);
    }
    if (r0 - kTile >= c0) fetch(r0 - kTile);
    __syncwarp();
#pragma unroll
    for (int i = kTile - 1; i >= 0; --i) {
      const ulonglong2 t = *reinterpret_cast<const ulonglong2 *>(&sm.dt[i][cl * 4]);
      const ulonglong2 x = *reinterpret_cast<const ulonglong2 *>(&sm.gv[i][cl * 4]);
      const ulonglong2 *c = reinterpret_cast<const ulonglong2 *>(&sm.C[i][n0]);
      const F2 dt2[2] = {{t.x}, {t.y}}, gv[2] = {{x.x}, {x.y}}, C[4] = {{c[0].x}, {c[0].y}, {c[1].x}, {c[1].y}};
#pragma unroll
      for (int p = 0; p < 2; ++p) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          r.v[p][k] = mul2(decays(dt2[p], A2.v[p][k]), fma2(C[k], gv[p], r.v[p][k]));
        total[p] = add2(total[p], dt2[p]);
      }
    }
    __syncwarp();
  }
  r.store(a.edge + (chunk - 1) * (int64_t)size, mine, has, n0, a);
  if (nl == 0) {
    const float2 x = unpack(total[0]), y = unpack(total[1]);
    const float t[4] = {x.x, x.y, y.x, y.y};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < has) a.sumdt[(chunk - 1) * a.D + mine + j] = t[j];
  }
}

// Pairs of channels a thread of the backward holds: one, but for the widest
// states, whose warps would have fewer elements than lanes.
template <int NP> constexpr int kBwdPairs = NP > 32 ? 2 : 1;

template <int NP> struct BwdSmem {
  static constexpr int P = kBwdPairs<NP>, CH = Lay<NP, P>::CH;
  float dt[kWarps][kTile][CH], dtu[kWarps][kTile][CH], gv[kWarps][kTile][CH];
  float out[kWarps][3][kHalf][2 * P][32];                            // each lane's part of <g, B>, <q, A log2 e>, <C, h>
  float B[kTile][NP], C[kTile][NP];                             // once: here the accesses cost more than doubling them
  float4 sum[kWarps][kHalf][2][32];                              // each lane's part of dB, dC of its states
  float4 own[kWarps][Lay<NP, P>::X::E][32];                      // u, dy silu'(z), softplus', dt of each lane's elements
  int seq[kWarps][kTile + 1];                                    // of the rows in front of and at beginnings
};

// All gradients of a chunk's rows.  The warps of a CTA stand side by side on a
// group's channels and add up their parts of dB and dC.
template <typename T, int NP> __global__ void __launch_bounds__(kThreads, NP > 32 ? 2 : kBwdCtas) k_scan_bwd(ScanArgs a) {
  constexpr int P = kBwdPairs<NP>;
  using L = Lay<NP, P>;
  using X = typename L::X;
  fb::pdl_enter();
  extern __shared__ __align__(16) unsigned char dyn[];
  BwdSmem<NP> &sm = *reinterpret_cast<BwdSmem<NP> *>(dyn);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int grp = blockIdx.x / a.ctas, cta = blockIdx.x % a.ctas;
  const int chunk = blockIdx.y;
  const int ch0 = (cta * kWarps + warp) * L::CH, left = a.per - ch0;        // may be <= 0: a warp without channels
  const int cb = grp * a.per + ch0, size = a.D * a.N;
  const int nl = lane % L::NL, cl = lane / L::NL, n0 = nl * 4;
  const int mine = cb + cl * (2 * P);
  const int has = left - cl * (2 * P);
  const int64_t rows = a.st.rows, c0 = chunk * a.chunk, c1 = min(c0 + a.chunk, rows);
  // from here on rows are counted from c0
  const int len = (int)(c1 - c0), lo = (int)max((int64_t)0, min(a.st[0] - c0, (int64_t)len)),
            hi = (int)max((int64_t)0, min(a.st[a.st.seqs] - c0, (int64_t)len));

  States<P> A2, r, dA;
  A2.load(a.A, mine, has, n0, a);
#pragma unroll
  for (int p = 0; p < P; ++p)
#pragma unroll
    for (int k = 0; k < 4; ++k) A2.v[p][k] = pack(scaled(unpack(A2.v[p][k]).x), scaled(unpack(A2.v[p][k]).y));
  dA.zero();
  r.zero();
  {
    const int s = owner(a.st, c1 - 1);
    const bool in = s >= 0 && s < a.st.seqs;
    if (c1 >= rows || !in || a.st[s + 1] <= c1) {
      if (in && a.dfin) r.load(a.dfin + (int64_t)s * size, mine, has, n0, a);
    } else {
      r.load(a.edge + chunk * (int64_t)size, mine, has, n0, a);
    }
  }

  float bias[X::W], skip[X::W], sumD[X::W] = {}, sumb[X::W] = {};
#pragma unroll
  for (int w = 0; w < X::W; ++w) {
    const int c = X::col(w);
    bias[w] = a.bias && c < left ? a.bias[cb + c] : 0.f;
    skip[w] = a.Ds && c < left ? a.Ds[cb + c] : 0.f;
  }
  const T none = from_f<T>(0.f);
  constexpr int EC = kTile * NP / kThreads > 0 ? kTile * NP / kThreads : 1;  // B (and C) elements a thread of the CTA
  T xu[X::E], xd[X::E], xy[X::E], xz[X::E], xb[EC], xc[EC];
  const auto fetch = [&](int t0) {
    const int ra = min(max(lo - t0, 0), kTile), rb = t0 >= 0 ? min(max(hi - t0, 0), kTile) : 0;
    const int64_t r0 = c0 + t0;
    X::fetch(xu, a.u, r0 * a.ldu + cb, a.ldu, left, ra, rb);
    X::fetch(xd, a.delta, r0 * a.ldd + cb, a.ldd, left, ra, rb);
    X::fetch(xy, a.dy, r0 * a.lddy + cb, a.lddy, left, ra, rb);
    if (a.z) X::fetch(xz, a.z, r0 * a.ldz + cb, a.ldz, left, ra, rb);
#pragma unroll
    for (int i = 0; i < EC; ++i) {
      const int at = threadIdx.x + kThreads * i, n = at % NP, row = at / NP;
      const bool ok = at < kTile * NP && n < a.N && row >= ra && row < rb;
      xb[i] = ok ? static_cast<const T *>(a.B)[(r0 + row) * a.ldb + grp * a.gsb + n] : none;
      xc[i] = ok ? static_cast<const T *>(a.C)[(r0 + row) * a.ldc + grp * a.gsc + n] : none;
    }
  };

  WalkDown walk;
  walk.begin(a.st, c1 - 1);
  int t0 = (len - 1) / kTile * kTile;
  fetch(t0);
  for (; t0 >= 0; t0 -= kTile) {
    // ---- the tile's rows, once for each (row, channel); rows of no sequence were fetched as zeros
    {
      const int ra = lo - t0, rb = hi - t0;
      float dt[X::E], slope[X::E];
      steps<true, X>(xd, bias, a.softplus, dt, slope);
#pragma unroll
      for (int i = 0; i < X::E; i += 2) {
        const F2 u = pack(to_f(xu[i]), to_f(xu[i + 1])), dy = pack(to_f(xy[i]), to_f(xy[i + 1]));
        F2 gv = dy, dg = both(0.f);
        if (a.z) {
          const F2 z = pack(to_f(xz[i]), to_f(xz[i + 1]));
          F2 rest;
          const F2 sg = sigmoid2<T>(z, rest);
          gv = mul2(dy, mul2(z, sg));
          dg = mul2(dy, silu_slope2<T>(z, sg, rest));
        }
        const F2 v = pack(only<X>(dt[i], i, ra, rb), only<X>(dt[i + 1], i + 1, ra, rb));
        const float2 fu = unpack(u), fg = unpack(gv), fd = unpack(dg), fv = unpack(v), fp = unpack(mul2(v, u));
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int row = X::row(i + j), c = X::col(i + j);
          sm.dt[warp][row][c] = j ? fv.y : fv.x;
          sm.dtu[warp][row][c] = j ? fp.y : fp.x;
          sm.gv[warp][row][c] = j ? fg.y : fg.x;
          sm.own[warp][i + j][lane] = j ? make_float4(fu.y, fd.y, slope[i + 1], fv.y) : make_float4(fu.x, fd.x, slope[i], fv.x);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < EC; ++i) {
      const int at = threadIdx.x + kThreads * i;
      if (at < kTile * NP) {
        const float b = to_f(xb[i]), c = to_f(xc[i]);
        sm.B[at / NP][at % NP] = b;
        sm.C[at / NP][at % NP] = c;
      }
    }
    const unsigned begins = walk.tile(a.st, c0 + t0);
    if (begins && (a.init || a.dfin || a.dinit)) {
#pragma unroll 1
      for (int i = 0; i <= kTile; ++i) {
        const int s = walk.sequence(a.st, c0 + t0 + i - 1);
        if (lane == 0) sm.seq[warp][i] = s >= 0 && s < a.st.seqs ? s : -1;
      }
    }
    States<P> from;                                              // the state in front of the rows in work
    from.load(a.keep + (c0 + t0) / kTile * size, mine, has, n0, a);
    __syncthreads();

    // What a sequence finds that begins at row i of the tile.
    const auto found = [&](States<P> &x, int i) {
      x.zero();
      if (a.init) {
        const int s = sm.seq[warp][i + 1];
        if (s >= 0) x.load(a.init + (int64_t)s * size, mine, has, n0, a);
      }
    };
    // The pairs' dt, dt u or gv of a row; B or C of the states, twice each.
    const auto pairs = [&](const float (&p)[kTile][L::CH], int i, F2 (&v)[P]) {
      if constexpr (P == 1) {
        v[0].v = *reinterpret_cast<const unsigned long long *>(&p[i][cl * 2]);
      } else {
        const ulonglong2 t = *reinterpret_cast<const ulonglong2 *>(&p[i][cl * 4]);
        v[0].v = t.x, v[1].v = t.y;
      }
    };
    const auto twice = [&](const float (&p)[kTile][NP], int i, F2 (&v)[4]) {
      const float4 f = *reinterpret_cast<const float4 *>(&p[i][n0]);
      v[0] = both(f.x), v[1] = both(f.y), v[2] = both(f.z), v[3] = both(f.w);
    };
    // h behind row i; the decays of the first pair are kept
    const auto ahead = [&](int i, States<P> &h, F2 (&kept)[4]) {
      F2 dt[P], dtu[P], B[4];
      pairs(sm.dt[warp], i, dt), pairs(sm.dtu[warp], i, dtu), twice(sm.B, i, B);
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const F2 d = decays(dt[p], A2.v[p][k]);
          if (p < kKept) kept[k] = d;
          h.v[p][k] = fma2(d, h.v[p][k], mul2(dtu[p], B[k]));
        }
    };
    // BEGINS: some row of the tile begins a sequence.
    const auto half = [&](auto some, auto from_row) {
      constexpr bool BEGINS = decltype(some)::value;
      constexpr int at = decltype(from_row)::value;
      F2 as[kHalf][4];
      if constexpr (at > 0) {
#pragma unroll
        for (int i = 0; i < kHalf; ++i) {
          if (BEGINS && (begins >> i & 1u)) found(from, i);
          ahead(i, from, as[0]);
        }
      } else {
        from.load(a.keep + (c0 + t0) / kTile * size, mine, has, n0, a);
      }
      // ---- states of half the rows
      States<P> hs[kHalf];
#pragma unroll
      for (int j = 0; j < kHalf; ++j) {
        hs[j] = j ? hs[j - 1] : from;
        if (BEGINS && (begins >> (at + j) & 1u)) found(hs[j], at + j);
        ahead(at + j, hs[j], as[j]);
      }
      // ---- back up the rows
#pragma unroll
      for (int j = kHalf - 1; j >= 0; --j) {
        const int i = at + j;
        F2 dt[P], dtu[P], gv[P], B[4], C[4];
        pairs(sm.dt[warp], i, dt), pairs(sm.dtu[warp], i, dtu), pairs(sm.gv[warp], i, gv);
        twice(sm.B, i, B), twice(sm.C, i, C);
        States<P> before = j ? hs[j - 1] : from;
        if (BEGINS && (begins >> i & 1u)) found(before, i);
        F2 gB[P], qA[P], cy[P];
        float vb[4], vc[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          F2 sb, sc;
#pragma unroll
          for (int p = 0; p < P; ++p) {
            const F2 g = fma2(C[k], gv[p], r.v[p][k]), h = hs[j].v[p][k];
            r.v[p][k] = mul2(p < kKept ? as[j][k] : decays(dt[p], A2.v[p][k]), g);
            const F2 q = mul2(r.v[p][k], before.v[p][k]);
            gB[p] = k == 0 ? mul2(g, B[k]) : fma2(g, B[k], gB[p]);
            qA[p] = k == 0 ? mul2(q, A2.v[p][k]) : fma2(q, A2.v[p][k], qA[p]);
            cy[p] = k == 0 ? mul2(C[k], h) : fma2(C[k], h, cy[p]);
            dA.v[p][k] = fma2(q, dt[p], dA.v[p][k]);
            sb = p == 0 ? mul2(g, dtu[p]) : fma2(g, dtu[p], sb);
            sc = p == 0 ? mul2(gv[p], h) : fma2(gv[p], h, sc);
          }
          const float2 x = unpack(sb), y = unpack(sc);
          vb[k] = x.x + x.y, vc[k] = y.x + y.y;
        }
#pragma unroll
        for (int p = 0; p < P; ++p) {
          const float2 v[3] = {unpack(gB[p]), unpack(qA[p]), unpack(cy[p])};
#pragma unroll
          for (int m = 0; m < 3; ++m) {
            sm.out[warp][m][j][2 * p][lane ^ L::turn(16 / P * (2 * p))] = v[m].x;
            sm.out[warp][m][j][2 * p + 1][lane ^ L::turn(16 / P * (2 * p + 1))] = v[m].y;
          }
        }
        sm.sum[warp][j][0][lane] = make_float4(vb[0], vb[1], vb[2], vb[3]);
        sm.sum[warp][j][1][lane] = make_float4(vc[0], vc[1], vc[2], vc[3]);
        if (BEGINS && (begins >> i & 1u)) {
          if (a.dinit && sm.seq[warp][i + 1] >= 0) r.store(a.dinit + (int64_t)sm.seq[warp][i + 1] * size, mine, has, n0, a);
          r.zero();
          if (a.dfin && sm.seq[warp][i] >= 0) r.load(a.dfin + (int64_t)sm.seq[warp][i] * size, mine, has, n0, a);
        }
      }
    };
    const auto both_ways = [&](auto from_row) {
      constexpr int at = decltype(from_row)::value;
      if (begins) half(std::true_type{}, from_row);
      else half(std::false_type{}, from_row);
      if constexpr (at == 0) fetch(t0 - kTile);                  // nothing in front of the chunk
      __syncthreads();

      // ---- results of the half
      const int end = len - t0;
      const int64_t to = (c0 + t0 + X::row(0)) * a.D + cb + X::col(0);
      const int skipped = at ? X::E / 2 : 0;                     // the lane's elements of the other half
#pragma unroll
      for (int e = 0; e < X::E / 2; ++e) {
        const int i = e + skipped, row = X::row(0) + X::RS * (i / X::W), w = e % X::W, c = X::col(w);
        const float4 own = sm.own[warp][i][lane];
        const auto total = [&](int m) {
          return lanes_sum<L::NL>(&sm.out[warp][m][row - at][c % (2 * P)][(c / (2 * P) * L::NL) ^ L::turn(16 / P * (c % (2 * P)))]);
        };
        const float gB = total(0), qA = total(1) * 0.6931471805599453f, gv = sm.gv[warp][row][c];
        const float dd = fmaf(own.x, gB, qA) * own.z;
        if (row >= end || c >= left) continue;
        sumD[w] = fmaf(gv, own.x, sumD[w]), sumb[w] += dd;
        const int64_t q = to + i / X::W * X::RS * (int64_t)a.D + 32 * w;
        if (a.z) static_cast<T *>(a.dz)[q] = from_f<T>(fmaf(skip[w], own.x, total(2)) * own.y);
        static_cast<T *>(a.du)[q] = from_f<T>(fmaf(own.w, gB, skip[w] * gv));
        static_cast<T *>(a.ddelta)[q] = from_f<T>(dd);
      }
      // dB and dC of 4 states of a row: kParts threads share the lanes' parts
      constexpr int kSums = kHalf * 2 * L::NL, kParts = kSums < kThreads ? kThreads / kSums : 1;
#pragma unroll
      for (int t = threadIdx.x; t < kSums * kParts; t += kThreads) {
        const int l = t % L::NL, part = t / L::NL % kParts, which = t / (L::NL * kParts) % 2, row = t / (L::NL * kParts * 2);
        F2 v01 = both(0.f), v23 = both(0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w)
#pragma unroll
          for (int m = part; m < L::CL; m += kParts) {
            const ulonglong2 f = *reinterpret_cast<const ulonglong2 *>(&sm.sum[w][row][which][m * L::NL + l]);
            v01 = add2(v01, F2{f.x}), v23 = add2(v23, F2{f.y});
          }
        const float2 v0 = unpack(v01), v2 = unpack(v23);
        float4 v = make_float4(v0.x, v0.y, v2.x, v2.y);
#pragma unroll
        for (int o = L::NL; o < L::NL * kParts; o *= 2) {
          v.x += __shfl_xor_sync(0xffffffffu, v.x, o), v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
          v.z += __shfl_xor_sync(0xffffffffu, v.z, o), v.w += __shfl_xor_sync(0xffffffffu, v.w, o);
        }
        if (at + row >= end || part) continue;
        const int64_t q = c0 + t0 + at + row;
        if (a.ctas > 1) {
          *reinterpret_cast<float4 *>(&a.pBC[(blockIdx.x * rows + q) * (2 * NP) + which * NP + l * 4]) = v;
        } else {
          T *const p = static_cast<T *>(which ? a.dC : a.dB) + (q * a.G + grp) * a.N + l * 4;
          const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (l * 4 + k < a.N) p[k] = from_f<T>(f[k]);
        }
      }
      if (at) __syncthreads();
    };
    both_ways(std::integral_constant<int, kHalf>{});
    both_ways(std::integral_constant<int, 0>{});
  }

  dA.store((a.nc > 1 ? a.pA + chunk * (int64_t)size : a.dA), mine, has, n0, a);
#pragma unroll
  for (int w = 0; w < X::W; ++w) {
    if (L::CH < 32) {
#pragma unroll
      for (int o = L::CH; o < 32; o <<= 1) {
        sumD[w] += __shfl_xor_sync(0xffffffffu, sumD[w], o);
        sumb[w] += __shfl_xor_sync(0xffffffffu, sumb[w], o);
      }
    }
    const int c = X::col(w);
    if (c < left && lane < L::CH) {
      if (a.nc > 1) a.pD[chunk * 2 * (int64_t)a.D + cb + c] = sumD[w], a.pD[(chunk * 2 + 1) * (int64_t)a.D + cb + c] = sumb[w];
      else a.dD[cb + c] = sumD[w], a.dbias[cb + c] = sumb[w];
    }
  }
  if (a.dinit) {
    for (int q = (int)chunk; q < a.st.seqs; q += 32 * a.nc) {          // empty sequences: dfinal passes through
      const int e = q + lane * a.nc;
      unsigned m = __ballot_sync(0xffffffffu, e < a.st.seqs && a.st[e] >= a.st[e + 1]);
      for (; m; m &= m - 1) {
        const int64_t s0 = q + (__ffs(m) - 1) * a.nc;
        States<P> x;
        x.zero();
        if (a.dfin) x.load(a.dfin + s0 * size, mine, has, n0, a);
        x.store(a.dinit + s0 * size, mine, has, n0, a);
      }
    }
  }
}

// Adds the partials in order: first the CTAs side by side (dB, dC; blocks below
// bc_blocks), then the chunks (dA, dD, ddelta_bias).
template <typename T> __global__ void __launch_bounds__(256) k_scan_sums(ScanArgs a, int NP, int64_t bc_blocks) {
  fb::pdl_enter();
  const int64_t rows = a.st.rows;
  if (blockIdx.x < bc_blocks) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;               // [G, rows, 2 NP]
    const int64_t width = rows * 2 * NP;
    if (i >= width * a.G) return;
    const int grp = (int)(i / width), col = (int)(i % (2 * NP));
    const int64_t q = i % width / (2 * NP);
    const float *p = a.pBC + grp * a.ctas * width + i % width;
    float v = 0.f;
#pragma unroll 8
    for (int k = 0; k < a.ctas; ++k) v += p[k * width];
    if (col % NP < a.N) static_cast<T *>(col < NP ? a.dB : a.dC)[(q * a.G + grp) * a.N + col % NP] = from_f<T>(v);
    return;
  }
  // 32 sums a CTA, 8 threads each
  __shared__ float part[8][32];
  const int64_t i = (blockIdx.x - bc_blocks) * 32 + threadIdx.x % 32, size = (int64_t)a.D * a.N, all = size + 2 * (int64_t)a.D;
  const float *p = i < size ? a.pA + i : a.pD + (i - size);
  const int64_t step = i < size ? size : 2 * (int64_t)a.D;
  float v = 0.f;
  if (i < all) {
#pragma unroll 8
    for (int k = threadIdx.x / 32; k < a.nc; k += 8) v += p[k * step];
  }
  part[threadIdx.x / 32][threadIdx.x % 32] = v;
  __syncthreads();
  if (threadIdx.x >= 32 || i >= all) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) v += part[k][threadIdx.x];
  if (i < size) a.dA[i] = v;
  else if (i < size + a.D) a.dD[i - size] = v;
  else a.dbias[i - size - a.D] = v;
}

// ---- host ------------------------------------------------------------------------------------------
int padded(int N) { return N <= 8 ? 8 : (N <= 16 ? 16 : (N <= 32 ? 32 : 64)); }

// Rows of a chunk, for `tiles` units of work side by side of which the GPU holds
// `resident`: whole waves of units as long as the chunks keep `shortest` rows, for
// then early ends of some chunks even out.  16,384 x 1,024 bf16, both passes:
// backward in one wave 922 us, two 881, three 866; forward in three 845, two
// 834.  Shorter chunks lose more to the passes between them than they gain:
// forward of 2,048 x 2,048 with chunks of at least 32, 48, 64, 96 rows 76, 73,
// 78, 111 us; both passes of 12,000 x 200 fp32 243, 243, 239, 242, with 32, 64, 96
// rows in the backward 260, 243, 246.
// Where one wave is not filled, a row's latency counts, not the instructions:
// chunks of down to kLeast rows (35 scans of sizes drawn from the whole range:
// 50.7 us in the geometric mean with 32, 47.8 with 24, 44.9 with 16).
constexpr int64_t kLeast = 16;
int64_t chunk_rows(int64_t rows, int64_t tiles, int64_t resident, int64_t waves, int64_t shortest) {
  for (;; --waves) {
    const int64_t want = std::max<int64_t>(1, resident * waves / tiles);
    const int64_t even = ((rows + want - 1) / want + kTile - 1) / kTile * kTile;
    if (even >= shortest) return even;
    if (waves == 1) return std::max(even, kLeast);
  }
}

int fill(const fb_selective_scan *s, ScanArgs &a, bool backward) {
  const char *const who = "selective_scan";
  if (!s) return fb::set_error(FB_ERR_ARG, "selective_scan: no arguments");
  const auto bad = [&](const char *what) { return fb::set_error(FB_ERR_ARG, std::string(who) + ": " + what); };
  if (s->type != FB_F32 && s->type != FB_BF16) return bad("unknown element type");
  if (s->rows < 0 || s->D < 1 || s->N < 1 || s->G < 1 || s->D % s->G || s->seqs < 0) return bad("bad sizes");
  if (!s->starts && s->seqs != 1) return bad("without starts there is one sequence");
  if (s->starts_type != FB_I32 && s->starts_type != FB_I64) return bad("unknown type of starts");
  if (s->N > kMaxStates) return fb::set_error(FB_ERR_UNSUPPORTED, "selective_scan: at most 64 states");
  if (s->D > (1 << 20) || s->rows > (int64_t)1 << 40 || s->seqs > (1 << 30))
    return fb::set_error(FB_ERR_UNSUPPORTED, "selective_scan: sizes beyond what the kernels index");
  if (s->rows && (!s->u || !s->delta || !s->B || !s->C)) return bad("missing operand");
  if (!s->A) return bad("missing operand");
  if (s->rows > 1 && (s->ldu < s->D || s->ld_delta < s->D || (s->z && s->ldz < s->D))) return bad("leading dimension below the width");
  if (s->rows && !backward && (!s->y || (s->rows > 1 && s->ldy < s->D))) return bad("missing or overlapping output");
  if (backward) {
    if (s->rows && (!s->dy || (s->rows > 1 && s->lddy < s->D) || !s->keep)) return bad("missing operand of the backward pass");
    if (s->rows && (!s->du || !s->ddelta || !s->dB || !s->dC || (s->z && !s->dz))) return bad("missing gradient");
    if (!s->dA || !s->dD || !s->ddelta_bias) return bad("missing gradient");
  }
  if (s->ldb < 0 || s->ldb_group < 0 || s->ldc < 0 || s->ldc_group < 0) return bad("negative pitch");
  const uintptr_t es = s->type == FB_F32 ? 4 : 2;
  if (!aligned(es, s->u, s->delta, s->B, s->C, s->z) ||
      !(backward ? aligned(es, s->dy, s->du, s->ddelta, s->dz, s->dB, s->dC) : aligned(es, s->y)))
    return bad("rows that are not aligned to their elements");
  if (!aligned(4, s->A, s->skip, s->delta_bias, s->init, s->keep) ||
      !(backward ? aligned(4, s->dfinal, s->dA, s->dD, s->ddelta_bias, s->dinit) : aligned(4, s->final)) ||
      !aligned(s->starts_type == FB_I64 ? 8 : 4, s->starts))
    return bad("parameters, states or starts that are not aligned to their elements");
  a = ScanArgs{};
  a.D = s->D, a.N = s->N, a.G = s->G, a.per = s->D / s->G, a.softplus = s->softplus;
  a.u = s->u, a.ldu = s->ldu, a.delta = s->delta, a.ldd = s->ld_delta;
  a.B = s->B, a.ldb = s->ldb, a.gsb = s->ldb_group, a.C = s->C, a.ldc = s->ldc, a.gsc = s->ldc_group;
  a.z = s->z, a.ldz = s->ldz, a.A = s->A, a.Ds = s->skip, a.bias = s->delta_bias, a.init = s->init, a.fin = s->final;
  a.y = s->y, a.ldy = s->ldy, a.keep = s->keep;
  a.dy = s->dy, a.lddy = s->lddy, a.du = s->du, a.ddelta = s->ddelta, a.dz = s->dz, a.dB = s->dB, a.dC = s->dC;
  a.dA = s->dA, a.dD = s->dD, a.dbias = s->ddelta_bias, a.dfin = s->dfinal, a.dinit = s->dinit;
  a.st = Starts{s->starts, s->starts_type == FB_I64, (int)s->seqs, s->rows};
  const uintptr_t at = (uintptr_t)s->A | (uintptr_t)s->init | (uintptr_t)s->final | (uintptr_t)s->keep | (uintptr_t)s->dfinal |
                       (uintptr_t)s->dinit | (uintptr_t)s->dA;
  a.vec = s->N % 4 == 0 && at % 16 == 0;
  return FB_OK;
}

constexpr int64_t kSms = 148;

// The forward's split, and its pieces of the workspace.
int plan_fwd(ScanArgs &a, int np, fbh::Call &c) {
  const int ch = 2 * 2 * 32 / (np / 4);
  a.tiles = (a.per + ch - 1) / ch;
  a.chunk = chunk_rows(a.st.rows, (int64_t)a.G * a.tiles, kSms * kFwdCtas * kWarps, 2, 48);
  a.nc = (int)std::max<int64_t>(1, (a.st.rows + a.chunk - 1) / a.chunk);
  if (a.nc > 1) {
    FBH_TAKE(edge, c, float, (a.nc - 1) * (int64_t)a.D * a.N);
    FBH_TAKE(sum, c, float, (a.nc - 1) * (int64_t)a.D);
    FBH_TAKE(cut, c, int, a.nc - 1);
    a.edge = edge, a.sumdt = sum, a.cut = cut;
  }
  return FB_OK;
}

int plan_bwd(ScanArgs &a, int np, fbh::Call &c) {
  const int ch = 2 * (np > 32 ? 2 : 1) * 32 / (np / 4);   // channels of a warp
  const int tiles = (a.per + ch - 1) / ch;
  a.ctas = (tiles + kWarps - 1) / kWarps;
  a.chunk = chunk_rows(a.st.rows, (int64_t)a.G * a.ctas, kSms * (np > 32 ? 2 : kBwdCtas), 3, 64);
  a.nc = (int)std::max<int64_t>(1, (a.st.rows + a.chunk - 1) / a.chunk);
  a.tiles = (a.per + 4 * 32 / (np / 4) - 1) / (4 * 32 / (np / 4));          // k_scan_rev's
  const int64_t size = (int64_t)a.D * a.N;
  if (a.nc > 1) {
    FBH_TAKE(edge, c, float, (a.nc - 1) * size);
    FBH_TAKE(sum, c, float, (a.nc - 1) * (int64_t)a.D);
    FBH_TAKE(cut, c, int, a.nc - 1);
    FBH_TAKE(pA, c, float, a.nc * size);
    FBH_TAKE(pD, c, float, a.nc * 2 * (int64_t)a.D);
    a.edge = edge, a.sumdt = sum, a.cut = cut, a.pA = pA, a.pD = pD;
  }
  if (a.ctas > 1) {
    FBH_TAKE(pBC, c, float, (int64_t)a.G * a.ctas * a.st.rows * 2 * np);
    a.pBC = pBC;
  }
  return FB_OK;
}

unsigned blocks(int64_t n, int64_t each) { return (unsigned)((n + each - 1) / each); }

// Shared memory above what a launch has without asking.
template <typename K> int allow(K *kernel, size_t bytes) {
  if (bytes > 48 * 1024) FB_TRY_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
  return FB_OK;
}

template <typename T, int NP> int run_fwd(const ScanArgs &a, cudaStream_t stream) {
  const int64_t nct = (int64_t)a.G * a.tiles;
  constexpr size_t smem = sizeof(FwdSmem<NP>) * kWarps;
  FBH_TRY((allow(k_scan_fwd<T, NP, true>, smem)));
  FBH_TRY((allow(k_scan_fwd<T, NP, false>, smem)));
  if (a.nc > 1) {
    FB_TRY_CUDA(fb::launch(k_scan_fwd<T, NP, true>, blocks(nct * (a.nc - 1), kWarps), kThreads, smem, stream, a));
    FB_TRY_CUDA(fb::launch(k_scan_join<false>, blocks((int64_t)a.D * a.N, 128), 128, 0, stream, a));
  }
  FB_TRY_CUDA(fb::launch(k_scan_fwd<T, NP, false>, blocks(nct * a.nc, kWarps), kThreads, smem, stream, a));
  return FB_OK;
}

template <typename T, int NP> int run_bwd(const ScanArgs &a, cudaStream_t stream) {
  constexpr size_t smem = sizeof(BwdSmem<NP>);
  FBH_TRY((allow(k_scan_bwd<T, NP>, smem)));
  if (a.nc > 1) {
    const int64_t nct = (int64_t)a.G * a.tiles;
    FB_TRY_CUDA(fb::launch(k_scan_rev<T, NP>, blocks(nct * (a.nc - 1), kWarps), kThreads, 0, stream, a));
    FB_TRY_CUDA(fb::launch(k_scan_join<true>, blocks((int64_t)a.D * a.N, 128), 128, 0, stream, a));
  }
  FB_TRY_CUDA(fb::launch(k_scan_bwd<T, NP>, dim3((unsigned)(a.G * a.ctas), (unsigned)a.nc), kThreads, smem, stream, a));
  const int64_t bc = a.ctas > 1 ? blocks((int64_t)a.G * a.st.rows * 2 * NP, 256) : 0;
  const int64_t rest = a.nc > 1 ? blocks((int64_t)a.D * (a.N + 2), 32) : 0;
  if (bc + rest) FB_TRY_CUDA(fb::launch(k_scan_sums<T>, dim3((unsigned)(bc + rest)), 256, 0, stream, a, (int)NP, bc));
  return FB_OK;
}

template <bool BWD, typename T> int run_states(const ScanArgs &a, int np, cudaStream_t st) {
  switch (np) {
    case 8: return BWD ? run_bwd<T, 8>(a, st) : run_fwd<T, 8>(a, st);
    case 16: return BWD ? run_bwd<T, 16>(a, st) : run_fwd<T, 16>(a, st);
    case 32: return BWD ? run_bwd<T, 32>(a, st) : run_fwd<T, 32>(a, st);
    default: return BWD ? run_bwd<T, 64>(a, st) : run_fwd<T, 64>(a, st);
  }
}

template <bool BWD> int run(const fb_selective_scan *s, void *ws, size_t ws_bytes, cudaStream_t stream) {
  ScanArgs a;
  FBH_TRY(fill(s, a, BWD));
  const size_t state = (size_t)s->seqs * s->D * s->N * sizeof(float);
  if (!s->rows) {                                          // nothing but empty sequences
    if (!BWD && s->final && state) {
      if (s->init) FB_TRY_CUDA(cudaMemcpyAsync(s->final, s->init, state, cudaMemcpyDeviceToDevice, stream));
      else FB_TRY_CUDA(cudaMemsetAsync(s->final, 0, state, stream));
    }
    if (BWD) {
      if (s->dinit && state) {
        if (s->dfinal) FB_TRY_CUDA(cudaMemcpyAsync(s->dinit, s->dfinal, state, cudaMemcpyDeviceToDevice, stream));
        else FB_TRY_CUDA(cudaMemsetAsync(s->dinit, 0, state, stream));
      }
      FB_TRY_CUDA(cudaMemsetAsync(s->dA, 0, (size_t)s->D * s->N * sizeof(float), stream));
      FB_TRY_CUDA(cudaMemsetAsync(s->dD, 0, (size_t)s->D * sizeof(float), stream));
      FB_TRY_CUDA(cudaMemsetAsync(s->ddelta_bias, 0, (size_t)s->D * sizeof(float), stream));
    }
    return FB_OK;
  }
  const int np = padded(s->N);
  fbh::Call need;
  {
    ScanArgs b = a;
    FBH_TRY(BWD ? plan_bwd(b, np, need) : plan_fwd(b, np, need));
  }
  if (need.peak) {
    FBH_TRY(fbh::check_ws(ws, "selective_scan"));
    if (ws_bytes < need.peak) return fb::set_error(FB_ERR_ARG, "selective_scan: workspace too small");
  }
  fbh::Call c(ws, ws_bytes, stream);
  FBH_TRY(BWD ? plan_bwd(a, np, c) : plan_fwd(a, np, c));
  return s->type == FB_F32 ? run_states<BWD, float>(a, np, stream) : run_states<BWD, bf16>(a, np, stream);
}

}  // namespace

extern "C" size_t fb_selective_scan_ws_bytes(const fb_selective_scan *s, int backward) {
  if (!s || s->rows <= 0 || s->D < 1 || s->N < 1 || s->N > kMaxStates || s->G < 1 || s->D % s->G) return 0;
  ScanArgs a{};
  a.D = s->D, a.N = s->N, a.G = s->G, a.per = s->D / s->G, a.st.rows = s->rows;
  fbh::Call c;
  if (backward ? plan_bwd(a, padded(s->N), c) : plan_fwd(a, padded(s->N), c)) return 0;
  return c.peak;
}

extern "C" int fb_selective_scan_fwd(const fb_selective_scan *s, void *ws, size_t ws_bytes, cudaStream_t stream) {
  return run<false>(s, ws, ws_bytes, stream);
}

extern "C" int fb_selective_scan_bwd(const fb_selective_scan *s, void *ws, size_t ws_bytes, cudaStream_t stream) {
  return run<true>(s, ws, ws_bytes, stream);
}
