// Short causal convolution of every column over packed histories, forward and
// backward.
//
//   p[t, d] = bias[d] + sum_k w[d, k] x[t - K + 1 + k, d],   y = p or silu(p)
//   dp = dy act'(p),  dx[i] = sum_j w[K - 1 - j] dp[i + j]  within the sequence
//   dw[k] = sum_t dp[t] x[t - K + 1 + k],  dbias = sum_t dp[t]
//
// Bound by memory: x read and y written, dy and x read and dx written.  A thread
// owns V columns and walks down a run of rows, 8 at a time, with the last K - 1
// inputs (and, backward, the last K - 1 dp) in registers, so every row is loaded
// once but for the K - 1 at a run's ends; the 8 loads of a step are in flight
// together.  Where sequences begin comes as one bit a row, which a CTA works out
// for its rows before it starts; a beginning replaces the window by assignment.
// p is computed again in the backward from x, which is there anyway.  dw and
// dbias are summed over a thread's run in registers, over a CTA in shared
// memory, and over the CTAs by a second launch in a fixed order.
#include <algorithm>
#include "head.cuh"
#include "history.cuh"

namespace {
using namespace fbq;

constexpr int kThreads = 256;
constexpr int kMaxTaps = 8;
constexpr int64_t kSms = 148;

struct ConvArgs {
  int D, K, silu;
  const void *x, *dy, *init, *dfin;
  void *y, *dx, *fin, *dinit;
  int64_t ldx, ldy, lddy, lddx;
  const float *w, *bias;
  float *part, *dw, *dbias;                // part [blocks, K + 1, D]
  Starts st;
  int cx, ry;                              // threads of a CTA along the columns, runs of rows
  int run;                                 // rows of a run, a multiple of 8
  int64_t blocks;                          // CTAs along the rows
};

// Sequence of a row, for one thread (few threads ask).
__device__ __forceinline__ int owner1(const Starts &st, int64_t row) {
  if (!st.p) return row < 0 ? -1 : (row < st.rows ? 0 : 1);
  int lo = 0, hi = st.seqs + 1;
  while (lo < hi) {
    const int m = lo + ((hi - lo) >> 1);
    if (st[m] <= row) lo = m + 1;
    else hi = m;
  }
  return lo - 1;
}

template <typename T, int V> __device__ __forceinline__ void load(const void *p, int64_t at, float (&v)[V]) {
  const Vec<T, V> e = *reinterpret_cast<const Vec<T, V> *>(static_cast<const T *>(p) + at);
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = to_f(e.e[i]);
}
template <typename T, int V> __device__ __forceinline__ void store(void *p, int64_t at, const float (&v)[V]) {
  Vec<T, V> e;
#pragma unroll
  for (int i = 0; i < V; ++i) e.e[i] = from_f<T>(v[i]);
  *reinterpret_cast<Vec<T, V> *>(static_cast<T *>(p) + at) = e;
}

// The beginnings of the rows from `from` (a multiple of 8) on, 8 to a byte.
__device__ __forceinline__ void fill_begins(const Starts &st, int64_t from, int tiles, uint8_t *bits) {
  const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int each = (tiles + warps - 1) / warps;
  Walk walk;
  const int a = warp * each, b = min(a + each, tiles);
  if (a >= b) return;
  walk.begin(st, from + 8 * (int64_t)a);
  for (int i = a; i < b; ++i) {
    const int64_t r0 = from + 8 * (int64_t)i;
    const unsigned m = r0 < 0 ? 0u : walk.tile(st, r0);
    if ((threadIdx.x & 31) == 0) bits[i] = (uint8_t)m;
  }
}

// What a thread works on.  KT: taps the registers hold; the first `skip` of them
// do not exist (they are left out, not multiplied by zero).
template <typename T, int V, int KT> struct Window {
  float x[KT - 1 + 8][V];                  // the last KT - 1 inputs, then 8 new ones
  // Inputs in front of the first row of sequence s, newest last.
  __device__ __forceinline__ void begin(const ConvArgs &a, int at, int64_t row, int64_t col, int skip) {
    int64_t s = -1;
    if (a.init) {
      s = owner1(a.st, row);
      if (s >= a.st.seqs) s = -1;
    }
#pragma unroll
    for (int m = 0; m < KT - 1; ++m)
#pragma unroll
      for (int i = 0; i < V; ++i)
        x[at + m][i] = s >= 0 && m >= skip
                           ? to_f(static_cast<const T *>(a.init)[(s * (a.K - 1) + m - skip) * (int64_t)a.D + col + i]) : 0.f;
  }
};

template <typename T, int V, int KT, bool BWD> __global__ void __launch_bounds__(kThreads) k_conv(ConvArgs a) {
  fb::pdl_enter();
  extern __shared__ __align__(16) unsigned char dyn[];
  const int64_t rows = a.st.rows;
  const int64_t block0 = (int64_t)blockIdx.y * a.ry * a.run;              // the CTA's first row
  uint8_t *const bits = dyn;                                              // rows block0 - 8 .. block0 + ry run + 15
  fill_begins(a.st, block0 - 8, a.ry * a.run / 8 + 3, bits);
  float *const sums = reinterpret_cast<float *>(dyn + (a.ry * a.run / 8 + 3 + 15) / 16 * 16);
  __syncthreads();

  const int c = threadIdx.x % a.cx, q = threadIdx.x / a.cx;
  const int64_t col = ((int64_t)blockIdx.x * a.cx + c) * V;
  const int64_t q0 = block0 + (int64_t)q * a.run, q1 = min(q0 + a.run, rows);
  const bool active = q < a.ry && col < a.D && q0 < q1;
  const int skip = KT - a.K;
  float dw[KT][V] = {}, db[V] = {};
  if (active) {
    const int64_t first = a.st[0], last = a.st[a.st.seqs];
    float w[KT][V], bias[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      bias[i] = a.bias ? a.bias[col + i] : 0.f;
#pragma unroll
      for (int k = 0; k < KT; ++k) w[k][i] = k >= skip ? a.w[(col + i) * a.K + k - skip] : 0.f;
    }
    const auto begins = [&](int64_t row) { return (bits[(row - block0 + 8) >> 3] >> (row & 7)) & 1u; };

    Window<T, V, KT> win;
    {
      // the inputs in front of the run: its own sequence's, as far as they go, older ones from init
      int64_t b = q0 - (KT - 1);                                           // first row of the sequence, if it is that near
      bool cut = false;
#pragma unroll
      for (int j = KT - 2; j >= 1; --j)
        if (q0 - j >= 0 && begins(q0 - j)) b = q0 - j, cut = true;
      if (q0 - (KT - 1) < 0 && !cut) b = 0, cut = true;
      int64_t s = -1;
      if (cut && a.init) {
        s = owner1(a.st, b);
        if (s >= a.st.seqs) s = -1;
      }
#pragma unroll
      for (int m = 0; m < KT - 1; ++m) {
        const int64_t r = q0 - (KT - 1) + m;
        const int64_t at = a.K - 1 + (r - b);                              // place in init, where r < b
        if (r >= b && r >= 0) load<T, V>(a.x, r * a.ldx + col, win.x[m]);
        else
#pragma unroll
          for (int i = 0; i < V; ++i)
            win.x[m][i] = s >= 0 && at >= 0 ? to_f(static_cast<const T *>(a.init)[(s * (a.K - 1) + at) * (int64_t)a.D + col + i]) : 0.f;
      }
    }
    float dp[BWD ? KT - 1 + 8 : 1][V];
    if constexpr (BWD) {
#pragma unroll
      for (int m = 0; m < KT - 1; ++m)
#pragma unroll
        for (int i = 0; i < V; ++i) dp[m][i] = 0.f;
    }
    // Backward, a dx row is complete K - 1 rows later: the walk goes on behind the run.
    const int64_t end = BWD ? q1 + KT - 1 : q1;
    for (int64_t t0 = q0; t0 < end; t0 += 8) {
      float dy[BWD ? 8 : 1][V];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool in = t0 + i < rows && t0 + i < end;
        if (in) load<T, V>(a.x, (t0 + i) * a.ldx + col, win.x[KT - 1 + i]);
        else
#pragma unroll
          for (int v = 0; v < V; ++v) win.x[KT - 1 + i][v] = 0.f;
        if constexpr (BWD) {
          if (in) load<T, V>(a.dy, (t0 + i) * a.lddy + col, dy[i]);
        }
      }
      const unsigned now = bits[(t0 - block0 + 8) >> 3];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int64_t t = t0 + i;
        if (now >> i & 1u) win.begin(a, i, t, col, skip);
        const bool live = t >= first && t < last && t < end;
        float p[V];
#pragma unroll
        for (int v = 0; v < V; ++v) p[v] = bias[v];
#pragma unroll
        for (int k = 0; k < KT; ++k)
          if (KT == 4 ? (k > 2 || k >= skip) : k >= skip)
#pragma unroll
            for (int v = 0; v < V; ++v) p[v] = fmaf(w[k][v], win.x[i + k][v], p[v]);
        if constexpr (!BWD) {
          if (t < q1) {
            float y[V];
#pragma unroll
            for (int v = 0; v < V; ++v) y[v] = live ? (a.silu ? p[v] * sigmoid(p[v]) : p[v]) : 0.f;
            store<T, V>(a.y, t * a.ldy + col, y);
          }
        } else {
          float(&d)[V] = dp[KT - 1 + i];
#pragma unroll
          for (int v = 0; v < V; ++v) {
            d[v] = live ? dy[i][v] : 0.f;
            if (a.silu && live) {
              const float sg = sigmoid(p[v]);
              d[v] *= sg * fmaf(p[v], 1.f - sg, 1.f);
            }
          }
          if (live && t < q1) {
#pragma unroll
            for (int v = 0; v < V; ++v) db[v] += d[v];
#pragma unroll
            for (int k = 0; k < KT; ++k)
              if (k >= skip)
#pragma unroll
                for (int v = 0; v < V; ++v) dw[k][v] = fmaf(d[v], win.x[i + k][v], dw[k][v]);
          }
        }
      }
      if constexpr (BWD) {
        // dx of the rows whose last dp has come
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int64_t r = t0 + i - (KT - 1);
          if (r < q0 || r >= q1) continue;
          float g[V];
#pragma unroll
          for (int v = 0; v < V; ++v) g[v] = w[KT - 1][v] * dp[i][v];
          bool same = true;
          int gap = KT;                                                    // rows to the sequence's end
#pragma unroll
          for (int j = 1; j < KT; ++j) {
            if (same && begins(r + j)) same = false, gap = j;
            if (same && KT - 1 - j >= skip)
#pragma unroll
              for (int v = 0; v < V; ++v) g[v] = fmaf(w[KT - 1 - j][v], dp[i + j][v], g[v]);
          }
          const bool live = r >= first && r < last;
          if (a.dfin && live && gap < a.K) {
            const int64_t s = owner1(a.st, r);
            if (s >= 0 && s < a.st.seqs)
#pragma unroll
              for (int v = 0; v < V; ++v)
                g[v] += to_f(static_cast<const T *>(a.dfin)[(s * (a.K - 1) + a.K - 1 - gap) * (int64_t)a.D + col + v]);
          }
          if (!live)
#pragma unroll
            for (int v = 0; v < V; ++v) g[v] = 0.f;
          store<T, V>(a.dx, r * a.lddx + col, g);
        }
#pragma unroll
        for (int m = 0; m < KT - 1; ++m)
#pragma unroll
          for (int v = 0; v < V; ++v) dp[m][v] = dp[m + 8][v];
      }
#pragma unroll
      for (int m = 0; m < KT - 1; ++m)
#pragma unroll
        for (int v = 0; v < V; ++v) win.x[m][v] = win.x[m + 8][v];
    }
  }
  if constexpr (BWD) {
    // the CTA's sums: the runs add up in order
    const int width = a.cx * V;
    for (int k = 0; k <= a.K; ++k) {
      if (q < a.ry && col < a.D)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          float x = db[v];
#pragma unroll
          for (int m = 0; m < KT; ++m)
            if (m == k + skip) x = dw[m][v];
          sums[q * width + c * V + v] = k < a.K ? x : db[v];
        }
      __syncthreads();
      for (int i = threadIdx.x; i < width; i += kThreads) {
        const int64_t d = (int64_t)blockIdx.x * width + i;
        if (d < a.D) {
          float x = 0.f;
          for (int j = 0; j < a.ry; ++j) x += sums[j * width + i];
          if (a.blocks > 1) a.part[((int64_t)blockIdx.y * (a.K + 1) + k) * a.D + d] = x;
          else if (k < a.K) a.dw[d * a.K + k] = x;
          else a.dbias[d] = x;
        }
      }
      __syncthreads();
    }
  }
}

__global__ void __launch_bounds__(256) k_conv_sums(ConvArgs a) {
  fb::pdl_enter();
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, n = (int64_t)(a.K + 1) * a.D;
  if (i >= n) return;
  float v = 0.f;
#pragma unroll 8
  for (int64_t b = 0; b < a.blocks; ++b) v += a.part[b * n + i];
  const int k = (int)(i / a.D);
  const int64_t d = i % a.D;
  if (k < a.K) a.dw[d * a.K + k] = v;
  else a.dbias[d] = v;
}

// final[s, m]: input number len - (K - 1) + m of sequence s; one thread an element.
template <typename T> __global__ void __launch_bounds__(256) k_conv_final(ConvArgs a) {
  fb::pdl_enter();
  const int64_t n = (int64_t)a.st.seqs * (a.K - 1) * a.D;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t d = i % a.D, m = i / a.D % (a.K - 1), s = i / a.D / (a.K - 1);
    const int64_t b = a.st[(int)s], e = max(a.st[(int)s + 1], b), p = e - b - (a.K - 1) + m;
    T v = from_f<T>(0.f);
    if (p >= 0) v = static_cast<const T *>(a.x)[(b + p) * a.ldx + d];
    else if (a.init) v = static_cast<const T *>(a.init)[(s * (a.K - 1) + a.K - 1 + p) * a.D + d];
    static_cast<T *>(a.fin)[i] = v;
  }
}

// dinit[s, m] = sum_{i <= m, i < len} w[m - i] dp[i] (+ dfinal[s, m - len]); one thread for a (sequence, column).
template <typename T> __global__ void __launch_bounds__(256) k_conv_dinit(ConvArgs a) {
  fb::pdl_enter();
  const int64_t n = (int64_t)a.st.seqs * a.D;
  for (int64_t j = (int64_t)blockIdx.x * 256 + threadIdx.x; j < n; j += (int64_t)gridDim.x * 256) {
    const int64_t d = j % a.D, s = j / a.D, b = a.st[(int)s], len = max(a.st[(int)s + 1] - b, (int64_t)0);
    const int K = a.K;
    const T *init = static_cast<const T *>(a.init) + s * (K - 1) * a.D + d;
    float w[kMaxTaps], x[2 * kMaxTaps], g[kMaxTaps];
    for (int k = 0; k < kMaxTaps; ++k) w[k] = k < K ? a.w[d * K + k] : 0.f;
    for (int m = 0; m < kMaxTaps - 1; ++m) {
      x[m] = m < K - 1 ? to_f(init[m * (int64_t)a.D]) : 0.f;
      g[m] = m < K - 1 && a.dfin && m >= len ? to_f(static_cast<const T *>(a.dfin)[(s * (K - 1) + m - len) * a.D + d]) : 0.f;
    }
    for (int i = 0; i < K - 1 && i < len; ++i) {
      x[K - 1 + i] = to_f(static_cast<const T *>(a.x)[(b + i) * a.ldx + d]);
      float p = a.bias ? a.bias[d] : 0.f, dp = to_f(static_cast<const T *>(a.dy)[(b + i) * a.lddy + d]);
      for (int k = 0; k < K; ++k) p = fmaf(w[k], x[i + k], p);
      if (a.silu) {
        const float sg = sigmoid(p);
        dp *= sg * fmaf(p, 1.f - sg, 1.f);
      }
      for (int m = i; m < K - 1; ++m) g[m] = fmaf(w[m - i], dp, g[m]);
    }
    for (int m = 0; m < K - 1; ++m) static_cast<T *>(a.dinit)[(s * (K - 1) + m) * a.D + d] = from_f<T>(g[m]);
  }
}

// ---- host ------------------------------------------------------------------------------------------
int fill(const fb_short_conv *s, ConvArgs &a, bool backward) {
  if (!s) return fb::set_error(FB_ERR_ARG, "short_conv: no arguments");
  const auto bad = [&](const char *what) { return fb::set_error(FB_ERR_ARG, std::string("short_conv: ") + what); };
  if (s->type != FB_F32 && s->type != FB_BF16) return bad("unknown element type");
  if (s->act != FB_ACT_NONE && s->act != FB_ACT_SILU) return bad("unknown activation");
  if (s->rows < 0 || s->D < 1 || s->K < 1 || s->seqs < 0) return bad("bad sizes");
  if (!s->starts && s->seqs != 1) return bad("without starts there is one sequence");
  if (s->starts_type != FB_I32 && s->starts_type != FB_I64) return bad("unknown type of starts");
  if (s->K > kMaxTaps) return fb::set_error(FB_ERR_UNSUPPORTED, "short_conv: at most 8 taps");
  if (s->D > (1 << 20) || s->rows > (int64_t)1 << 40 || s->seqs > (1 << 30))
    return fb::set_error(FB_ERR_UNSUPPORTED, "short_conv: sizes beyond what the kernels index");
  if (!s->w || (s->rows && !s->x)) return bad("missing operand");
  if (s->rows > 1 && s->ldx < s->D) return bad("leading dimension below the width");
  if (!backward && s->rows && (!s->y || (s->rows > 1 && s->ldy < s->D))) return bad("missing or overlapping output");
  if (backward && s->rows && (!s->dy || !s->dx || (s->rows > 1 && (s->lddy < s->D || s->lddx < s->D))))
    return bad("missing or overlapping operand of the backward pass");
  if (backward && (!s->dw || !s->dbias)) return bad("missing gradient");
  if (backward && s->dinit && !s->init) return bad("dinit without init");
  a = ConvArgs{};
  a.D = s->D, a.K = s->K, a.silu = s->act == FB_ACT_SILU;
  a.x = s->x, a.ldx = s->ldx, a.dy = s->dy, a.lddy = s->lddy, a.init = s->K > 1 ? s->init : nullptr;
  a.dfin = s->K > 1 ? s->dfinal : nullptr, a.fin = s->K > 1 ? s->final : nullptr, a.dinit = s->K > 1 ? s->dinit : nullptr;
  a.y = s->y, a.ldy = s->ldy, a.dx = s->dx, a.lddx = s->lddx, a.w = s->w, a.bias = s->bias, a.dw = s->dw, a.dbias = s->dbias;
  a.st = Starts{s->starts, s->starts_type == FB_I64, (int)s->seqs, s->rows};
  return FB_OK;
}

// Columns a thread moves at once: as many (up to 4) as bases, pitches and the width allow.
int vector_of(const fb_short_conv *s, bool backward) {
  const int es = s->type == FB_F32 ? 4 : 2;
  const void *p[2] = {backward ? s->dy : s->y, backward ? s->dx : nullptr};
  const int64_t ld[2] = {backward ? s->lddy : s->ldy, backward ? s->lddx : 0};
  uint64_t bits = (uint64_t)(uintptr_t)s->x / es | (uint64_t)s->D;
  if ((uintptr_t)s->x % es) return 0;
  if (s->rows > 1) bits |= (uint64_t)s->ldx;
  for (int i = 0; i < 2; ++i)
    if (p[i]) {
      if ((uintptr_t)p[i] % es) return 0;
      bits |= (uint64_t)(uintptr_t)p[i] / es;
      if (s->rows > 1) bits |= (uint64_t)ld[i];
    }
  return bits % 4 == 0 ? 4 : (bits % 2 == 0 ? 2 : 1);
}

// Columns of a CTA, runs side by side, rows of a run: long runs load few rows
// twice, but the SMs want two CTAs and more each.
void plan(ConvArgs &a, int V, bool backward) {
  const int groups = (a.D + V - 1) / V;
  a.cx = std::min(groups, kThreads);
  a.ry = kThreads / a.cx;
  const int64_t across = (groups + a.cx - 1) / a.cx;
  const int64_t want = std::max<int64_t>(1, kSms * (backward ? 4 : 8) / across);
  int64_t run = (a.st.rows + want * a.ry - 1) / (want * a.ry);
  run = std::min<int64_t>(std::max<int64_t>((run + 7) / 8 * 8, backward ? 32 : 16), 256);
  while (run * a.ry > 8192 && run > 8) run -= 8;
  a.run = (int)run;
  a.blocks = (a.st.rows + a.run * (int64_t)a.ry - 1) / (a.run * (int64_t)a.ry);
  // CTAs along the rows are a grid's y
  while (a.blocks > 65535) a.run *= 2, a.blocks = (a.st.rows + a.run * (int64_t)a.ry - 1) / (a.run * (int64_t)a.ry);
}

template <typename T, int V, int KT, bool BWD> int launch_main(const ConvArgs &a, cudaStream_t st) {
  const int width = a.cx * V;
  const size_t smem = (size_t)(a.ry * a.run / 8 + 3 + 15) / 16 * 16 + (BWD ? (size_t)a.ry * width * 4 : 0);
  if (smem > 48 * 1024) return fb::set_error(FB_ERR_UNSUPPORTED, "short_conv: too many rows");
  const dim3 grid((unsigned)((a.D + width - 1) / width), (unsigned)a.blocks);
  FB_TRY_CUDA(fb::launch(k_conv<T, V, KT, BWD>, grid, kThreads, smem, st, a));
  return FB_OK;
}

template <typename T, bool BWD> int launch_v(const ConvArgs &a, int V, cudaStream_t st) {
  if (a.K <= 4) return V == 4 ? launch_main<T, 4, 4, BWD>(a, st) : V == 2 ? launch_main<T, 2, 4, BWD>(a, st) : launch_main<T, 1, 4, BWD>(a, st);
  return V == 4 ? launch_main<T, 4, 8, BWD>(a, st) : V == 2 ? launch_main<T, 2, 8, BWD>(a, st) : launch_main<T, 1, 8, BWD>(a, st);
}

unsigned some_blocks(int64_t n) { return (unsigned)std::min<int64_t>((n + 255) / 256, kSms * 8); }

template <typename T> int run_conv(const fb_short_conv *s, ConvArgs &a, bool backward, void *ws, size_t ws_bytes, cudaStream_t st) {
  const int64_t state = (int64_t)a.st.seqs * (a.K - 1) * a.D;
  if (s->rows) {
    const int V = vector_of(s, backward);
    if (!V) return fb::set_error(FB_ERR_ARG, "short_conv: rows that are not aligned to their elements");
    plan(a, V, backward);
    if (backward && a.blocks > 1) {
      const size_t need = (size_t)a.blocks * (a.K + 1) * a.D * sizeof(float);
      FBH_TRY(fbh::check_ws(ws, "short_conv"));
      if (ws_bytes < need) return fb::set_error(FB_ERR_ARG, "short_conv: workspace too small");
      a.part = static_cast<float *>(ws);
    }
    FBH_TRY((backward ? launch_v<T, true>(a, V, st) : launch_v<T, false>(a, V, st)));
    if (backward && a.blocks > 1) FB_TRY_CUDA(fb::launch(k_conv_sums, dim3((unsigned)(((a.K + 1) * (int64_t)a.D + 255) / 256)), 256, 0, st, a));
  } else if (backward) {
    FB_TRY_CUDA(cudaMemsetAsync(a.dw, 0, (size_t)a.D * a.K * sizeof(float), st));
    FB_TRY_CUDA(cudaMemsetAsync(a.dbias, 0, (size_t)a.D * sizeof(float), st));
  }
  if (!backward && a.fin && state) FB_TRY_CUDA(fb::launch(k_conv_final<T>, some_blocks(state), 256, 0, st, a));
  if (backward && a.dinit && state) FB_TRY_CUDA(fb::launch(k_conv_dinit<T>, some_blocks(a.st.seqs * (int64_t)a.D), 256, 0, st, a));
  return FB_OK;
}

int run_any(const fb_short_conv *s, bool backward, void *ws, size_t ws_bytes, cudaStream_t st) {
  ConvArgs a;
  FBH_TRY(fill(s, a, backward));
  return s->type == FB_F32 ? run_conv<float>(s, a, backward, ws, ws_bytes, st) : run_conv<bf16>(s, a, backward, ws, ws_bytes, st);
}

}  // namespace

extern "C" size_t fb_short_conv_ws_bytes(const fb_short_conv *s, int backward) {
  if (!s || !backward || s->rows <= 0 || s->D < 1 || s->K < 1 || s->K > kMaxTaps) return 0;
  size_t most = 0;
  for (int V = 1; V <= 4; V *= 2) {        // whatever alignment the call's rows turn out to have
    ConvArgs a{};
    a.D = s->D, a.K = s->K, a.st.rows = s->rows;
    plan(a, V, true);
    most = std::max(most, a.blocks > 1 ? (size_t)a.blocks * (s->K + 1) * s->D * sizeof(float) : (size_t)0);
  }
  return most;
}

extern "C" int fb_short_conv_fwd(const fb_short_conv *s, void *ws, size_t ws_bytes, cudaStream_t stream) {
  return run_any(s, false, ws, ws_bytes, stream);
}

extern "C" int fb_short_conv_bwd(const fb_short_conv *s, void *ws, size_t ws_bytes, cudaStream_t stream) {
  return run_any(s, true, ws, ws_bytes, stream);
}
