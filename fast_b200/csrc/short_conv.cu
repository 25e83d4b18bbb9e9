// Short causal convolution of every column over packed histories, forward and
// backward.
//
//   p[t, d] = bias[d] + sum_k w[d, k] x[t - K + 1 + k, d],   y = p or silu(p)
//   dp = dy act'(p),  dx[i] = sum_j w[K - 1 - j] dp[i + j]  within the sequence
//   dw[k] = sum_t dp[t] x[t - K + 1 + k],  dbias = sum_t dp[t]
//
// Bound by memory: x read and y written, dy and x read and dx written.  A thread
// owns up to 4 columns and walks down a run of rows with the last K - 1 inputs
// (and, backward, the last K - 1 dp) in registers, so every row is loaded once
// but for the K - 1 at a run's ends.  Loads are asynchronous copies into places
// of the thread's own, two batches of four rows ahead: held in registers instead
// they cost the warps that hide the latency (32,768 x 2,048 bf16 forward and
// backward: loads where they are used 646 + 118 us, two batches of registers
// 208 + 88, copies 121 + 61; the bytes take 61 + 41).  What holds them now is neither
// memory nor issue slots (53% and 57% used): 14 and 19 warps an SM wait for the
// results of their own instructions.  Above four taps one form of eight serves
// all, which spills at four columns (16,384 x 2,048 bf16: five taps 258 + 79 us,
// eight 272 + 92).  The arithmetic runs on pairs of columns.  Where sequences
// begin comes as one bit a row, which a CTA gathers for its rows before it starts;
// batches inside one sequence run without a branch, others replace the window by
// assignment where a sequence begins. p is computed again in the backward from x,
// which is there anyway.  dw and dbias are summed over a thread's run in
// registers, over a CTA in shared memory, and over the CTAs by a second launch in
// a fixed order.
#include <algorithm>
#include <type_traits>
#include "head.cuh"
#include "history.cuh"

namespace {
using namespace fbq;

constexpr int kThreads = 128;
constexpr int kMaxTaps = 8;
constexpr int64_t kSms = 148;

struct ConvArgs {
  int D, K, silu;
  const void *x, *dy, *init, *dfin;
  void *y, *dx, *fin, *dinit;
  int ldx, ldy, lddy, lddx;
  const float *w, *bias;
  float *part, *dw, *dbias;                // part [blocks, K + 1, D]
  Starts st;
  int cx, ry;                              // threads of a CTA along the columns, runs of rows
  int run;                                 // rows of a run, a multiple of 8
  int64_t blocks;                          // CTAs along the rows
  int ring;                                // where the rows on their way begin in shared memory
};

// Sequence of a row, -1: none, for one thread (few threads ask).
__device__ __forceinline__ int owner1(const Starts &st, int64_t row) {
  if (!st.p) return row >= 0 && row < st.rows ? 0 : -1;
  int lo = 0, hi = st.seqs + 1;
  while (lo < hi) {
    const int m = lo + ((hi - lo) >> 1);
    if (st[m] <= row) lo = m + 1;
    else hi = m;
  }
  return lo - 1 < st.seqs ? lo - 1 : -1;
}

// V elements as pairs (one element: with a zero).
template <typename T, int V> struct Pairs {
  static constexpr int P = (V + 1) / 2;
  static __device__ __forceinline__ void widen(const Vec<T, V> &e, F2 (&v)[P]) {
#pragma unroll
    for (int i = 0; i < P; ++i) v[i] = pack(to_f(e.e[2 * i]), 2 * i + 1 < V ? to_f(e.e[2 * i + 1 < V ? 2 * i + 1 : 0]) : 0.f);
  }
  static __device__ __forceinline__ Vec<T, V> narrow(const F2 (&v)[P]) {
    Vec<T, V> e;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const float2 f = unpack(v[i]);
      e.e[2 * i] = from_f<T>(f.x);
      if (2 * i + 1 < V) e.e[2 * i + 1 < V ? 2 * i + 1 : 0] = from_f<T>(f.y);
    }
    return e;
  }
};

// The beginnings of the rows from `from` on, a bit each, 32 * words of them.
__device__ __forceinline__ void fill_begins(const Starts &st, int64_t from, int words, uint32_t *bits) {
  for (int i = threadIdx.x; i < words; i += blockDim.x) bits[i] = 0;
  __syncthreads();
  const auto mark = [&](int64_t b) {
    if (b >= from && b < from + 32 * words) atomicOr(&bits[(b - from) >> 5], 1u << ((b - from) & 31));
  };
  if (!st.p) {
    if (threadIdx.x == 0) mark(0), mark(st.rows);
    __syncthreads();
    return;
  }
  for (int i = owner(st, from - 1) + 1 + threadIdx.x;; i += blockDim.x) {
    const int64_t b = i <= st.seqs ? st[i] : INT64_MAX;
    if (b < INT64_MAX) mark(b);
    if (!__syncthreads_and(b < from + 32 * words)) break;
  }
}

template <typename E> __device__ __forceinline__ void copy_async(E *to, const void *from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from), "n"(sizeof(E))
               : "memory");
}

// Rows of a batch: 8 single bf16 elements, which no asynchronous copy moves and
// only their number keeps memory busy with; else 4.
template <typename T, int V> constexpr int kRows = sizeof(T) * V < 4 ? 8 : 4;

// KT taps in registers; KT 2, 3, 4: exactly K, KT 8: the first 8 - K of them do
// not exist and are left out, not multiplied by zero.
template <typename T, int V, int KT, bool BWD> __global__ void __launch_bounds__(kThreads, BWD ? 4 : 6) k_conv(ConvArgs a) {
  using PV = Pairs<T, V>;
  using E = Vec<T, V>;
  constexpr int P = PV::P, H = KT - 1;                                     // pairs of columns; rows of history
  constexpr bool ASYNC = sizeof(E) >= 4;                                   // what an asynchronous copy moves
  constexpr int R = kRows<T, V>;                                           // rows at a time
  fb::pdl_enter();
  extern __shared__ __align__(16) unsigned char dyn[];
  const int64_t rows = a.st.rows;
  const int64_t block0 = (int64_t)blockIdx.y * a.ry * a.run;               // the CTA's first row
  const int words = (a.ry * a.run + 24 + 31) / 32;
  uint32_t *const bits = reinterpret_cast<uint32_t *>(dyn);                // rows from block0 - 8 on
  float *const sums = reinterpret_cast<float *>(dyn + (words * 4 + 15) / 16 * 16);
  fill_begins(a.st, block0 - 8, words, bits);

  const int c = threadIdx.x % a.cx, q = threadIdx.x / a.cx;
  const int col = (blockIdx.x * a.cx + c) * V;
  const int K = KT == 8 ? a.K : KT, skip = KT - K;
  const int64_t q0 = block0 + (int64_t)q * a.run;
  const int len = (int)max((int64_t)0, min((int64_t)a.run, rows - q0));    // rows of the run
  const bool active = q < a.ry && col < a.D && len > 0;
  F2 dw[BWD ? KT : 1][P], db[P];
#pragma unroll
  for (int p = 0; p < P; ++p) {
    db[p] = both(0.f);
    if constexpr (BWD)
#pragma unroll
      for (int k = 0; k < KT; ++k) dw[k][p] = both(0.f);
  }
  if (active) {
    // rows counted from q0: those of sequences, and those of the tensor
    const int first = (int)max((int64_t)-64, min(a.st[0] - q0, (int64_t)a.run + 64));
    const int last = (int)max((int64_t)-64, min(a.st[a.st.seqs] - q0, (int64_t)a.run + 64));
    const int all = (int)min(rows - q0, (int64_t)a.run + 64);
    F2 w[KT][P], bias[P];
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int c0 = col + 2 * p, c1 = 2 * p + 1 < V ? c0 + 1 : c0;
      bias[p] = a.bias ? pack(a.bias[c0], a.bias[c1]) : both(0.f);
#pragma unroll
      for (int k = 0; k < KT; ++k)
        w[k][p] = k >= skip ? pack(a.w[(int64_t)c0 * K + k - skip], a.w[(int64_t)c1 * K + k - skip]) : both(0.f);
    }
    const T *const px = static_cast<const T *>(a.x) + q0 * a.ldx + col;
    const T *const pdy = BWD ? static_cast<const T *>(a.dy) + q0 * a.lddy + col : nullptr;
    T *const py = static_cast<T *>(BWD ? a.dx : a.y) + q0 * (BWD ? a.lddx : a.ldy) + col;
    const int ldo = BWD ? a.lddx : a.ldy;
    // 16 beginnings, of the rows t - 8 .. t + 7
    const auto around = [&](int t) {
      const int o = q * a.run + t;                                         // bit of row t - 8
      return (bits[o >> 5] >> (o & 31) | ((o & 31) > 16 ? bits[(o >> 5) + 1] << (32 - (o & 31)) : 0u)) & 0xffffu;
    };
    // The m-th oldest of the K - 1 inputs in front of sequence s.
    const auto older = [&](int s, int m, F2 (&v)[P]) {
      E e;
#pragma unroll
      for (int i = 0; i < V; ++i)
        e.e[i] = s >= 0 && m >= 0 ? static_cast<const T *>(a.init)[((int64_t)s * (K - 1) + m) * a.D + col + i] : from_f<T>(0.f);
      PV::widen(e, v);
    };

    F2 win[H + R][P];                                                      // the last H inputs, then R new ones
    {
      // in front of the run: its own sequence's inputs as far as they go, then those of init
      const unsigned m = around(0);
      int b = -H;
      bool cut = false;
#pragma unroll
      for (int j = H; j >= 1; --j)
        if (m >> (8 - j) & 1u) b = -j, cut = true;
      if (!cut && q0 < H) b = (int)-q0, cut = true;
      const int s = cut && a.init ? owner1(a.st, q0 + b) : -1;
#pragma unroll
      for (int i = 0; i < H; ++i) {
        const int t = i - H;
        if (t >= b) {
          E e = *reinterpret_cast<const E *>(px + (int64_t)t * a.ldx);
          PV::widen(e, win[i]);
        } else {
          older(s, K - 1 + t - b, win[i]);
        }
      }
    }
    F2 dp[BWD ? H + R : 1][P];
    if constexpr (BWD) {
#pragma unroll
      for (int i = 0; i < H; ++i)
#pragma unroll
        for (int p = 0; p < P; ++p) dp[i][p] = both(0.f);
    }
    // Backward, a dx row is complete K - 1 rows later: the walk goes on behind the run.
    const int end = BWD ? len + H : len, have = min(end, all);
    // Two batches of R rows are on their way while one is in work, each thread's into places of its own.
    E *const ring = reinterpret_cast<E *>(dyn + a.ring) + threadIdx.x;     // [3 batches, R rows, x and dy][thread]
    const auto fetch = [&](int t0, int b) {
      if constexpr (ASYNC) {
        const T *x = px + (int64_t)t0 * a.ldx, *y = BWD ? pdy + (int64_t)t0 * a.lddy : nullptr;
        E *to = ring + b * (R * (BWD ? 2 : 1) * kThreads);
#pragma unroll
        for (int i = 0; i < R; ++i)
          if (t0 + i < have) {
            copy_async(to + i * kThreads, x + (int64_t)i * a.ldx);
            if constexpr (BWD) copy_async(to + (R + i) * kThreads, y + (int64_t)i * a.lddy);
          }
        asm volatile("cp.async.commit_group;" ::: "memory");
      }
    };
    fetch(0, 0);
    fetch(R, 1);
    int batch = 0;
    for (int t0 = 0; t0 < end; t0 += R) {
      const unsigned m = around(t0);
      unsigned live = (1u << R) - 1u;
      if (t0 < first || t0 + R > last || t0 + R > have) {
#pragma unroll
        for (int i = 0; i < R; ++i)
          if (t0 + i < first || t0 + i >= last || t0 + i >= have) live &= ~(1u << i);
      }
      fetch(t0 + 2 * R, batch == 0 ? 2 : batch - 1);
      if constexpr (ASYNC) asm volatile("cp.async.wait_group 2;" ::: "memory");
      const E *const here = ring + batch * (R * (BWD ? 2 : 1) * kThreads);
      batch = batch == 2 ? 0 : batch + 1;
      E rx[ASYNC ? 1 : R], ry[BWD && !ASYNC ? R : 1];
      if constexpr (!ASYNC) {
#pragma unroll
        for (int i = 0; i < R; ++i)
          if (t0 + i < have) {
            rx[i] = *reinterpret_cast<const E *>(px + (int64_t)(t0 + i) * a.ldx);
            if constexpr (BWD) ry[i] = *reinterpret_cast<const E *>(pdy + (int64_t)(t0 + i) * a.lddy);
          }
      }
      // PLAIN: rows of one sequence, inside the run
      const auto work = [&](auto plain) {
        constexpr bool PLAIN = decltype(plain)::value;
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const int t = t0 + i;
        PV::widen(ASYNC ? here[i * kThreads] : rx[ASYNC ? 0 : i], win[H + i]);
        F2 g[P];
        if constexpr (BWD) PV::widen(ASYNC ? here[(R + i) * kThreads] : ry[ASYNC ? 0 : i], g);
        if (!PLAIN && (m >> (8 + i) & 1u)) {                                          // a sequence begins: what was before it
          const int s = a.init ? owner1(a.st, q0 + t) : -1;
#pragma unroll
          for (int k = 0; k < H; ++k) older(s, k - skip, win[i + k]);
        }
        F2 z[P], sg[P], rest[P];
#pragma unroll
        for (int p = 0; p < P; ++p) {
          z[p] = bias[p];
#pragma unroll
          for (int k = 0; k < KT; ++k)
            if (k >= skip) z[p] = fma2(w[k][p], win[i + k][p], z[p]);
          if (a.silu) sg[p] = sigmoid2<T>(z[p], rest[p]);
        }
        if constexpr (!BWD) {
          if (PLAIN || t < len) {
            if (a.silu)
#pragma unroll
              for (int p = 0; p < P; ++p) z[p] = mul2(z[p], sg[p]);
            if (!PLAIN && !(live >> i & 1u))
#pragma unroll
              for (int p = 0; p < P; ++p) z[p] = both(0.f);
            *reinterpret_cast<E *>(py + (int64_t)t * ldo) = PV::narrow(z);
          }
        } else {
          if (PLAIN || (live >> i & 1u)) {
            if (a.silu)
#pragma unroll
              for (int p = 0; p < P; ++p) g[p] = mul2(g[p], silu_slope2<T>(z[p], sg[p], rest[p]));
            if (PLAIN || t < len)
#pragma unroll
              for (int p = 0; p < P; ++p) {
                db[p] = add2(db[p], g[p]);
#pragma unroll
                for (int k = 0; k < KT; ++k)
                  if (k >= skip) dw[k][p] = fma2(g[p], win[i + k][p], dw[k][p]);
              }
          } else {
#pragma unroll
            for (int p = 0; p < P; ++p) g[p] = both(0.f);
          }
#pragma unroll
          for (int p = 0; p < P; ++p) dp[H + i][p] = g[p];
          // the row whose last dp this was
          const int r = t - H;
          if (PLAIN || (r >= 0 && r < len)) {
            const unsigned ends = PLAIN ? 0u : m >> (8 + i - H + 1);       // bit j - 1: row r + j begins another sequence
            F2 o[P];
#pragma unroll
            for (int p = 0; p < P; ++p) o[p] = mul2(w[KT - 1][p], dp[i][p]);
#pragma unroll
            for (int j = 1; j < KT; ++j)
              if (KT - 1 - j >= skip && (PLAIN || !(ends & ((1u << j) - 1u))))
#pragma unroll
                for (int p = 0; p < P; ++p) o[p] = fma2(w[KT - 1 - j][p], dp[i + j][p], o[p]);
            if (!PLAIN && a.dfin && (ends & ((1u << (K - 1)) - 1u))) {               // one of the last K - 1 inputs
              const int s = owner1(a.st, q0 + r), gap = __ffs(ends);
              if (s >= 0) {
                E e;
#pragma unroll
                for (int v = 0; v < V; ++v)
                  e.e[v] = static_cast<const T *>(a.dfin)[((int64_t)s * (K - 1) + K - 1 - gap) * a.D + col + v];
                F2 f[P];
                PV::widen(e, f);
#pragma unroll
                for (int p = 0; p < P; ++p) o[p] = add2(o[p], f[p]);
              }
            }
            *reinterpret_cast<E *>(py + (int64_t)r * ldo) = PV::narrow(o);
          }
        }
      }
      };
      if (live == (1u << R) - 1u && !(m >> (8 - H + 1) & ((1u << (R + H - 1)) - 1u)) && t0 >= (BWD ? H : 0) && t0 + R <= len) work(std::true_type{});
      else work(std::false_type{});
#pragma unroll
      for (int i = 0; i < H; ++i)
#pragma unroll
        for (int p = 0; p < P; ++p) {
          win[i][p] = win[i + R][p];
          if constexpr (BWD) dp[i][p] = dp[i + R][p];
        }
    }
  }
  if constexpr (BWD) {
    // the CTA's sums: the runs add up in order
    const int width = a.cx * V;
#pragma unroll
    for (int k = 0; k <= KT; ++k) {
      if (k < skip) continue;
      if (q < a.ry && col < a.D)
#pragma unroll
        for (int p = 0; p < P; ++p) {
          const float2 f = unpack(k < KT ? dw[k < KT ? k : 0][p] : db[p]);
          sums[q * width + c * V + 2 * p] = f.x;
          if (2 * p + 1 < V) sums[q * width + c * V + 2 * p + 1] = f.y;
        }
      __syncthreads();
      for (int i = threadIdx.x; i < width; i += kThreads) {
        const int d = blockIdx.x * width + i;
        if (d < a.D) {
          float x = 0.f;
          for (int j = 0; j < a.ry; ++j) x += sums[j * width + i];
          if (a.blocks > 1) a.part[((int64_t)blockIdx.y * (K + 1) + k - skip) * a.D + d] = x;
          else if (k < KT) a.dw[(int64_t)d * K + k - skip] = x;
          else a.dbias[d] = x;
        }
      }
      __syncthreads();
    }
  }
}

// Adds the CTAs' sums in a fixed order: 8 columns a CTA, 32 threads a column.
__global__ void __launch_bounds__(256) k_conv_sums(ConvArgs a) {
  fb::pdl_enter();
  __shared__ float part[8][8];
  const int64_t n = (int64_t)(a.K + 1) * a.D, i = (int64_t)blockIdx.x * 8 + threadIdx.x % 8;
  float v = 0.f;
  if (i < n) {
#pragma unroll 8
    for (int64_t b = threadIdx.x / 8; b < a.blocks; b += 32) v += a.part[b * n + i];
  }
  v += __shfl_xor_sync(0xffffffffu, v, 8);
  v += __shfl_xor_sync(0xffffffffu, v, 16);
  if (threadIdx.x % 32 < 8) part[threadIdx.x / 32][threadIdx.x % 8] = v;
  __syncthreads();
  if (threadIdx.x >= 8 || i >= n) return;
  v = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) v += part[j][threadIdx.x];
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
    if (p >= 0) v = static_cast<const T *>(a.x)[(b + p) * (int64_t)a.ldx + d];
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
      x[K - 1 + i] = to_f(static_cast<const T *>(a.x)[(b + i) * (int64_t)a.ldx + d]);
      float p = a.bias ? a.bias[d] : 0.f, dp = to_f(static_cast<const T *>(a.dy)[(b + i) * (int64_t)a.lddy + d]);
      for (int k = 0; k < K; ++k) p = fmaf(w[k], x[i + k], p);
      if (a.silu) {
        float rest;
        const float sg = sigmoid<T>(p, rest);
        dp *= sg * fmaf(p, rest, 1.f);
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
  if (std::max(std::max(s->ldx, s->ldy), std::max(s->lddy, s->lddx)) > (1 << 28))
    return fb::set_error(FB_ERR_UNSUPPORTED, "short_conv: leading dimension beyond what the kernels index");
  if (!s->w || (s->rows && !s->x)) return bad("missing operand");
  if (s->rows > 1 && s->ldx < s->D) return bad("leading dimension below the width");
  if (!backward && s->rows && (!s->y || (s->rows > 1 && s->ldy < s->D))) return bad("missing or overlapping output");
  if (backward && s->rows && (!s->dy || !s->dx || (s->rows > 1 && (s->lddy < s->D || s->lddx < s->D))))
    return bad("missing or overlapping operand of the backward pass");
  if (backward && (!s->dw || !s->dbias)) return bad("missing gradient");
  if (backward && s->dinit && !s->init) return bad("dinit without init");
  const uintptr_t es = s->type == FB_F32 ? 4 : 2;
  if (!aligned(es, s->x, s->init) || !(backward ? aligned(es, s->dy, s->dfinal, s->dx, s->dinit) : aligned(es, s->y, s->final)))
    return bad("rows that are not aligned to their elements");
  if (!aligned(4, s->w, s->bias) || (backward && !aligned(4, s->dw, s->dbias)) || !aligned(s->starts_type == FB_I64 ? 8 : 4, s->starts))
    return bad("parameters or starts that are not aligned to their elements");
  a = ConvArgs{};
  a.D = s->D, a.K = s->K, a.silu = s->act == FB_ACT_SILU;
  a.x = s->x, a.ldx = (int)s->ldx, a.dy = s->dy, a.lddy = (int)s->lddy, a.init = s->K > 1 ? s->init : nullptr;
  a.dfin = s->K > 1 ? s->dfinal : nullptr, a.fin = s->K > 1 ? s->final : nullptr, a.dinit = s->K > 1 ? s->dinit : nullptr;
  a.y = s->y, a.ldy = (int)s->ldy, a.dx = s->dx, a.lddx = (int)s->lddx, a.w = s->w, a.bias = s->bias, a.dw = s->dw, a.dbias = s->dbias;
  a.st = Starts{s->starts, s->starts_type == FB_I64, (int)s->seqs, s->rows};
  return FB_OK;
}

// Columns a thread moves at once: as many as bases, pitches and the width allow,
// up to 4 where that leaves 8 warps an SM (runs of 32 rows), else 2: a lone warp
// issues an instruction every four cycles (12,000 x 200 fp32, both passes: 2
// columns 35 us, 4 columns 43, one 40).  8 columns of bf16 take more registers
// than the wider accesses give back (forward of 32,768 x 2,048: 75 us, with 4
// columns 63).
int vector_of(const fb_short_conv *s, bool backward) {
  const int es = s->type == FB_F32 ? 4 : 2;
  const void *p[2] = {backward ? s->dy : s->y, backward ? s->dx : nullptr};
  const int64_t ld[2] = {backward ? s->lddy : s->ldy, backward ? s->lddx : 0};
  uint64_t bits = (uint64_t)(uintptr_t)s->x / es | (uint64_t)s->D;
  if (s->rows > 1) bits |= (uint64_t)s->ldx;
  for (int i = 0; i < 2; ++i)
    if (p[i]) {
      bits |= (uint64_t)(uintptr_t)p[i] / es;
      if (s->rows > 1) bits |= (uint64_t)ld[i];
    }
  const bool many = s->rows / 32 * (s->D / 128) >= kSms * 8;
  return bits % 4 == 0 && many ? 4 : (bits % 2 == 0 ? 2 : 1);
}

// Columns of a CTA, runs side by side, rows of a run: long runs load few rows
// twice, but the SMs want their CTAs each.
void plan(ConvArgs &a, int V, bool backward) {
  const int groups = (a.D + V - 1) / V;
  a.cx = std::min(groups, kThreads);
  a.ry = kThreads / a.cx;
  const int64_t across = (groups + a.cx - 1) / a.cx;
  const int64_t want = std::max<int64_t>(1, kSms * (backward ? 4 : 6) / across);
  int64_t run = (a.st.rows + want * a.ry - 1) / (want * a.ry);
  run = std::min<int64_t>(std::max<int64_t>((run + 7) / 8 * 8, 16), 256);
  while (run * a.ry > 8192 && run > 8) run -= 8;
  a.run = (int)run;
  a.blocks = (a.st.rows + a.run * (int64_t)a.ry - 1) / (a.run * (int64_t)a.ry);
  // CTAs along the rows are a grid's y
  while (a.blocks > 65535) a.run *= 2, a.blocks = (a.st.rows + a.run * (int64_t)a.ry - 1) / (a.run * (int64_t)a.ry);
}

template <typename T, int V, int KT, bool BWD> int launch_main(ConvArgs &a, cudaStream_t st) {
  const int width = a.cx * V;
  a.ring = ((a.ry * a.run + 24 + 31) / 32 * 4 + 15) / 16 * 16 + (BWD ? (a.ry * width * 4 + 15) / 16 * 16 : 0);
  const size_t ring = sizeof(T) * V < 4 ? 0 : (size_t)3 * kRows<T, V> * (BWD ? 2 : 1) * kThreads * V * sizeof(T);
  const size_t smem = a.ring + ring;
  if (smem > 96 * 1024) return fb::set_error(FB_ERR_UNSUPPORTED, "short_conv: too many rows");
  if (smem > 48 * 1024)
    FB_TRY_CUDA(cudaFuncSetAttribute(k_conv<T, V, KT, BWD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  const dim3 grid((unsigned)((a.D + width - 1) / width), (unsigned)a.blocks);
  FB_TRY_CUDA(fb::launch(k_conv<T, V, KT, BWD>, grid, kThreads, smem, st, a));
  return FB_OK;
}

template <typename T, int V, bool BWD> int launch_k(ConvArgs &a, cudaStream_t st) {
  switch (a.K) {
    case 2: return launch_main<T, V, 2, BWD>(a, st);
    case 3: return launch_main<T, V, 3, BWD>(a, st);
    case 4: return launch_main<T, V, 4, BWD>(a, st);
    default: return launch_main<T, V, 8, BWD>(a, st);
  }
}

template <typename T, bool BWD> int launch_v(ConvArgs &a, int V, cudaStream_t st) {
  return V == 4 ? launch_k<T, 4, BWD>(a, st) : V == 2 ? launch_k<T, 2, BWD>(a, st) : launch_k<T, 1, BWD>(a, st);
}

unsigned some_blocks(int64_t n) { return (unsigned)std::min<int64_t>((n + 255) / 256, kSms * 8); }

template <typename T> int run_conv(const fb_short_conv *s, ConvArgs &a, bool backward, void *ws, size_t ws_bytes, cudaStream_t st) {
  const int64_t state = (int64_t)a.st.seqs * (a.K - 1) * a.D;
  if (s->rows) {
    const int V = vector_of(s, backward);
    plan(a, V, backward);
    if (backward && a.blocks > 1) {
      const size_t need = (size_t)a.blocks * (a.K + 1) * a.D * sizeof(float);
      FBH_TRY(fbh::check_ws(ws, "short_conv"));
      if (ws_bytes < need) return fb::set_error(FB_ERR_ARG, "short_conv: workspace too small");
      a.part = static_cast<float *>(ws);
    }
    FBH_TRY((backward ? launch_v<T, true>(a, V, st) : launch_v<T, false>(a, V, st)));
    if (backward && a.blocks > 1) FB_TRY_CUDA(fb::launch(k_conv_sums, dim3((unsigned)(((a.K + 1) * (int64_t)a.D + 7) / 8)), 256, 0, st, a));
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
