// See few_rows.cuh.
//
// A warp takes R = 4 weight rows at a time and MT (1, 2, 4, 8) rows of x:
// lane l multiplies elements l V .. l V + V - 1 of every 32 V, V of them per
// load (16 bytes where the weights' base, pitch and width allow), against x
// kept as fp32 in shared memory, and each x element read there serves R rows.
// The R MT sums are then reduced over the lanes by halving: each exchange
// keeps half of the values, so 32 sums take 31 shuffles, and lane i ends with
// sum i / (32 / (R MT)).  Where the weight has too few rows to fill the GPU,
// KS warps share a row's elements and their sums meet in shared memory.
// Gate and up weights are taken in pairs of rows (kGlu: the block's hidden row;
// kGateUp: both sums, for the backward).
//
// The gated block's second product asks the L2 for its first rows before it
// waits for the first product, which they do not come from.  (Asking for every
// turn's rows ahead made the single-pass kernels 10% slower.)
#include "few_rows.cuh"
#include <cuda_bf16.h>
#include <algorithm>
#include <cmath>
#include "act.cuh"

namespace {

using namespace fbh;

constexpr int R = 4;
constexpr int kWarps = 16;
constexpr int kMaxSmem = 200 * 1024;

enum : int { kGlu = 0, kPlain = 1, kLogits = 2, kGateUp = 3 };
template <int MODE> __host__ __device__ constexpr bool two() { return MODE == kGlu || MODE == kGateUp; }   // two weights

struct Args {
  const void *x;
  int64_t ldx;
  int x_f32;                                  // x is fp32 (else of the weights' type)
  const void *w, *w2;
  int64_t ldw, ldw2;
  int n, K;
  int64_t rows;                               // weight rows (kGlu: of each)
  int ks;
  int act;
  void *out;
  int64_t ldo;
  float2 *part;
  int out_f32;                                // kPlain: out is fp32 (else of the weights' type)
};

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

// V elements of a weight row as floats; zeros when !in.  Volatile: a load must
// not be moved ahead of the wait for the kernel before, which may have written
// the weights.
template <typename T, int V> struct Raw;
template <> struct Raw<__nv_bfloat16, 8> {
  uint4 v;
  __device__ __forceinline__ void load(const __nv_bfloat16 *p, bool in) {
    v = make_uint4(0, 0, 0, 0);
    if (in)                                   // read once: past the L1
      asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0, %1, %2, %3}, [%4];"
          : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
          : "l"(p));
  }
  __device__ __forceinline__ float get(int e) const {
    const uint32_t w = e < 2 ? v.x : (e < 4 ? v.y : (e < 6 ? v.z : v.w));
    return __uint_as_float(e & 1 ? w & 0xFFFF0000u : w << 16);
  }
};
template <> struct Raw<float, 4> {
  float4 v;
  __device__ __forceinline__ void load(const float *p, bool in) {
    v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (in)
      asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.f32 {%0, %1, %2, %3}, [%4];"
          : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
          : "l"(p));
  }
  __device__ __forceinline__ float get(int e) const { return e == 0 ? v.x : (e == 1 ? v.y : (e == 2 ? v.z : v.w)); }
};
template <typename T> struct Raw<T, 1> {
  T v;
  __device__ __forceinline__ void load(const T *p, bool in) { v = in ? *p : T(0.f); }
  __device__ __forceinline__ float get(int) const { return to_f(v); }
};

template <int V> __device__ __forceinline__ void load_x(float (&o)[V], const float *p) {
  if constexpr (V >= 4) {
#pragma unroll
    for (int e = 0; e < V; e += 4) *reinterpret_cast<float4 *>(o + e) = *reinterpret_cast<const float4 *>(p + e);
  } else {
    o[0] = p[0];
  }
}

// NV sums over 32 lanes; lane i returns the total of v[i / (32 / NV)].
template <int NV> __device__ __forceinline__ float reduce(float (&v)[NV], int lane) {
  int n = NV;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    if (n > 1) {
      n >>= 1;
#pragma unroll
      for (int i = 0; i < NV / 2; ++i)
        if (i < n) {
          const bool up = (lane & o) != 0;
          const float keep = up ? v[i + n] : v[i], send = up ? v[i] : v[i + n];
          v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
        }
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
    }
  }
  return v[0];
}

__device__ __forceinline__ float act1(int act, float g) {
  if (act == fbact::kSilu) return fbact::act_exact<fbact::kSilu>(g).x;
  if (act == fbact::kGelu) return fbact::act_exact<fbact::kGelu>(g).x;
  return fbact::act_exact<fbact::kRelu>(g).x;
}

template <typename T> __device__ __forceinline__ void put(const Args &a, int64_t at, float v) {
  if (sizeof(T) == 2 && !a.out_f32) static_cast<__nv_bfloat16 *>(a.out)[at] = __float2bfloat16_rn(v);
  else static_cast<float *>(a.out)[at] = v;
}

// x's pitch in shared memory: whole 32-lane steps, zeros past K.
template <int V> __host__ __device__ constexpr int x_pitch(int K) { return (K + 32 * V - 1) / (32 * V) * (32 * V); }

template <typename T, int V, int MT, int MODE>
__global__ void __launch_bounds__(kWarps * 32, MT == 8 ? 1 : 2) k_few_rows(const Args a) {
  constexpr int NV = R * MT;
  extern __shared__ __align__(16) float xs[];
  __shared__ float red[kWarps][NV];
  __shared__ float2 ms[kWarps][NV];
  const int Kp = x_pitch<V>(a.K);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int part = warp % a.ks, slot = warp / a.ks, slots = kWarps / a.ks;
  const int steps = Kp / (32 * V), per = (steps + a.ks - 1) / a.ks;
  const int s0 = part * per, s1 = min(steps, s0 + per);
  constexpr int kRowsPer = two<MODE>() ? R / 2 : R;       // weight rows (of each matrix) a warp takes at a time
  const int64_t groups = (a.rows + kRowsPer - 1) / kRowsPer;
  // asks the L2 for this warp's part of the rows of group g
  auto ahead = [&](int64_t g) {
    if (V == 1 || lane >= R) return;
    const int64_t row = (g + slot) * kRowsPer + (two<MODE>() ? lane / 2 : lane);
    const int k0 = s0 * 32 * V, k1 = min(a.K, s1 * 32 * V);
    if (row >= a.rows || k1 <= k0) return;
    const T *p = (two<MODE>() && (lane & 1)) ? static_cast<const T *>(a.w2) + row * a.ldw2
                                              : static_cast<const T *>(a.w) + row * a.ldw;
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p + k0), "r"((uint32_t)((k1 - k0) * sizeof(T)))
                 : "memory");
  };
  const int64_t turn = (int64_t)gridDim.x * slots;
  if (MODE == kPlain) ahead((int64_t)blockIdx.x * slots);
  fb::pdl_enter();
  for (int i = threadIdx.x; i < MT * Kp; i += blockDim.x) {
    const int m = i / Kp, k = i - m * Kp;
    float v = 0.f;
    if (m < a.n && k < a.K)
      v = a.x_f32 ? static_cast<const float *>(a.x)[m * a.ldx + k] : to_f(static_cast<const T *>(a.x)[m * a.ldx + k]);
    xs[i] = v;
  }
  __syncthreads();
  float mx = -INFINITY, sum = 0.f;            // kLogits: of this lane's (row of R, m) stream
  for (int64_t g0 = (int64_t)blockIdx.x * slots; g0 < groups; g0 += turn) {
    const int64_t row0 = (g0 + slot) * kRowsPer;
    const T *p[R];
    bool in[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = two<MODE>() ? row0 + r / 2 : row0 + r;
      in[r] = row < a.rows;
      const int64_t q = in[r] ? row : 0;
      p[r] = (two<MODE>() && (r & 1)) ? static_cast<const T *>(a.w2) + q * a.ldw2
                                       : static_cast<const T *>(a.w) + q * a.ldw;
    }
    float acc[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) acc[i] = 0.f;
#pragma unroll 2
    for (int s = s0; s < s1; ++s) {
      const int k = (s * 32 + lane) * V;
      Raw<T, V> w[R];
#pragma unroll
      for (int r = 0; r < R; ++r) w[r].load(p[r] + k, in[r] && k < a.K);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        float x[V];
        load_x<V>(x, xs + m * Kp + k);
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int e = 0; e < V; ++e) acc[r * MT + m] = fmaf(w[r].get(e), x[e], acc[r * MT + m]);
      }
    }
    const float v = reduce<NV>(acc, lane);
    const int idx = lane / (32 / NV), m = idx % MT;
    if (MODE == kLogits) {                    // ks == 1: the warp has the whole logit
      const int64_t row = row0 + idx / MT;
      if (row < a.rows && lane % (32 / NV) == 0 && m < a.n) {
        const float l = v * 1.44269504088896340736f, nm = fmaxf(mx, l), base = nm == -INFINITY ? 0.f : nm;
        sum = sum * exp2f(mx - base) + exp2f(l - base);
        mx = nm;
      }
      continue;
    }
    if (a.ks > 1 || two<MODE>()) {
      __syncthreads();                        // the turn before has been read
      if (lane % (32 / NV) == 0) red[warp][idx] = v;
      __syncthreads();
    }
    if (MODE == kPlain && a.ks == 1) {
      const int64_t row = row0 + idx / MT;
      if (lane % (32 / NV) == 0 && row < a.rows && m < a.n) {
        put<T>(a, m * a.ldo + row, v);
      }
      continue;
    }
    // one thread per result: sums of the KS warps, in order
    constexpr int kOut = two<MODE>() ? NV / 2 : NV;
    for (int t = threadIdx.x; t < slots * kOut; t += blockDim.x) {
      const int sl = t / kOut, i = t - sl * kOut, r = i / MT, mm = i - r * MT;
      const int64_t row = (g0 + sl) * kRowsPer + r;
      if (row >= a.rows || mm >= a.n) continue;
      if (two<MODE>()) {
        float g = 0.f, u = 0.f;
        for (int q = 0; q < a.ks; ++q) {
          g += red[sl * a.ks + q][(2 * r) * MT + mm];
          u += red[sl * a.ks + q][(2 * r + 1) * MT + mm];
        }
        float *o = static_cast<float *>(a.out) + mm * a.ldo + row;
        if (MODE == kGateUp) o[0] = g, o[a.rows] = u;
        else *o = act1(a.act, g) * u;
      } else {
        float s = 0.f;
        for (int q = 0; q < a.ks; ++q) s += red[sl * a.ks + q][i];
        put<T>(a, mm * a.ldo + row, s);
      }
    }
  }
  if (MODE == kLogits) {
    const int idx = lane / (32 / NV);
    if (lane % (32 / NV) == 0) ms[warp][idx] = make_float2(mx, sum);
    __syncthreads();
    if (threadIdx.x < (unsigned)min(MT, a.n)) {
      const int m = threadIdx.x;
      float bm = -INFINITY;
      for (int w = 0; w < kWarps; ++w)
        for (int r = 0; r < R; ++r) bm = fmaxf(bm, ms[w][r * MT + m].x);
      const float base = bm == -INFINITY ? 0.f : bm;
      float s = 0.f;
      for (int w = 0; w < kWarps; ++w)
        for (int r = 0; r < R; ++r) s += ms[w][r * MT + m].y * exp2f(ms[w][r * MT + m].x - base);
      a.part[(int64_t)m * gridDim.x + blockIdx.x] = make_float2(bm, s);
    }
  }
}

int sms() {
  static int n[64] = {0};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!n[dev & 63]) {
    int v = 0;
    cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev);
    n[dev & 63] = v > 0 ? v : 148;
  }
  return n[dev & 63];
}

template <typename T, int V, int MT, int MODE> int go(const Args &a, unsigned grid, cudaStream_t st) {
  constexpr auto k = k_few_rows<T, V, MT, MODE>;
  const size_t smem = sizeof(float) * MT * x_pitch<V>(a.K);
  if (smem > 40 * 1024) {                     // the 48 KB that need no asking include the static arrays
    static bool set[64] = {false};
    int dev = 0;
    cudaGetDevice(&dev);
    if (!set[dev & 63]) {
      FB_TRY_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem));
      set[dev & 63] = true;
    }
  }
  FB_TRY_CUDA(fb::launch(k, grid, kWarps * 32, smem, st, a));
  FB_LAUNCHED("k_few_rows");
  return FB_OK;
}
template <typename T, int V, int MODE> int by_rows(const Args &a, unsigned grid, cudaStream_t st) {
  if (a.n == 1) return go<T, V, 1, MODE>(a, grid, st);
  if (a.n == 2) return go<T, V, 2, MODE>(a, grid, st);
  if constexpr (MODE != kGateUp || sizeof(T) == 4) {   // bf16 backward: at most 2 rows
    if (a.n <= 4) return go<T, V, 4, MODE>(a, grid, st);
    return go<T, V, 8, MODE>(a, grid, st);
  }
  return fb::set_error(FB_ERR_ARG, "few rows: more rows than this path takes");
}
template <int MODE> int run(int type, Args a, cudaStream_t st) {
  const int es = elem(type), v = 16 / es;
  uintptr_t m = reinterpret_cast<uintptr_t>(a.w) | (uintptr_t)(a.ldw * es);
  if (two<MODE>()) m |= reinterpret_cast<uintptr_t>(a.w2) | (uintptr_t)(a.ldw2 * es);
  const bool wide = (m & 15) == 0 && a.K % v == 0;
  // warps sharing a row until every SM has two CTAs, while each keeps two steps of the row
  const int64_t per = two<MODE>() ? R / 2 : R, groups = (a.rows + per - 1) / per;
  const int steps = (a.K + 32 * (wide ? v : 1) - 1) / (32 * (wide ? v : 1));
  a.ks = 1;
  if (MODE != kLogits)
    while (a.ks < kWarps && groups * a.ks * 2 <= 2ll * sms() * kWarps && steps >= 4 * a.ks) a.ks *= 2;
  const int64_t ctas = (groups * a.ks + kWarps - 1) / kWarps;
  const unsigned grid = MODE == kLogits ? (unsigned)few_rows_parts() : (unsigned)std::min<int64_t>(ctas, 2 * sms());
  if (type == FB_F32) return wide ? by_rows<float, 4, MODE>(a, grid, st) : by_rows<float, 1, MODE>(a, grid, st);
  return wide ? by_rows<__nv_bfloat16, 8, MODE>(a, grid, st) : by_rows<__nv_bfloat16, 1, MODE>(a, grid, st);
}

}  // namespace

namespace fbh {

bool few_rows_ok(int type, bool bwd, int64_t n, int64_t K, int64_t weight_elements) {
  const int64_t most = type == FB_F32 ? 8 : (weight_elements > (1 << 20) ? 2 : (bwd ? 0 : 8));
  const int64_t mt = n == 1 ? 1 : (n == 2 ? 2 : (n <= 4 ? 4 : 8));
  return n >= 1 && n <= most && mt * round_up(K, 256) * (int64_t)sizeof(float) <= kMaxSmem;
}

int few_rows_glu(Call &c, int type, int act, const Mat &x, int64_t n, int D, const Mat &wg, const Mat &wu, int F,
                 float *h) {
  Args a{x.p, x.ld, type == FB_F32, wg.p, wu.p, wg.ld, wu.ld, (int)n, D, F, 1, act, h, F, nullptr, 1};
  return c.dry ? FB_OK : run<kGlu>(type, a, c.stream);
}

int few_rows_product(Call &c, int type, const float *x, int64_t n, int K, const Mat &w, int N, void *out, int64_t ldo) {
  Args a{x, K, 1, w.p, nullptr, w.ld, 0, (int)n, K, N, 1, 0, out, ldo, nullptr, type == FB_F32};
  return c.dry ? FB_OK : run<kPlain>(type, a, c.stream);
}

int few_rows_parts() { return 2 * sms(); }

int few_rows_lse(Call &c, int type, const Mat &h, int64_t n, int D, const Mat &w, int64_t V, float2 *part) {
  Args a{h.p, h.ld, type == FB_F32, w.p, nullptr, w.ld, 0, (int)n, D, V, 1, 0, nullptr, 0, part, 0};
  return c.dry ? FB_OK : run<kLogits>(type, a, c.stream);
}

int few_rows_gate_up(Call &c, int type, const Mat &x, int64_t n, int D, const Mat &wg, const Mat &wu, int F, float *gu) {
  Args a{x.p, x.ld, type == FB_F32, wg.p, wu.p, wg.ld, wu.ld, (int)n, D, F, 1, 0, gu, 2 * F, nullptr, 1};
  return c.dry ? FB_OK : run<kGateUp>(type, a, c.stream);
}

int few_rows_logits(Call &c, int type, const Mat &h, int64_t n, int D, const Mat &w, int64_t V, float *l) {
  Args a{h.p, h.ld, type == FB_F32, w.p, nullptr, w.ld, 0, (int)n, D, V, 1, 0, l, V, nullptr, 1};
  return c.dry ? FB_OK : run<kPlain>(type, a, c.stream);
}

}  // namespace fbh
