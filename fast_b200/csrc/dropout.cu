// Dropout from a counter, with the residual sum behind it:
//
//   y = res + keep x / (1 - p),  keep[r, c] = (word c % 4 of Philox4x32-10(counter (c / 4, r, offset), key seed)) / 2^32 >= p
//
// decided on the word's upper 24 bits, as everywhere in the framework.  Nothing
// is stored: the backward, keep dy / (1 - p), draws the same numbers again.
// Bound by memory (x, res, y) once the generator is lean: a thread keeps its
// group of four columns and goes down the rows, so nothing is divided; the ten
// rounds' keys come with the launch; the comparison is one of whole numbers
// (16,384 x 4,096 bf16 with a residual: 107 us with an index divided for each
// group and the words converted to fractions).  One row at a time and
// many warps: with four rows loaded ahead the registers leave too few (95 us
// against 89).
#include <algorithm>
#include <cmath>
#include "history.cuh"
#include "runtime.cuh"

namespace {
using namespace fbq;

struct DropArgs {
  const void *x, *res;
  void *y;
  int64_t ldx, ldr, ldy, rows;
  int D, quads;                            // groups of four columns
  int cx, ry;                              // groups, rows side by side in a CTA
  uint32_t from;                           // words from here on keep
  float scale;
  uint32_t key[10][2];                     // the rounds' keys
  uint64_t offset;
  const int64_t *offset_dev;
};

// Philox4x32-10 (fb::philox4x32_10) with the keys of the rounds at hand.
__device__ __forceinline__ fb::Philox4 draw(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, const uint32_t (&key)[10][2]) {
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = (uint64_t)0xD2511F53u * c0, p1 = (uint64_t)0xCD9E8D57u * c2;
    c0 = (uint32_t)(p1 >> 32) ^ c1 ^ key[r][0];
    c2 = (uint32_t)(p0 >> 32) ^ c3 ^ key[r][1];
    c1 = (uint32_t)p1, c3 = (uint32_t)p0;
  }
  return fb::Philox4{{c0, c1, c2, c3}};
}

constexpr int kThreads = 256;

// Q groups of four columns a thread.  VEC: they are moved at once (D is a multiple
// of 4 Q, rows aligned to them).
template <typename T, int Q, bool VEC, bool RES>
__global__ void __launch_bounds__(kThreads, Q > 1 ? 6 : 8) k_dropout(const __grid_constant__ DropArgs a) {
  fb::pdl_enter();
  using E = Vec<T, 4 * Q>;
  const uint64_t off = a.offset + (a.offset_dev ? (uint64_t)*a.offset_dev : 0);
  const int tr = threadIdx.x / a.cx, q = (blockIdx.x * a.cx + threadIdx.x % a.cx) * Q;
  if (tr >= a.ry || q >= a.quads) return;
  const int c = q * 4, left = VEC ? 4 * Q : a.D - c;
  const int64_t step = (int64_t)gridDim.y * a.ry;
  const auto load = [&](const T *p, E &e) {
    if (VEC) {
      e = *reinterpret_cast<const E *>(p);
    } else {
#pragma unroll
      for (int k = 0; k < 4 * Q; ++k)
        if (k < left) e.e[k] = p[k];
    }
  };
  for (int64_t r = (int64_t)blockIdx.y * a.ry + tr; r < a.rows; r += step) {
    E x, res, y;
    load(static_cast<const T *>(a.x) + r * a.ldx + c, x);
    if (RES) load(static_cast<const T *>(a.res) + r * a.ldr + c, res);
#pragma unroll
    for (int j = 0; j < Q; ++j) {
      fb::Philox4 w = {};
      if (a.from) w = draw((uint32_t)(q + j), (uint32_t)r, (uint32_t)off, (uint32_t)(off >> 32), a.key);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k = 4 * j + i;
        float v = RES ? to_f(res.e[k]) : 0.f;
        if (w.v[i] >= a.from) v = RES ? fmaf(to_f(x.e[k]), a.scale, v) : to_f(x.e[k]) * a.scale;
        y.e[k] = from_f<T>(v);
      }
    }
    T *const p = static_cast<T *>(a.y) + r * a.ldy + c;
    if (VEC) {
      *reinterpret_cast<E *>(p) = y;
    } else {
#pragma unroll
      for (int k = 0; k < 4 * Q; ++k)
        if (k < left) p[k] = y.e[k];
    }
  }
}

template <typename T, int Q, bool VEC> int run(DropArgs &a, cudaStream_t st) {
  const int groups = (a.quads + Q - 1) / Q;
  a.cx = std::min(groups, kThreads);
  a.ry = kThreads / a.cx;
  const int64_t across = (groups + a.cx - 1) / a.cx, down = (a.rows + a.ry - 1) / a.ry;
  // two waves of CTAs (8 an SM) that go down the rows, or a CTA for each few rows
  const dim3 grid((unsigned)across, (unsigned)std::min<int64_t>(std::max<int64_t>(1, std::min(down, 148 * 16 / across)), 65535));
  if (a.res) FB_TRY_CUDA(fb::launch(k_dropout<T, Q, VEC, true>, grid, kThreads, 0, st, a));
  else FB_TRY_CUDA(fb::launch(k_dropout<T, Q, VEC, false>, grid, kThreads, 0, st, a));
  return FB_OK;
}

}  // namespace

extern "C" int fb_dropout(int type, const void *x, int64_t ldx, const void *res, int64_t ldr, void *y, int64_t ldy, int64_t rows,
                          int D, float p, uint64_t seed, uint64_t offset, const int64_t *offset_dev, cudaStream_t stream) {
  const auto bad = [&](const char *what) { return fb::set_error(FB_ERR_ARG, std::string("dropout: ") + what); };
  if (type != FB_F32 && type != FB_BF16) return bad("unknown element type");
  if (!(p >= 0.f && p < 1.f)) return bad("p must be in [0, 1)");
  if (rows < 0 || D < 1) return bad("bad sizes");
  if (rows >= (int64_t)1 << 32) return fb::set_error(FB_ERR_UNSUPPORTED, "dropout: rows are counted in 32 bits");
  if (D > (1 << 20)) return fb::set_error(FB_ERR_UNSUPPORTED, "dropout: too many columns");
  if (rows && (!x || !y)) return bad("missing operand");
  if (rows > 1 && (ldx < D || ldy < D || (res && ldr < D))) return bad("leading dimension below the width");
  if (!rows) return FB_OK;
  const int es = type == FB_F32 ? 4 : 2;
  const uint64_t at = (uint64_t)(uintptr_t)x | (uint64_t)(uintptr_t)y | (uint64_t)(uintptr_t)res;
  if (at % es) return bad("rows that are not aligned to their elements");
  if (!aligned(8, offset_dev)) return bad("an offset that is not aligned to its element");
  uint64_t bits = at / es | (uint64_t)D;
  if (rows > 1) bits |= (uint64_t)ldx | (uint64_t)ldy | (res ? (uint64_t)ldr : 0);
  DropArgs a{};
  a.x = x, a.ldx = ldx, a.res = res, a.ldr = ldr, a.y = y, a.ldy = ldy, a.rows = rows, a.D = D, a.quads = (D + 3) / 4;
  // a word's upper 24 bits as a fraction are not below p: the word is not below ceil(p 2^24) 2^8 (p has 24 bits, the product is exact)
  a.from = (uint32_t)std::ceil(p * 16777216.f) << 8;
  a.scale = 1.f / (1.f - p);
  for (int r = 0; r < 10; ++r)
    a.key[r][0] = (uint32_t)seed + (uint32_t)r * 0x9E3779B9u, a.key[r][1] = (uint32_t)(seed >> 32) + (uint32_t)r * 0xBB67AE85u;
  a.offset = offset, a.offset_dev = offset_dev;
  if (type == FB_F32) return bits % 4 == 0 ? run<float, 1, true>(a, stream) : run<float, 1, false>(a, stream);
  return bits % 8 == 0 ? run<bf16, 2, true>(a, stream) : bits % 4 == 0 ? run<bf16, 1, true>(a, stream) : run<bf16, 1, false>(a, stream);
}
