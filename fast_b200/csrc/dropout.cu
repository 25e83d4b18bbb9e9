// Dropout from a counter, with the residual sum behind it:
//
//   y = res + keep x / (1 - p),  keep[r, c] = (word c % 4 of Philox4x32-10(counter (c / 4, r, offset), key seed)) / 2^32 >= p
//
// decided on the word's upper 24 bits, as everywhere in the framework.  Nothing
// is stored: the backward, keep dy / (1 - p), draws the same numbers again.
// Bound by memory (x, res, y) and, in bf16, nearly as much by the generator's
// ten rounds for four columns, which is why a thread holds several groups of
// four at once and loads them before it draws.
#include <algorithm>
#include "history.cuh"
#include "runtime.cuh"

namespace {
using namespace fbq;

struct DropArgs {
  const void *x, *res;
  void *y;
  int64_t ldx, ldr, ldy, rows;
  int D, quads;                            // groups of four columns
  float p, scale;
  uint64_t seed, offset;
  const int64_t *offset_dev;
};

// VEC: whole groups are moved at once (D is a multiple of 4, rows aligned).
template <typename T, bool VEC, bool RES> __global__ void __launch_bounds__(256) k_dropout(DropArgs a) {
  fb::pdl_enter();
  const uint64_t off = a.offset + (a.offset_dev ? (uint64_t)*a.offset_dev : 0);
  const int64_t n = a.rows * a.quads, stride = (int64_t)gridDim.x * 256;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += stride) {
    const int64_t r = i / a.quads;
    const int q = (int)(i - r * a.quads), c = q * 4, left = VEC ? 4 : a.D - c;
    Vec<T, 4> x, res;
    const T *px = static_cast<const T *>(a.x) + r * a.ldx + c;
    const T *pr = RES ? static_cast<const T *>(a.res) + r * a.ldr + c : nullptr;
    if (VEC) {
      x = *reinterpret_cast<const Vec<T, 4> *>(px);
      if (RES) res = *reinterpret_cast<const Vec<T, 4> *>(pr);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (k < left) {
          x.e[k] = px[k];
          if (RES) res.e[k] = pr[k];
        }
    }
    const fb::Philox4 w = fb::philox4x32_10((uint32_t)q, (uint32_t)r, (uint32_t)off, (uint32_t)(off >> 32), (uint32_t)a.seed,
                                            (uint32_t)(a.seed >> 32));
    Vec<T, 4> y;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool keep = (float)(w.v[k] >> 8) * (1.0f / 16777216.0f) >= a.p;
      float v = keep ? to_f(x.e[k]) * a.scale : 0.f;
      if (RES) v += to_f(res.e[k]);
      y.e[k] = from_f<T>(v);
    }
    T *py = static_cast<T *>(a.y) + r * a.ldy + c;
    if (VEC) {
      *reinterpret_cast<Vec<T, 4> *>(py) = y;
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (k < left) py[k] = y.e[k];
    }
  }
}

template <typename T> int run(const DropArgs &a, bool vec, cudaStream_t st) {
  const int64_t n = a.rows * a.quads;
  const dim3 grid((unsigned)std::min<int64_t>((n + 255) / 256, 148 * 32));
  if (vec) {
    if (a.res) FB_TRY_CUDA(fb::launch(k_dropout<T, true, true>, grid, 256, 0, st, a));
    else FB_TRY_CUDA(fb::launch(k_dropout<T, true, false>, grid, 256, 0, st, a));
  } else {
    if (a.res) FB_TRY_CUDA(fb::launch(k_dropout<T, false, true>, grid, 256, 0, st, a));
    else FB_TRY_CUDA(fb::launch(k_dropout<T, false, false>, grid, 256, 0, st, a));
  }
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
  if (rows && (!x || !y)) return bad("missing operand");
  if (rows > 1 && (ldx < D || ldy < D || (res && ldr < D))) return bad("leading dimension below the width");
  if (!rows) return FB_OK;
  const int es = type == FB_F32 ? 4 : 2;
  const uint64_t at = (uint64_t)(uintptr_t)x | (uint64_t)(uintptr_t)y | (uint64_t)(uintptr_t)res;
  if (at % es) return bad("rows that are not aligned to their elements");
  uint64_t bits = at / es | (uint64_t)D;
  if (rows > 1) bits |= (uint64_t)ldx | (uint64_t)ldy | (res ? (uint64_t)ldr : 0);
  const DropArgs a{x, res, y, ldx, ldr, ldy, rows, D, (D + 3) / 4, p, 1.f / (1.f - p), seed, offset, offset_dev};
  return type == FB_F32 ? run<float>(a, bits % 4 == 0, stream) : run<bf16>(a, bits % 4 == 0, stream);
}
