// Host-side pieces the node-ranking head's operators share: workspace
// carving, operands laid out for the tensor maps, products.
#pragma once
#include <cstddef>
#include "runtime.cuh"

namespace fbh {

inline int elem(int type) { return type == FB_F32 ? 4 : 2; }
inline int64_t round_up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

// One call of an operator.  A `dry` run walks the same steps without a launch
// and so measures the workspace they take.
struct Call {
  uint8_t *base;
  size_t off = 0, peak = 0, cap;
  bool dry;
  cudaStream_t stream;
  Call(void *ws, size_t ws_bytes, cudaStream_t st)
      : base(static_cast<uint8_t *>(ws)), cap(ws_bytes), dry(false), stream(st) {}
  Call() : base(reinterpret_cast<uint8_t *>((uintptr_t)1 << 20)), cap((size_t)-1), dry(true), stream(nullptr) {}
  // 256-byte aligned piece of the workspace; null when it is used up.  Steps
  // run in stream order, so a step's pieces are given back by restoring `off`.
  void *take(size_t bytes) {
    const size_t at = off;
    off += (bytes + 255) / 256 * 256;
    peak = off > peak ? off : peak;
    return off <= cap ? base + at : nullptr;
  }
};

// A row-major matrix [rows, cols] of the operator's type.
struct Mat {
  const void *p;
  int64_t ld;
};

// m as the products read it: 16-byte aligned base and pitch.  Copies into the
// workspace when m is not.
int aligned(Call &c, int type, const Mat &m, int64_t rows, int cols, Mat *out);

// C (+)= A B^T (NT), A B (NN) or A^T B (TN: C [N, K] over M rows), as
// fb_gemm_group / fb_gemm_bf16_group define them; C is fp32.
int product(Call &c, int type, int kind, const Mat &A, const Mat &B, float *C, int64_t ldc, int64_t M, int N, int K,
            int accumulate);

// dst (fp32 or bf16) = src (fp32), or += when accumulate (fp32 dst).
int store_rows(Call &c, const float *src, int64_t lds, void *dst, int64_t ldd, int dst_type, int64_t rows, int cols,
               int accumulate);

}  // namespace fbh

#define FBH_TAKE(var, call, T, count)                                                        \
  T *var = static_cast<T *>((call).take((size_t)(count) * sizeof(T)));                       \
  if (!var) return fb::set_error(FB_ERR_ARG, "workspace too small")
#define FBH_TRY(x)            \
  do {                        \
    const int _rc = (x);      \
    if (_rc) return _rc;      \
  } while (0)
