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

// A row-major matrix [rows, cols] of the operator's type; as an operand of the
// products a bf16 matrix, or (plane > 0) the three bf16 planes of an fp32 one,
// `plane` elements apart.
struct Mat {
  const void *p;
  int64_t ld;
  int64_t plane = 0;
};

// The matrices of a call as the products read them: bf16 with a 16-byte
// aligned base and pitch (copied into the workspace when they are not), fp32
// split into planes; one launch for all of them.
constexpr int kMaxOperands = 6;
struct Operand {
  Mat src;
  int64_t rows;
  int cols;
  Mat *out;
};
int operands(Call &c, int type, const Operand *ops, int n);

// Where a product goes: rows of fp32 or bf16, written, or (fp32) added to.
struct Out {
  void *p;
  int64_t ld;
  int type, accumulate;
};

// Products on pairs of SMs (pair_gemm.cuh); operands as `operands` leaves
// them, fp32 accumulation, one rounding at the end (planes: fp32 results).
//   rows: C[m, n] = sum over 1 or 2 terms of A[m, ax_t + k] B_t(n, k), A [M, acols], k < K_t; B_t is [N, K_t], or
//         [K_t, N] when b_mn.  ax_t is a multiple of 64.
struct Term {
  Mat B;
  int ax, K;
};
//   b_n < N: B has only b_n of the N rows (columns); the rest of C is zeros.
int pair_rows(Call &c, const Mat &A, int64_t M, int acols, const Term *terms, int n_terms, bool b_mn, int N,
              const Out &out, int b_n = 0);
//   rows2: C_p = A B_p^T for two B [b_n, K] (C's columns past b_n are zeros)
int pair_rows2(Call &c, const Mat &A, int64_t M, const Mat *B, int K, int N, const Out *out, int b_n);
//   columns: C_p[m, n] = sum over the `rows` rows r of A[r, p * aprob + m] B[r, n], m < M, n < N, for p < probs
//         (1 or 2) outputs; A has acols columns.
int pair_columns(Call &c, const Mat &A, int64_t rows, int acols, int aprob, int probs, int M, const Mat &B, int N,
                 const Out *out);

}  // namespace fbh

#define FBH_TAKE(var, call, T, count)                                                        \
  T *var = static_cast<T *>((call).take((size_t)(count) * sizeof(T)));                       \
  if (!var) return fb::set_error(FB_ERR_ARG, "workspace too small")
#define FBH_TRY(x)            \
  do {                        \
    const int _rc = (x);      \
    if (_rc) return _rc;      \
  } while (0)
