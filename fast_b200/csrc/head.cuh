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

// Pieces of a workspace are accessed 16 bytes at a time and mapped for bulk copies.
inline int check_ws(const void *ws, const char *name) {
  if (!ws) return fb::set_error(FB_ERR_ARG, std::string(name) + ": no workspace");
  if (reinterpret_cast<uintptr_t>(ws) & 15u)
    return fb::set_error(FB_ERR_ARG, std::string(name) + ": the workspace must be 16-byte aligned");
  return FB_OK;
}

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
// split into planes; one launch for all of them.  Rows held out of a loss are
// laid out as zeros: their gradient's zeros alone would not keep an infinity
// or a NaN out of a sum over the rows.
constexpr int kMaxOperands = 6;
struct Operand {
  Mat src;
  int64_t rows;
  int cols;
  Mat *out;
  const int64_t *target = nullptr;           // given: rows whose target is not one of V are laid out as zeros
  int64_t V = 0;
  bool twice = false;                        // laid out a second time below itself (2 rows in all); bf16
};
int operands(Call &c, int type, const Operand *ops, int n);

// Where a product goes: rows of fp32 or bf16, written, or (fp32) added to.
struct Out {
  void *p;
  int64_t ld;
  int type, accumulate;
};

// Products on pairs of SMs (pair_gemm.cuh), operands as `operands` leaves
// them, fp32 accumulation, one rounding at the end (planes: fp32 results).
//   rows:    C[m, n] = sum over 1 or 2 terms of A[m, ax_t + k] B_t(n, k), A [M, acols], k < K_t; B_t is [b_n, K_t], or
//            [K_t, b_n] when b_mn; C's columns from b_n to N are zeros.  ax_t is a multiple of 64.
//   columns: C[m, n] = sum over the `rows` rows r of A[r, m] B_0[r, n]
struct Term {
  Mat B;
  int ax, K;
};
struct Product {
  bool columns, b_mn;
  Mat A;
  int acols;
  int64_t rows;
  Term term[2];
  int terms;
  int64_t M;
  int N, b_n;
  Out out;
  bool fold = false;                         // the result is the M / 2 sums of rows m and m + M / 2
};
inline Product rows_product(const Mat &A, int64_t M, int K, const Mat &B, bool b_mn, int N, const Out &out) {
  return Product{false, b_mn, A, K, M, {{B, 0, K}, {}}, 1, M, N, N, out};
}
inline Product columns_product(const Mat &A, int64_t rows, int M, const Mat &B, int N, const Out &out) {
  return Product{true, true, A, M, rows, {{B, 0, 0}, {}}, 1, M, N, N, out};
}
// Up to 4 independent products, all over bf16 or all over planes, in one
// launch (and one for the sums of those whose reduction is split).
int products(Call &c, const Product *p, int n);

}  // namespace fbh

#define FBH_TAKE(var, call, T, count)                                                        \
  T *var = static_cast<T *>((call).take((size_t)(count) * sizeof(T)));                       \
  if (!var) return fb::set_error(FB_ERR_ARG, "workspace too small")
#define FBH_TRY(x)            \
  do {                        \
    const int _rc = (x);      \
    if (_rc) return _rc;      \
  } while (0)
