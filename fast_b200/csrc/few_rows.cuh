// Products of a few rows (single queries) with a whole weight matrix: bound by
// reading the weights once, so they run on the CUDA cores with wide loads
// along the weights' rows instead of tensor-core tiles that would be empty.
#pragma once
#include "head.cuh"

namespace fbh {

// The head's forward operators take this path up to 8 rows.  Both sides at
// (D, F) = (2048, 8192), bf16: FIGURES
constexpr int kFewRows = 8;

// Whether n rows of width K fit the kernels (their fp32 copy in shared memory).
bool few_rows_ok(int64_t n, int64_t K);
// h [n, F] (fp32, pitch F) = act(x Wg^T) (x Wu^T)
int few_rows_glu(Call &c, int type, int act, const Mat &x, int64_t n, int D, const Mat &wg, const Mat &wu, int F,
                 float *h);
// out [n, N] (pitch ldo, of `type`) = x W^T, x fp32 [n, K]
int few_rows_product(Call &c, int type, const float *x, int64_t n, int K, const Mat &w, int N, void *out, int64_t ldo);
// part [n][np]: (max, sum of exp2) of the rows' logits against w [V, D] in
// units of log2; np = few_rows_parts().
int few_rows_parts();
int few_rows_lse(Call &c, int type, const Mat &h, int64_t n, int D, const Mat &w, int64_t V, float2 *part);

}  // namespace fbh
