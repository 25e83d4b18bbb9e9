// Products of a few rows (single queries) with a whole weight matrix: bound by
// reading the weights once, so they run on the CUDA cores with wide loads
// along the weights' rows instead of tensor-core tiles that would be empty.
#pragma once
#include "head.cuh"

namespace fbh {

// Whether a call of n rows takes this path: x's fp32 copy (rows of width K) has
// to fit into shared memory, and n is at most
//   fp32: 8.  The tensor cores would do six products for one.
//   bf16: 2, where the tensor cores' 256-row tiles cost little more than the
//     reading; with weights of at most 2^20 elements, where launches are what
//     costs, 8 forward (two launches, no partial results) and none backward
//     (six launches against four).
// us, this path / tensor cores, n rows (the tensor cores take 9 and 16 rows in
// the same time, so their 9 rows stand for fewer here):
//   gated block 2,048 x 8,192   fp32 fwd 1: 41 / 184, 4: 62 / 184;  bwd 1: 110 / 460, 8: 187 / 460
//                               bf16 fwd 1: 26 / 35, 2: 30 / 35, 4: 56 / 35;  bwd 1: 78 / 129, 2: 82 / 129, 4: 100 / 129
//   logits 2,048 x 50,000       fp32 fwd 1: 69 / 381, 8: 109 / 381;  bwd 1: 219 / 1221, 8: 327 / 1221
//                               bf16 fwd 1: 39 / 59, 2: 42 / 59, 4: 77 / 59;  bwd 1: 136 / 312, 2: 151 / 312, 4: 213 / 312
//   gated block 100 x 400       bf16 fwd 1: 8.2 / 12.4, 8: 9.9 / 12.4;  bwd 1: 19.7 / 16.9, 8: 24.5 / 16.9
//   logits 1,590 x 20,011       bf16 bwd 1: 125 / 126, 2: 130 / 126, 4: 155 / 126 (rows that no wide load lines up with:
//                               2 of them lose 3% here, 4 us of a call that no rule of its own is made for)
bool few_rows_ok(int type, bool bwd, int64_t n, int64_t K, int64_t weight_elements);
// h [n, F] (fp32, pitch F) = act(x Wg^T) (x Wu^T)
int few_rows_glu(Call &c, int type, int act, const Mat &x, int64_t n, int D, const Mat &wg, const Mat &wu, int F,
                 float *h);
// out [n, N] (pitch ldo, of `type`) = x W^T, x fp32 [n, K]
int few_rows_product(Call &c, int type, const float *x, int64_t n, int K, const Mat &w, int N, void *out, int64_t ldo);
// part [n][np]: (max, sum of exp2) of the rows' logits against w [V, D] in
// units of log2; np = few_rows_parts().
int few_rows_parts();
int few_rows_lse(Call &c, int type, const Mat &h, int64_t n, int D, const Mat &w, int64_t V, float2 *part);
// gu [n, 2 F] = [x Wg^T | x Wu^T], l [n, V] = h w^T (fp32)
int few_rows_gate_up(Call &c, int type, const Mat &x, int64_t n, int D, const Mat &wg, const Mat &wu, int F, float *gu);
int few_rows_logits(Call &c, int type, const Mat &h, int64_t n, int D, const Mat &w, int64_t V, float *l);
// The backward passes as a whole (few_rows_bwd.cu); V or F of at most 2^24,
// whose splits fit a grid.
constexpr int64_t kFewRowsTable = 1 << 24;
int few_rows_ffn_bwd(Call &c, const fb_gated_ffn &a);
int few_rows_xent_bwd(Call &c, const fb_softmax_xent &a);

}  // namespace fbh
