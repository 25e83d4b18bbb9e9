// See head.cuh.
#include "head.cuh"
#include <algorithm>

namespace {

// rows x cols elements of `es` bytes into a pitch with zeros past cols.
template <typename U>
__global__ void k_copy_rows(const U *src, int64_t lds, U *dst, int64_t ldd, int64_t rows, int cols) {
  fb::pdl_enter();
  const int64_t total = rows * ldd;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / ldd;
    const int c = (int)(i - r * ldd);
    dst[i] = c < cols ? src[r * lds + c] : (U)0;
  }
}

unsigned blocks_for(int64_t n) { return (unsigned)std::max<int64_t>(1, std::min<int64_t>((n + 255) / 256, 148 * 16)); }

}  // namespace

namespace fbh {

int aligned(Call &c, int type, const Mat &m, int64_t rows, int cols, Mat *out) {
  const int es = elem(type);
  *out = m;
  if (((reinterpret_cast<uintptr_t>(m.p) | (uintptr_t)(m.ld * es)) & 15u) == 0) return FB_OK;
  const int64_t ld = round_up(cols, 16 / es);
  void *p = c.take((size_t)(rows * ld * es));
  if (!p) return fb::set_error(FB_ERR_ARG, "workspace too small");
  *out = Mat{p, ld};
  if (c.dry || rows == 0) return FB_OK;
  if (type == FB_F32)
    FB_TRY_CUDA(fb::launch(k_copy_rows<uint32_t>, blocks_for(rows * ld), 256, 0, c.stream,
                           static_cast<const uint32_t *>(m.p), m.ld, static_cast<uint32_t *>(p), ld, rows, cols));
  else
    FB_TRY_CUDA(fb::launch(k_copy_rows<uint16_t>, blocks_for(rows * ld), 256, 0, c.stream,
                           static_cast<const uint16_t *>(m.p), m.ld, static_cast<uint16_t *>(p), ld, rows, cols));
  FB_LAUNCHED("k_copy_rows");
  return FB_OK;
}

int product(Call &c, int kind, const Mat &A, const Mat &B, float *C, int64_t ldc, int64_t M, int N, int K,
            int accumulate) {
  fb_gemm_problem p{};
  p.kind = kind;
  p.A = static_cast<const float *>(A.p); p.lda = A.ld; p.k1 = K;
  p.B = static_cast<const float *>(B.p); p.ldb = B.ld;
  p.C = C; p.ldc = ldc; p.M = M; p.N = N; p.K = K; p.accumulate = accumulate;
  const size_t bytes = fb_gemm_group_ws_bytes(&p, 1), mark = c.off;
  void *ws = c.take(bytes);
  if (!ws) return fb::set_error(FB_ERR_ARG, "workspace too small");
  if (!c.dry) FBH_TRY(fb_gemm_group(&p, 1, ws, bytes, c.stream));
  c.off = mark;
  return FB_OK;
}

}  // namespace fbh
