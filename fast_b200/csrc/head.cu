// See head.cuh.
#include "head.cuh"
#include <algorithm>

namespace {

struct Job {
  const void *src;
  int64_t lds, rows, ldd, plane;
  void *dst;
  int cols;
  unsigned first;                            // first CTA of the job
};
struct Jobs {
  Job j[fbh::kMaxOperands];
  int n;
};
constexpr int kPerCta = 256 * 8;             // elements a CTA lays out

// bf16 rows into a pitch, or (planes) fp32 x as x0 + x1 + x2: the leading 8
// significant bits, the next 8, the last 8.  Cutting bits off is exact and
// cannot overflow; x0 of an infinity or NaN carries it alone.
template <bool PLANES> __global__ void __launch_bounds__(256) k_operands(const __grid_constant__ Jobs a) {
  fb::pdl_enter();
  int q = 0;
  while (q + 1 < a.n && blockIdx.x >= a.j[q + 1].first) ++q;
  const Job &j = a.j[q];
  const int64_t total = j.rows * j.cols, at = (int64_t)(blockIdx.x - j.first) * kPerCta;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int64_t i = at + e * 256 + threadIdx.x;
    if (i >= total) return;
    const int64_t r = i / j.cols;
    const int c = (int)(i - r * j.cols);
    uint16_t *d = static_cast<uint16_t *>(j.dst) + r * j.ldd + c;
    if (!PLANES) {
      *d = static_cast<const uint16_t *>(j.src)[r * j.lds + c];
    } else {
      const float x = static_cast<const float *>(j.src)[r * j.lds + c];
      const uint32_t b0 = __float_as_uint(x) & 0xFFFF0000u;
      const bool fin = (b0 & 0x7F800000u) != 0x7F800000u;
      const float r1 = fin ? x - __uint_as_float(b0) : 0.f;
      const uint32_t b1 = __float_as_uint(r1) & 0xFFFF0000u;
      const uint32_t b2 = __float_as_uint(r1 - __uint_as_float(b1));
      d[0] = (uint16_t)(b0 >> 16);
      d[j.plane] = (uint16_t)(b1 >> 16);
      d[2 * j.plane] = (uint16_t)(b2 >> 16);
    }
  }
}

}  // namespace

namespace fbh {

int operands(Call &c, int type, const Operand *ops, int n) {
  Jobs jobs;
  jobs.n = 0;
  unsigned ctas = 0;
  const bool planes = type == FB_F32;
  for (int i = 0; i < n; ++i) {
    const Operand &o = ops[i];
    *o.out = Mat{o.src.p, o.src.ld};
    if (!planes && ((reinterpret_cast<uintptr_t>(o.src.p) | (uintptr_t)(o.src.ld * 2)) & 15u) == 0) continue;
    // rows on 128-byte boundaries: a 128-byte box row that crosses one costs the copy engine two requests
    const int64_t ld = round_up(o.cols, 64), plane = o.rows * ld;
    void *p = c.take((size_t)(plane * (planes ? 6 : 2)));
    if (!p) return fb::set_error(FB_ERR_ARG, "workspace too small");
    *o.out = Mat{p, ld, planes ? plane : 0};
    if (o.rows == 0) continue;
    jobs.j[jobs.n++] = Job{o.src.p, o.src.ld, o.rows, ld, plane, p, o.cols, ctas};
    ctas += (unsigned)((o.rows * o.cols + kPerCta - 1) / kPerCta);
  }
  if (c.dry || jobs.n == 0) return FB_OK;
  FB_TRY_CUDA(fb::launch(planes ? k_operands<true> : k_operands<false>, ctas, 256, 0, c.stream, jobs));
  FB_LAUNCHED("k_operands");
  return FB_OK;
}

}  // namespace fbh
