// See head.cuh.
#include "head.cuh"
#include <algorithm>
#include "planes.cuh"

namespace {

struct Job {
  const void *src;
  int64_t lds, plane;
  void *dst;
  int ldd, cols, wide;                       // wide: 16-byte (8-byte) loads of the source's groups of 4
  const int64_t *target;                     // Operand's
  int64_t V, again;                          // elements to the second copy (0: none)
  uint32_t groups, per_row;                  // groups of 4 columns, in all and a row
  unsigned first;                            // first CTA of the job
};
struct Jobs {
  Job j[fbh::kMaxOperands];
  int n;
};
constexpr int kGroups = 2;                   // groups of 4 a thread lays out

// bf16 rows into a pitch of whole 128-byte lines, or (planes) fp32 rows split.
template <bool PLANES> __global__ void __launch_bounds__(256) k_operands(const __grid_constant__ Jobs a) {
  fb::pdl_enter();
  int q = 0;
  while (q + 1 < a.n && blockIdx.x >= a.j[q + 1].first) ++q;
  const Job &j = a.j[q];
  const uint32_t at = (blockIdx.x - j.first) * (256 * kGroups) + threadIdx.x;
#pragma unroll
  for (int e = 0; e < kGroups; ++e) {
    const uint32_t i = at + e * 256;
    if (i >= j.groups) return;
    const uint32_t r = i / j.per_row;
    const int c = (int)(i - r * j.per_row) * 4;
    uint16_t *d = static_cast<uint16_t *>(j.dst) + (int64_t)r * j.ldd + c;
    const bool live = !j.target || (j.target[r] >= 0 && j.target[r] < j.V);
    if constexpr (PLANES) {
      const float *s = static_cast<const float *>(j.src) + r * j.lds + c;
      float v[4] = {0.f, 0.f, 0.f, 0.f};
      if (j.wide && live) *reinterpret_cast<float4 *>(v) = *reinterpret_cast<const float4 *>(s);
      else if (live)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (c + k < j.cols) v[k] = s[k];
      fbplanes::put4(d, j.plane, v[0], v[1], v[2], v[3]);
    } else {
      const uint16_t *s = static_cast<const uint16_t *>(j.src) + r * j.lds + c;
      ushort4 v = make_ushort4(0, 0, 0, 0);
      if (j.wide && live) v = *reinterpret_cast<const ushort4 *>(s);
      else if (live) {
        v.x = s[0];
        if (c + 1 < j.cols) v.y = s[1];
        if (c + 2 < j.cols) v.z = s[2];
        if (c + 3 < j.cols) v.w = s[3];
      }
      *reinterpret_cast<ushort4 *>(d) = v;
      if (j.again) *reinterpret_cast<ushort4 *>(d + j.again) = v;
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
    if (!planes && !o.target && !o.twice && ((reinterpret_cast<uintptr_t>(o.src.p) | (uintptr_t)(o.src.ld * 2)) & 15u) == 0) continue;
    // rows on 128-byte boundaries: a 128-byte box row that crosses one costs the copy engine two requests
    const int64_t ld = round_up(o.cols, 64), plane = o.rows * ld;
    void *p = c.take((size_t)(plane * (planes ? 6 : (o.twice ? 4 : 2))));
    if (!p) return fb::set_error(FB_ERR_ARG, "workspace too small");
    *o.out = Mat{p, ld, planes ? plane : 0};
    if (o.rows == 0) continue;
    const uint32_t per_row = (uint32_t)(o.cols + 3) / 4;
    const int64_t groups = o.rows * per_row;
    if (groups > UINT32_MAX / 2) return fb::set_error(FB_ERR_UNSUPPORTED, "operand of more than 2^33 elements");
    const int es = elem(type);
    const bool wide = o.cols % 4 == 0 && ((reinterpret_cast<uintptr_t>(o.src.p) | (uintptr_t)(o.src.ld * es)) & (4 * es - 1)) == 0;
    jobs.j[jobs.n++] = Job{o.src.p, o.src.ld, plane, p, (int)ld, o.cols, wide, o.target, o.V, o.twice ? plane : 0, (uint32_t)groups, per_row, ctas};
    ctas += (unsigned)((groups + 256 * kGroups - 1) / (256 * kGroups));
  }
  if (c.dry || jobs.n == 0) return FB_OK;
  FB_TRY_CUDA(fb::launch(planes ? k_operands<true> : k_operands<false>, ctas, 256, 0, c.stream, jobs));
  FB_LAUNCHED("k_operands");
  return FB_OK;
}

}  // namespace fbh
