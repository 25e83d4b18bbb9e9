// bf16 products on pairs of SMs for the node-ranking head: tcgen05.mma with
// cta_group::2, operands by TMA, fp32 accumulators in tensor memory, and the
// operators' own arithmetic in the epilogue.
//
//   kernel k_pair<EPI, P>: C[m, n] = sum_k A(m, k) B(n, k)
//   a_mn / b_mn: the operand lies with its m (n) index contiguous (the matrix
//   is stored [k][m]); else with k contiguous.
//   EPI = kStore takes up to kMaxProbs independent products in one launch
//   (their layouts, tile widths and output types are fields): a backward pass's
//   products are short, and a launch of its own costs one 3 to 4 us of ramp.
//   P = 3: fp32 operands, each as three bf16 planes x = x0 + x1 + x2 of 8
//   significant bits (exact: 24 bits in all; planes.cuh).  Six of the nine plane
//   products are summed, smallest first.  The three left out are below 2^-21 of
//   the product (x1 < 2^-7 x, x2 < 2^-15 x), 2^-24.5 on average, all of its sign.
//   The tensor cores' accumulation truncates, so it runs over 64 k
//   only: the epilogue warps add each such slab to an fp32 sum in registers
//   while the next one is computed.  kLsePlanes and kProbPlanes are kLse and
//   kProb on that sum, in registers: the logits of fp32 rows are not stored
//   either, and G leaves as its three planes.
//
// A cluster of two CTAs works on a 256 x BN tile: each CTA stages 128 rows of
// A and BN / 2 rows of B, the MMA of the even CTA reads both halves from both
// SMs, and each CTA's tensor memory holds its own 128 rows of the tile.  So
// every operand byte is staged once per pair: a BN = 256 tile moves 64 bytes
// of shared memory a cycle and SM in each direction (TMA writes, MMA reads),
// half of what one SM alone would need.
//
// CTA = 12 or 20 warps: 0 TMA producer (one lane), 1 TMEM allocator and, in the
// even CTA, MMA issuer (one lane), the rest from 4 on epilogue: two per TMEM
// lane quadrant, each half of the columns.  Where the epilogue takes an
// exponential of every element there are two such sets, one for each
// accumulator: they work on alternate tiles, so that one's exponentials (the
// XU pipe) fall into the other's loads, maxima and stores.  Stages of 64 k travel through a ring
// of kStages; the loads of both CTAs count on the even CTA's barrier, MMA
// completion frees the stage in both.  Accumulators: two of up to 256 columns
// (the epilogue drains one while the other fills).  kGluBwd's tile takes 384:
// g | u has one place and dh two, dh comes first, and the g | u stages wait for
// the epilogue of the tile before, which has had dh's time to drain them.
// kGluBwdLong gives each slab of g | u one of the two places, and then dh.
//
// No load uses cluster multicast.  Every wait is bounded: past the limit a
// CTA records an error, stops, gives its copies time to land and leaves.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <algorithm>
#include <cstring>
#include "act.cuh"
#include "head.cuh"
#include "planes.cuh"
#include "tc_common.cuh"

namespace fbpair {

using namespace fbtc;

enum : int { kStore = 0, kGluFwd = 2, kGluBwd = 3, kLse = 4, kProb = 5, kLseLong = 6, kLsePlanes = 7, kProbPlanes = 8, kGluBwdLong = 9,
              kProbTwo = 10 };
using fbact::kGelu;
using fbact::kRelu;
using fbact::kSilu;

constexpr int BK = 64;                        // k per stage: one 128-byte swizzle row of bf16
constexpr int kHalfM = 128;                   // rows of a tile per CTA
constexpr int kABytes = kHalfM * BK * 2;      // 16 KB
// B of a stage: BN / 2 <= 128 rows; planes (a stage holds one plane of a slab): 64 rows
template <int P> __host__ __device__ constexpr int b_bytes() { return (P == 3 ? 64 : 128) * BK * 2; }
template <int P> __host__ __device__ constexpr int stage_bytes() { return kABytes + b_bytes<P>(); }
constexpr int kBox = BK * 128;                // MN-major box: 64 k rows of 64 elements
constexpr int kWarpEpi0 = 4;
template <int EPI> __host__ __device__ constexpr int epi_warps() {
  return EPI == kLse || EPI == kLseLong || EPI == kProb ? 16 : 8;
}
template <int EPI> __host__ __device__ constexpr int threads_of() { return (kWarpEpi0 + epi_warps<EPI>()) * 32; }
constexpr int kTmemCols = 512;
constexpr int kStageOut = 4096;               // one staged output block: 32 rows of 128 bytes
constexpr int kLseSlab = 16;                  // kLseLong: stages summed in tensor memory at a time
constexpr int kGluSlab = 4;                   // kGluBwdLong: the same for g and u
// Stages after which an accumulator of the first term goes to registers; 0: at the end.
template <int EPI> __host__ __device__ constexpr int slab_of() {
  return EPI == kLseLong ? kLseSlab : (EPI == kGluBwdLong ? kGluSlab : 0);
}
template <int EPI> __host__ __device__ constexpr int out_bytes() {
  return EPI == kGluBwd || EPI == kGluBwdLong ? 3 * kStageOut : EPI == kProbTwo ? 2 * kStageOut : (EPI == kLse || EPI == kLseLong ? 0 : kStageOut);
}
template <int EPI, int P> __host__ __device__ constexpr int stages() {
  return P == 3 ? 8 : (EPI == kGluBwd || EPI == kGluBwdLong ? 4 : (EPI == kProb || EPI == kProbTwo ? 5 : 6));
}
template <int EPI, int P> __host__ __device__ constexpr int smem_bytes() {
  return 1024 + stages<EPI, P>() * stage_bytes<P>() + epi_warps<EPI>() * out_bytes<EPI>() + 256;
}
static_assert(smem_bytes<kGluBwd, 1>() <= 232448 && smem_bytes<kGluBwdLong, 1>() <= 232448 && smem_bytes<kProbTwo, 1>() <= 232448 && smem_bytes<kProb, 1>() <= 232448 &&
                  smem_bytes<kStore, 1>() <= 232448 &&
                  smem_bytes<kStore, 3>() <= 232448 && smem_bytes<kProbPlanes, 3>() <= 232448, "shared memory exceeds 227 KB");

constexpr int kMaxProbs = 4;

// One product.  Two terms may feed a tile: kGluBwd's first one fills the dh
// columns, its second g | u (kGluBwdLong: the other way round); elsewhere the second continues the same sum (dx = dg Wg + du Wu) and its
// stages follow the first's.
struct PairProb {
  CUtensorMap ta[2], tb[2];                   // by term; kGlu*: tb[0] = Wg, tb[1] = Wu
  CUtensorMap tc;                             // output (has_tc); the splits' partial results, one above the other
  int a_mn, b_mn, bn, f32;                    // layouts, tile width, output type
  int mt, nt, splits, kb[2], kper;            // tiles along m and n, splits of k; stages per term and per split
  int ax[2];                                  // A's first column per term (k contiguous)
  int M, N;                                   // rows and columns of the result
  int has_tc, accumulate;                     // accumulate (fp32): add to what is there
  int split_rows;                             // rows of tc between two splits
  void *C;                                    // no has_tc: the result, row pitch ldc
  int64_t ldc;
};
// Fields of one launch; all but kStore have one product.
struct PairArgs {
  PairProb p[kMaxProbs];
  int n, tile0[kMaxProbs + 1];                // products; tiles before each
  int32_t *err;
  CUtensorMap tw, tc2[2];                     // kGluBwd: Wd; outputs dg, du (kProbPlanes: G's planes 1, 2; kProbTwo: its second part)
  int act;
  float2 *part;                               // kLse*: [M][2 nt] (kLseLong: [M][4 nt]) (max, sum of exp2) partials
  const int64_t *target;                      // kProb*
  const float *lse, *dloss;
  int64_t V, v0;
};
static_assert(sizeof(PairArgs) <= 4096, "kernel parameters exceed 4 KB");

// ---- PTX -----------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t cta_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// One lane of the (converged) warp.  The loops around the single-lane work run
// on all lanes: their values then are warp-uniform to the compiler, which an
// MMA's descriptors have to be (in a one-lane branch every MMA cost 173 cycles
// whatever its width).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// Shared-memory address of `p` in the even CTA of the pair.
__device__ __forceinline__ uint32_t leader_addr(const void *p) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem_u32(p)));
  return a;
}
// Arrival from either CTA.  What it orders are tensor-memory reads, fenced by
// tcgen05.fence before it, so the default CTA scope is enough; a cluster-scope
// release or acquire here also waits for every global store in flight (2x the
// time of the short products).
__device__ __forceinline__ void arrive_at(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// mbar_wait whose first try, which mostly succeeds, reads no clock.
__device__ __forceinline__ bool wait(uint64_t *bar, uint32_t parity, volatile int *abort_flag, int32_t *err) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  while (!mbar_try_wait(bar, parity)) {
    if (*abort_flag) return false;
    if (clock64() - t0 > kWaitCycles) {
      *abort_flag = 1;
      atomicOr(err, kErrTimeout);
      return false;
    }
  }
  return true;
}
// The same from plane z of a matrix kept as planes.
__device__ __forceinline__ void load3(void *dst, const CUtensorMap *map, uint32_t bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, "
      "%5}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
      : "memory");
}
// A tile of this CTA's shared memory, counted on a barrier of the even CTA.
__device__ __forceinline__ void load2(void *dst, const CUtensorMap *map, uint32_t bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], "
      "[%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y)
      : "memory");
}
__device__ __forceinline__ void alloc2(uint32_t *holder, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(holder)), "r"(ncols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void dealloc2(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
__device__ __forceinline__ void mma2(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(ad), "l"(bd), "r"(idesc), "r"(accumulate)
      : "memory");
}
// The barrier at this offset in both CTAs, once every MMA issued so far is complete.
__device__ __forceinline__ void commit2(uint64_t *bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}
__device__ __forceinline__ void store_tile(const CUtensorMap *map, const void *src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(smem_u32(src)), "r"(x), "r"(y)
               : "memory");
}
__device__ __forceinline__ void add_tile(const CUtensorMap *map, const void *src, int x, int y) {
  asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(smem_u32(src)), "r"(x), "r"(y)
               : "memory");
}
__device__ __forceinline__ void store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void store_wait() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}
// 32 accumulator columns without the wait (tmem_wait before the values are used).
__device__ __forceinline__ void tmem_ld32_nowait(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld16_nowait(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// Shared-memory matrix descriptor (128-byte swizzle, 1024-byte aligned tile).
// K-major: rows of 128 B, 8-row groups 1024 B apart; 16 k = 32 B further on.
// MN-major: [64 k][64 mn] boxes side by side along mn, 8-row groups 1024 B
// apart; 16 k = 2 KB further on.
__device__ __forceinline__ uint64_t sdesc(uint32_t saddr, bool mn) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr >> 4) & 0x3FFFu);
  d |= (uint64_t)(mn ? (kBox >> 4) : 1) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;                     // descriptor version (sm_100)
  d |= (uint64_t)2 << 61;                     // SWIZZLE_128B
  return d;
}
// D fp32, A and B bf16, dense, M = 256 over the pair
__host__ __device__ constexpr uint32_t idesc2(int bn, bool a_mn, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) |
         ((uint32_t)(bn >> 3) << 17) | ((uint32_t)(256 >> 4) << 24);
}

// 2^x by the hardware's approximation (2 ulp, denormal results are zeros)
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ---- epilogue pieces -----------------------------------------------------------------------------
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&v);
}

// One lane's row (128 bytes in eight 16-byte pieces) of a staged block: the
// layout a 128-byte-swizzled tensor map stores from.
__device__ __forceinline__ void stage_row(uint8_t *buf, int lane, const uint32_t (&w)[32]) {
#pragma unroll
  for (int c = 0; c < 8; ++c)
    *reinterpret_cast<uint4 *>(buf + lane * 128 + ((c ^ (lane & 7)) << 4)) =
        make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
}

// Its first or second 64 bytes.
__device__ __forceinline__ void stage_half(uint8_t *buf, int lane, int which, const uint32_t (&w)[16]) {
#pragma unroll
  for (int k = 0; k < 4; ++k)
    *reinterpret_cast<uint4 *>(buf + lane * 128 + (((4 * which + k) ^ (lane & 7)) << 4)) =
        make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
}

// Sends a staged block (32 rows from `row`, 64 bf16 or 32 fp32 columns from
// `col`) to the product's output.  Rows past M and columns past N stay out.
template <bool F32OUT>
__device__ __forceinline__ void send(const PairProb &a, const CUtensorMap *tc, const uint8_t *buf, int ybase, int row,
                                     int col, int lane) {
  fence_async_smem();
  __syncwarp();
  const bool in = row < a.M && col < a.N;
  if (lane == 0) {                            // one bulk group per block, empty or not
    if (in && a.has_tc) {
      if (F32OUT && a.accumulate) add_tile(tc, buf, col, ybase + row);
      else store_tile(tc, buf, col, ybase + row);
    }
    store_commit();
  }
  if (!in || a.has_tc) return;
  const int nr = min(32, a.M - row);
  if (F32OUT) {
    float *p = static_cast<float *>(a.C) + row * a.ldc + col + lane;
    if (col + lane < a.N)
      for (int r = 0; r < nr; ++r) {
        const float v = *reinterpret_cast<const float *>(buf + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4);
        p[r * a.ldc] = a.accumulate ? p[r * a.ldc] + v : v;
      }
  } else {
    uint16_t *p = static_cast<uint16_t *>(a.C) + row * a.ldc + col;
    for (int r = 0; r < nr; ++r)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c = lane + 32 * h;
        if (col + c < a.N)
          p[r * a.ldc + c] =
              *reinterpret_cast<const uint16_t *>(buf + r * 128 + (((c >> 3) ^ (r & 7)) << 4) + (c & 7) * 2);
      }
  }
}

// 64 values of a lane's row as their planes (planes.cuh), one plane after the other, to the launch's three outputs.
template <bool FINITE>
__device__ __forceinline__ void send_planes(const PairArgs &a, float (&v)[64], uint8_t *buf, int row, int col, int lane) {
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    uint32_t r[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      if (k == 2) {
        r[i] = fbplanes::pair(__float_as_uint(v[2 * i]), __float_as_uint(v[2 * i + 1]));
        continue;
      }
      const fbplanes::Cut lo = fbplanes::cut<FINITE>(v[2 * i]), hi = fbplanes::cut<FINITE>(v[2 * i + 1]);
      r[i] = fbplanes::pair(lo.lead, hi.lead);
      v[2 * i] = lo.rest;
      v[2 * i + 1] = hi.rest;
    }
    if (lane == 0) store_wait<0>();
    __syncwarp();
    stage_row(buf, lane, r);
    send<false>(a.p[0], k == 0 ? &a.p[0].tc : &a.tc2[k - 1], buf, 0, row, col, lane);
    __syncwarp();
  }
}

// Maximum and sum of exp2 of a row's 64 logits, of which `left` are inside the table, in units of log2.
__device__ __forceinline__ float2 max_sum(float (&v)[64], int left) {
  constexpr float kLog2e = 1.44269504088896340736f;
  if (left < 64) {
#pragma unroll
    for (int i = 0; i < 64; ++i)
      if (i >= left) v[i] = -INFINITY;        // past the table
  }
  float m = v[0];
#pragma unroll
  for (int i = 1; i < 64; ++i) m = fmaxf(m, v[i]);
  m *= kLog2e;
  // nothing but -inf: subtract 0, so that exp2 gives zeros (and NaN stays NaN)
  const float base = m == -INFINITY ? 0.f : m;
  float s0 = 0.f, s1 = 0.f;
#pragma unroll
  for (int i = 0; i < 64; i += 2) {
    s0 += ex2(fmaf(v[i], kLog2e, -base));
    s1 += ex2(fmaf(v[i + 1], kLog2e, -base));
  }
  return make_float2(m, s0 + s1);
}

struct Tile {
  int p, m, n, k0, k1;                        // k0 .. k1 - 1: stages, the terms' one after the other
  int ybase;                                  // first row of this split's results
};

// Products one after the other, then splits; tiles run along m inside groups
// of 8 m-tiles, so that a wave's tiles share few distinct operand rows.
template <int EPI> __device__ __forceinline__ Tile tile_at(const PairArgs &a, int t) {
  Tile q;
  q.p = 0;
  if (EPI == kStore)
    while (q.p + 1 < a.n && t >= a.tile0[q.p + 1]) ++q.p;
  const PairProb &b = a.p[q.p];
  t -= EPI == kStore ? a.tile0[q.p] : 0;
  const int mt = b.mt, nt = b.nt, per = mt * nt;
  const int s = EPI == kStore ? t / per : 0;
  int r = t - s * per;
  const int grp = 8 * nt, g = r / grp;
  r -= g * grp;
  const int gm = min(8, mt - 8 * g);
  q.m = 8 * g + r % gm;
  q.n = r / gm;
  q.k0 = s * b.kper;
  q.k1 = min(b.kb[0] + b.kb[1], q.k0 + b.kper);
  q.ybase = s * b.split_rows;
  return q;
}

// Columns c .. c + 31 of g (and + 128: u, and of dh at td) of this warp's 32 rows:
// h (and dg, du) staged as half of the warp's 128-byte rows, sent off with the
// second half: the copy engine takes a 64-byte row no faster than a 128-byte one.
// h, dg and du are rounded to bf16 here, once each: they are the next products'
// operands, and the tensor cores' bf16 products are what a bf16 call is for (fp32
// operands take six of them).  The results then carry two roundings, their own
// and this one: 0.0024 off in the 2-norm, 0.0017 with h, dg, du in fp32 (12,000 x
// 172 x 688).  A module of elementary bf16 operations rounds g, u, act(g) and h.
template <int ACT, bool BWD>
__device__ __forceinline__ void glu_block(const PairArgs &a, uint32_t t, uint32_t td, int c, int which, uint8_t *buf, int row,
                                          int col, int lane) {
  uint32_t w[BWD ? 3 : 1][16];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    uint32_t g[16], u[16], d[BWD ? 16 : 1];
    tmem_ld16_nowait(t + c + 16 * q, g);
    tmem_ld16_nowait(t + 128 + c + 16 * q, u);
    if constexpr (BWD) tmem_ld16_nowait(td + c + 16 * q, d);
    tmem_wait();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float h[2], dg[2], du[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float2 f = fbact::act_fast<ACT>(__uint_as_float(g[2 * i + e]));
        const float uv = __uint_as_float(u[2 * i + e]);
        h[e] = f.x * uv;
        if constexpr (BWD) {
          const float dv = __uint_as_float(d[2 * i + e]);
          dg[e] = dv * uv * f.y;
          du[e] = dv * f.x;
        }
      }
      w[0][8 * q + i] = pack(h[0], h[1]);
      if constexpr (BWD) {
        w[1][8 * q + i] = pack(dg[0], dg[1]);
        w[2][8 * q + i] = pack(du[0], du[1]);
      }
    }
  }
  if (which == 0) {
    if (lane == 0) store_wait<0>();           // the tile before has left the buffers
    __syncwarp();
  }
#pragma unroll
  for (int o = 0; o < (BWD ? 3 : 1); ++o) stage_half(buf + o * kStageOut, lane, which, w[o]);
  if (which == 0) return;
  fence_async_smem();
  __syncwarp();
  if (lane == 0) {
    if (row < a.p[0].M && col < a.p[0].N)
#pragma unroll
      for (int o = 0; o < (BWD ? 3 : 1); ++o) store_tile(o ? &a.tc2[o - 1] : &a.p[0].tc, buf + o * kStageOut, col, row);
    store_commit();
  }
}

template <int EPI, int P = 1>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(threads_of<EPI>(), 1) k_pair(const __grid_constant__ PairArgs a) {
  static_assert((P == 3) == (EPI == kLsePlanes || EPI == kProbPlanes) || EPI == kStore, "the epilogue fits its operands");
  constexpr int kStages = stages<EPI, P>(), kStageBytes = stage_bytes<P>(), kBBytes = b_bytes<P>();
  constexpr int kBufs = EPI == kGluBwd ? 1 : 2, kEpiWarps = epi_warps<EPI>();
  constexpr bool kAlt = EPI == kLse || EPI == kProb;            // two sets of epilogue warps, alternate tiles
  constexpr bool kDual = EPI == kGluFwd || EPI == kGluBwd || EPI == kGluBwdLong;   // B: 128 rows of Wg in one CTA, of Wu in the other
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = align1024(smem_raw);
  auto sA = [&](int s) { return smem + s * kStageBytes; };
  auto sB = [&](int s) { return smem + s * kStageBytes + kABytes; };
  uint8_t *outs = smem + kStages * kStageBytes;
  uint64_t *bars = reinterpret_cast<uint64_t *>(outs + kEpiWarps * out_bytes<EPI>());
  uint64_t *full = bars, *empty = bars + kStages, *accf = bars + 2 * kStages, *acce = accf + 2;
  uint32_t *holder = reinterpret_cast<uint32_t *>(acce + 2);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(holder + 1);

  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = cta_rank();
  if (warp == 0) {
    if (lane < kStages) {
      mbar_init(full + lane, 1);              // the even CTA's: its own expect, both CTAs' bytes
      mbar_init(empty + lane, 1);
    } else if (lane >= 16 && lane < 18) {
      mbar_init(accf + lane - 16, 1);
      mbar_init(acce + lane - 16, kAlt ? kEpiWarps : 2 * kEpiWarps);   // the even CTA's: both CTAs' epilogue warps
    } else if (lane == 18) {
      *abort_flag = 0;
    }
    fence_barrier_init();
    __syncwarp();
  }
  cluster_arrive();                           // the wait comes before a CTA first signals its peer
  if (warp == 1) alloc2(holder, kTmemCols);
  if (warp == 2 && lane < a.n) {
    const PairProb &b = a.p[lane];
    prefetch_map(&b.ta[0]);
    prefetch_map(&b.tb[0]);
    if (b.kb[1]) prefetch_map(&b.ta[1]);
    if (b.kb[1] || kDual) prefetch_map(&b.tb[1]);
    if (EPI == kGluBwd || EPI == kGluBwdLong) prefetch_map(&a.tw);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *holder;
  fb::pdl_enter();
  cluster_wait();                             // both CTAs' barriers exist

  const int total = a.tile0[a.n];
  const int first = blockIdx.x >> 1, step = gridDim.x >> 1;
  int32_t *err = a.err;

  if (warp == 0) {
    const bool one = elect_one();
    int s = 0;
    uint32_t turn = 0;                        // turns of the ring so far
    bool stop = false;
    for (int t = first; t < total && !stop; t += step) {
      const Tile q = tile_at<EPI>(a, t);
      const PairProb &b = a.p[EPI == kStore ? q.p : 0];
      const int m0 = q.m * 256 + (int)rank * kHalfM, kb0 = b.kb[0];
      const bool amn = EPI == kStore && b.a_mn, bmn_ = EPI == kStore && b.b_mn;
      const int bn_ = P == 3 ? 128 : (EPI == kStore ? b.bn : 256);
      for (int j = q.k0; j < q.k1; ++j) {
        const int p = j >= kb0 ? 1 : 0, jj = j - (p ? kb0 : 0);
        const bool dh = (EPI == kGluBwd && p == 0) || (EPI == kGluBwdLong && p == 1);
        const int bn = dh ? 128 : bn_;
        const bool bmn = dh || bmn_;
        const CUtensorMap *ma = &b.ta[p], *mb = dh ? &a.tw : &b.tb[kDual ? rank : p];
        const int n0 = kDual && !dh ? q.n * 128 : q.n * bn + (int)rank * (bn / 2);
#pragma unroll 1
        for (int k = 0; k < P; ++k) {
          if (turn > 0 && !wait(empty + s, (turn - 1) & 1, abort_flag, err)) {
            stop = true;
            break;
          }
          if (one) {
            const int z = (3 - k) % 3;        // planes 0, 2, 1: the order the products need them in
            const uint32_t full_at = leader_addr(full + s);
            uint8_t *sa = sA(s), *sb = sB(s);
            if (rank == 0) mbar_expect_tx(full + s, 2u * (uint32_t)(kABytes + bn / 2 * BK * 2));
            auto load = [&](void *dst, const CUtensorMap *map, int x, int y) {
              if (P == 1) load2(dst, map, full_at, x, y);
              else load3(dst, map, full_at, x, y, z);
            };
            if (amn) {
              load(sa, ma, m0, BK * jj);
              load(sa + kBox, ma, m0 + 64, BK * jj);
            } else {
              load(sa, ma, b.ax[p] + BK * jj, m0);
            }
            if (bmn) {
              load(sb, mb, n0, BK * jj);
              if (bn == 256) load(sb + kBox, mb, n0 + 64, BK * jj);
            } else {
              load(sb, mb, BK * jj, n0);
            }
          }
          __syncwarp();
          if (++s == kStages) s = 0, ++turn;
        }
        if (stop) break;
      }
    }
    // the MMAs have read every stage (and their arrivals reached this CTA) before it leaves
    for (int k = 0; k < kStages && !stop; ++k) {
      if (turn > 0 && !wait(empty + s, (turn - 1) & 1, abort_flag, err)) stop = true;
      if (++s == kStages) s = 0, ++turn;
    }
  } else if (warp == 1) {
    if (rank == 0) {
      const bool one = elect_one();
      int s = 0;
      uint32_t turn = 0, it = 0;              // turns of the ring, accumulators used so far
      bool stop = false;
      for (int t = first; t < total && !stop; t += step) {
        const Tile q = tile_at<EPI>(a, t);
      const PairProb &b = a.p[EPI == kStore ? q.p : 0];
        const bool amn = EPI == kStore && b.a_mn, bmn_ = EPI == kStore && b.b_mn;
        const int bn = P == 3 ? 128 : (EPI == kStore ? b.bn : 256), kb0 = b.kb[0];
        const uint64_t ad0 = sdesc(smem_u32(smem), amn), adv_a = amn ? (2048 >> 4) : 2;
        for (int j = q.k0; j < q.k1; ++j) {
          const bool dh = (EPI == kGluBwd && j < kb0) || (EPI == kGluBwdLong && j >= kb0), bmn = dh || bmn_;
          const uint32_t idesc = dh ? idesc2(128, false, true) : idesc2(bn, amn, bmn);
          const uint64_t bd0 = sdesc(smem_u32(smem + kABytes), bmn), adv_b = bmn ? (2048 >> 4) : 2;
          // a new accumulator at the tile's start (kGluBwd: where g | u start), or for every slab (kGluBwdLong: and dh)
          constexpr int kSlab = slab_of<EPI>();
          const bool next = P == 3 || (EPI == kGluBwd ? j == kb0 : j == q.k0) || (EPI == kGluBwdLong && j == kb0) ||
                            (kSlab && !dh && (j & (kSlab - 1)) == 0);
          const bool fresh = next || (EPI == kGluBwd && j == q.k0);
          const uint32_t buf = it % kBufs, use = it / kBufs;
          if (next && use >= 1 && !wait(acce + buf, (use - 1) & 1, abort_flag, err)) {
            stop = true;
            break;
          }
          if (!wait(full + s, turn & 1, abort_flag, err)) {
            stop = true;
            break;
          }
          const bool last = P == 3 || j + 1 == q.k1 || (EPI == kGluBwdLong && j + 1 == kb0) ||
                            (kSlab && !dh && ((j + 1) & (kSlab - 1)) == 0);
          const uint32_t d = tmem + (EPI == kGluBwd && dh ? 256u + (it & 1) * 128u : buf * 256u);
          // one product of 64 k: A of stage sa, B of stage sb
          auto issue = [&](int sa, int sb, bool first) {
            const uint64_t ad = ad0 + (uint64_t)(sa * (kStageBytes >> 4)), bd = bd0 + (uint64_t)(sb * (kStageBytes >> 4));
#pragma unroll
            for (int kk = 0; kk < BK / 16; ++kk)
              mma2(d, ad + kk * adv_a, bd + kk * adv_b, idesc, (first && kk == 0) ? 0u : 1u);
          };
          if constexpr (P == 1) {
            tc_fence_after();
            if (one) {
              issue(s, s, fresh);
              commit2(empty + s);
              if (last) commit2(accf + buf);
            }
            __syncwarp();
            if (++s == kStages) s = 0, ++turn;
          } else {
            // the slab's planes 0, 2, 1 in stages s, s1, s2: products 20, 02, 11, 10, 01, 00, smallest first, each
            // stage freed after its last one
            const int s1 = s + 1 == kStages ? 0 : s + 1, s2 = s1 + 1 == kStages ? 0 : s1 + 1;
            const uint32_t t1 = turn + (s1 == 0 ? 1 : 0), t2 = t1 + (s2 == 0 ? 1 : 0);
            if (!wait(full + s1, t1 & 1, abort_flag, err)) {
              stop = true;
              break;
            }
            tc_fence_after();
            if (one) {
              issue(s1, s, true);
              issue(s, s1, false);
              commit2(empty + s1);
            }
            __syncwarp();
            if (!wait(full + s2, t2 & 1, abort_flag, err)) {
              stop = true;
              break;
            }
            tc_fence_after();
            if (one) {
              issue(s2, s2, false);
              issue(s2, s, false);
              issue(s, s2, false);
              commit2(empty + s2);
              issue(s, s, false);
              commit2(empty + s);
              commit2(accf + buf);
            }
            __syncwarp();
            s = s2 + 1 == kStages ? 0 : s2 + 1;
            turn = t2 + (s == 0 ? 1 : 0);
          }
          if (last) ++it;
        }
      }
    }
    __syncwarp();
  } else if (warp >= kWarpEpi0) {
    const int e = warp - kWarpEpi0, qd = warp & 3, half = kAlt ? e >> 2 & 1 : e >> 2;   // (kLseLong: the quarter)
    const uint32_t tlane = (uint32_t)(qd * 32) << 16;
    uint8_t *obuf = outs + e * out_bytes<EPI>();
    uint32_t it = 0;
    for (int t = first; t < total; t += step, ++it) {
      const Tile q = tile_at<EPI>(a, t);
      const PairProb &b = a.p[EPI == kStore ? q.p : 0];
      if constexpr (P == 3) {
        const int row = q.m * 256 + (int)rank * kHalfM + qd * 32;
        float acc[64];
#pragma unroll
        for (int i = 0; i < 64; ++i) acc[i] = 0.f;
        bool ok = true;
        const int slabs = q.k1 - q.k0;
        for (int k = 0; k < slabs && ok; ++k, ++it) {
          const int buf = it % kBufs;
          ok = __all_sync(0xffffffffu, wait(accf + buf, (it / kBufs) & 1, abort_flag, err) ? 1 : 0);
          if (!ok) break;
          tc_fence_after();
          const uint32_t tb = tmem + tlane + (uint32_t)(buf * 256 + half * 64);
#pragma unroll
          for (int c = 0; c < 64; c += 32) {
            uint32_t r[32];
            tmem_ld32_nowait(tb + c, r);
            tmem_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) acc[c + i] += __uint_as_float(r[i]);
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive_at(leader_addr(acce + buf));
        }
        --it;                                 // the loop header counts one
        if (!ok) break;
        const int col = q.n * 128 + half * 64;
        if constexpr (EPI == kLsePlanes) {
          if (row + lane < b.M)
            a.part[(int64_t)(row + lane) * (2 * b.nt) + 2 * q.n + half] = max_sum(acc, b.N - col);
        } else if constexpr (EPI == kProbPlanes) {
          const int i0 = row + lane;
          const int64_t tg = i0 < b.M ? a.target[i0] : -1;
          const bool live = tg >= 0 && tg < a.V;
          const float z = live ? a.lse[i0] : 0.f, d = live ? a.dloss[i0] : 0.f;
          const int64_t tc = live ? tg - a.v0 - col : -1;         // the target's column among these
#pragma unroll
          for (int i = 0; i < 64; ++i) {      // a held-out row is zeros whatever its logits are
            const float e = expf(acc[i] - z) - (tc == i ? 1.f : 0.f);
            acc[i] = live ? d * e : 0.f;
          }
          float fin = 0.f;
#pragma unroll
          for (int i = 0; i < 64; ++i) fin = fbplanes::probe(acc[i], fin);
          if (__all_sync(0xffffffffu, fin == 0.f)) send_planes<true>(a, acc, obuf, row, col, lane);
          else send_planes<false>(a, acc, obuf, row, col, lane);
        } else {
#pragma unroll
          for (int c = 0; c < 64; c += 32) {
            uint32_t r[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(acc[c + i]);
            if (lane == 0) store_wait<0>();
            __syncwarp();
            stage_row(obuf, lane, r);
            send<true>(b, &b.tc, obuf, q.ybase, row, col + c, lane);
            __syncwarp();
          }
        }
        continue;
      }
      if constexpr (EPI == kLseLong) {
        // kLse for more than kLseSlab stages: the tensor cores' accumulation truncates (6e-8 of the logit a stage,
        // all one way) and a loss is fp32, so tensor memory sums kLseSlab stages at a time and registers the rest.
        float v[64];
        const int row = q.m * 256 + (int)rank * kHalfM + qd * 32, c0 = half * 64, left = b.N - (q.n * 256 + c0);
        bool ok = true;
        for (int j = q.k0; j < q.k1; j += kLseSlab, ++it) {
          const int buf = it % kBufs;
          ok = __all_sync(0xffffffffu, wait(accf + buf, (it / kBufs) & 1, abort_flag, err) ? 1 : 0);
          if (!ok) break;
          tc_fence_after();
          const uint32_t tb = tmem + tlane + (uint32_t)(buf * 256 + c0);
#pragma unroll
          for (int c = 0; c < 64; c += 32) {
            uint32_t r[32];
            tmem_ld32_nowait(tb + c, r);
            tmem_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) v[c + i] = j == q.k0 ? __uint_as_float(r[i]) : v[c + i] + __uint_as_float(r[i]);
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive_at(leader_addr(acce + buf));
        }
        --it;                                 // the loop header counts one
        if (!ok) break;
        if (row + lane < b.M) a.part[(int64_t)(row + lane) * (4 * b.nt) + 4 * q.n + half] = max_sum(v, left);
        continue;
      }
      if constexpr (EPI == kGluBwdLong) {
        // g and u of 64 columns, slab by slab, then dh: relu'(g) turns with the sign of g, so g is summed like fp32.
        // (Tensor memory alone, whose additions truncate, turned ten signs of 6,330 x 6,112 at width 2,306, fp32 two.)
        float g[64], u[64];
#pragma unroll
        for (int i = 0; i < 64; ++i) g[i] = u[i] = 0.f;
        bool ok = true;
        auto take = [&]() {
          const int at = it % kBufs;
          ok = __all_sync(0xffffffffu, wait(accf + at, (it / kBufs) & 1, abort_flag, err) ? 1 : 0);
          if (ok) tc_fence_after();
          return tmem + tlane + (uint32_t)(at * 256 + half * 64);
        };
        auto give = [&]() {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive_at(leader_addr(acce + it % kBufs));
          ++it;
        };
        for (int j = 0; j < b.kb[0]; j += kGluSlab) {
          const uint32_t at = take();
          if (!ok) break;
#pragma unroll
          for (int c = 0; c < 128; c += 16) {
            uint32_t r[16];
            tmem_ld16_nowait(at + (c < 64 ? c : 64 + c), r);
            tmem_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              float &s = c < 64 ? g[(c + i) & 63] : u[(c + i) & 63];
              s += __uint_as_float(r[i]);
            }
          }
          give();
        }
        if (!ok) break;
        const uint32_t at = take();
        if (!ok) break;
        const int row = q.m * 256 + (int)rank * kHalfM + qd * 32, col = q.n * 128 + half * 64;
        if (lane == 0) store_wait<0>();       // the tile before has left the buffers
        __syncwarp();
#pragma unroll
        for (int c = 0; c < 64; c += 16) {
          uint32_t d[16];
          tmem_ld16_nowait(at + c, d);
          tmem_wait();
#pragma unroll
          for (int k = 0; k < 16; k += 8) {   // 8 columns: one 16-byte piece of the row (stage_row)
            uint32_t w[3][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float h[2], dg[2], du[2];
#pragma unroll
              for (int o = 0; o < 2; ++o) {
                const float dv = __uint_as_float(d[k + 2 * i + o]), uv = u[c + k + 2 * i + o];
                const float2 f = fbact::act_fast<kRelu>(g[c + k + 2 * i + o]);
                h[o] = f.x * uv;
                dg[o] = dv * uv * f.y;
                du[o] = dv * f.x;
              }
              w[0][i] = pack(h[0], h[1]);
              w[1][i] = pack(dg[0], dg[1]);
              w[2][i] = pack(du[0], du[1]);
            }
#pragma unroll
            for (int o = 0; o < 3; ++o)
              *reinterpret_cast<uint4 *>(obuf + o * kStageOut + lane * 128 + ((((c + k) / 8) ^ (lane & 7)) << 4)) =
                  make_uint4(w[o][0], w[o][1], w[o][2], w[o][3]);
          }
        }
        give();
        --it;                                 // the loop header counts one
        fence_async_smem();
        __syncwarp();
        if (lane == 0) {
          if (row < b.M && col < b.N)
#pragma unroll
            for (int o = 0; o < 3; ++o) store_tile(o ? &a.tc2[o - 1] : &b.tc, obuf + o * kStageOut, col, row);
          store_commit();
        }
        continue;
      }
      const int buf = it % kBufs;
      if (kAlt && buf != e >> 3) continue;
      if (!__all_sync(0xffffffffu, wait(accf + buf, (it / kBufs) & 1, abort_flag, err) ? 1 : 0)) break;
      tc_fence_after();
      const uint32_t tb = tmem + tlane + (uint32_t)(buf * 256);
      const int row = q.m * 256 + (int)rank * kHalfM + qd * 32;   // this warp's first row
      if constexpr (EPI == kGluFwd || EPI == kGluBwd) {
        constexpr bool bwd = EPI == kGluBwd;
        const uint32_t td = tb + 256 + (it & 1) * 128;
#pragma unroll 1
        for (int which = 0; which < 2; ++which) {
          const int c = half * 64 + 32 * which, col = q.n * 128 + half * 64;
          if (a.act == kSilu) glu_block<kSilu, bwd>(a, tb, td, c, which, obuf, row, col, lane);
          else if (a.act == kGelu) glu_block<kGelu, bwd>(a, tb, td, c, which, obuf, row, col, lane);
          else glu_block<kRelu, bwd>(a, tb, td, c, which, obuf, row, col, lane);
        }
      } else if constexpr (EPI == kStore) {
        const int w0 = half * (b.bn / 2), w1 = w0 + b.bn / 2, n0 = q.n * b.bn;
        if (b.f32) {
#pragma unroll 1
          for (int c = w0; c < w1; c += 32) {
            uint32_t r[32];
            tmem_ld32_nowait(tb + c, r);
            tmem_wait();
            if (lane == 0) store_wait<0>();
            __syncwarp();
            stage_row(obuf, lane, r);
            send<true>(b, &b.tc, obuf, q.ybase, row, n0 + c, lane);
            __syncwarp();
          }
        } else {
#pragma unroll 1
          for (int c = w0; c < w1; c += 64) {
            uint32_t r0[32], r1[32], w[32];
            tmem_ld32_nowait(tb + c, r0);
            tmem_ld32_nowait(tb + c + 32, r1);
            tmem_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              w[i] = pack(__uint_as_float(r0[2 * i]), __uint_as_float(r0[2 * i + 1]));
              w[16 + i] = pack(__uint_as_float(r1[2 * i]), __uint_as_float(r1[2 * i + 1]));
            }
            if (lane == 0) store_wait<0>();
            __syncwarp();
            stage_row(obuf, lane, w);
            send<false>(b, &b.tc, obuf, q.ybase, row, n0 + c, lane);
            __syncwarp();
          }
        }
      } else if constexpr (EPI == kLse) {
        // maximum and sum of exp2 of this lane's row over its half of the tile's columns
        constexpr float kLog2e = 1.44269504088896340736f;
        float m = -INFINITY, s = 0.f;
#pragma unroll 1
        for (int c = half * 128; c < half * 128 + 128; c += 32) {
          const int left = b.N - (q.n * 256 + c);
          uint32_t r[32];
          tmem_ld32_nowait(tb + c, r);
          tmem_wait();
          if (left < 32) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (i >= left) r[i] = 0xFF800000u;                  // -inf: past the table
          }
          float cm = __uint_as_float(r[0]);
#pragma unroll
          for (int i = 1; i < 32; ++i) cm = fmaxf(cm, __uint_as_float(r[i]));
          const float nm = fmaxf(m, cm * kLog2e);
          // nothing but -inf so far: subtract 0, so that exp2 gives zeros (and NaN stays NaN)
          const float base = nm == -INFINITY ? 0.f : nm;
          s *= ex2(m - base);
          float s0 = 0.f, s1 = 0.f;
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            s0 += ex2(fmaf(__uint_as_float(r[i]), kLog2e, -base));
            s1 += ex2(fmaf(__uint_as_float(r[i + 1]), kLog2e, -base));
          }
          s += s0 + s1;
          m = nm;
        }
        if (row + lane < b.M) a.part[(int64_t)(row + lane) * (2 * b.nt) + 2 * q.n + half] = make_float2(m, s);
      } else if constexpr (EPI == kProb || EPI == kProbTwo) {
        constexpr float kLog2e = 1.44269504088896340736f;
        const int i0 = row + lane;
        const int64_t tg = i0 < b.M ? a.target[i0] : -1;
        const bool live = tg >= 0 && tg < a.V;
        const float z = live ? a.lse[i0] * kLog2e : 0.f, d = live ? a.dloss[i0] : 0.f;
        // G is rounded to bf16 as h, dg, du are (glu_block): dh and dw 0.0024 off in the 2-norm, 0.0017 with G in fp32
        // (4,000 x 100, 16,700 nodes); kProbTwo keeps what the rounding leaves as a second bf16 part
        const uint32_t mask = live ? 0xFFFFFFFFu : 0u;            // a held-out row is zeros whatever its logits are
        const int64_t tc = live ? tg - a.v0 : -1;                 // the target's column of this piece
#pragma unroll 1
        for (int c64 = half * 128; c64 < half * 128 + 128; c64 += 64) {
#pragma unroll
          for (int c = 0; c < 64; c += 32) {
            const int col = q.n * 256 + c64 + c;
            uint32_t r[32], w[16];
            tmem_ld32_nowait(tb + c64 + c, r);
            tmem_wait();
            const int hit = (tc >= col && tc < col + 32) ? (int)(tc - col) : -1;
#pragma unroll
            for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(ex2(fmaf(__uint_as_float(r[i]), kLog2e, -z)));
            if (__any_sync(0xffffffffu, hit >= 0)) {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (hit == i) r[i] = __float_as_uint(__uint_as_float(r[i]) - 1.f);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float v0 = __uint_as_float(r[2 * i]) * d, v1 = __uint_as_float(r[2 * i + 1]) * d;
              w[i] = pack(v0, v1) & mask;
              if (EPI == kProbTwo)            // what the rounding left
                r[i] = pack(v0 - __uint_as_float(w[i] << 16), v1 - __uint_as_float(w[i] & 0xFFFF0000u)) & mask;
            }
            if (c == 0) {
              if (lane == 0) store_wait<0>(); // the block before has left the buffer
              __syncwarp();
            }
            stage_half(obuf, lane, c / 32, w);
            if constexpr (EPI == kProbTwo) {
#pragma unroll
              for (int i = 0; i < 16; ++i) w[i] = r[i];
              stage_half(obuf + kStageOut, lane, c / 32, w);
            }
          }
          send<false>(b, &b.tc, obuf, 0, row, q.n * 256 + c64, lane);
          if (EPI == kProbTwo) send<false>(b, &a.tc2[0], obuf + kStageOut, 0, row, q.n * 256 + c64, lane);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_at(leader_addr(acce + buf));
    }
    if (lane == 0) store_wait<0>();
    __syncwarp();
  }
  __syncwarp();
  if (*abort_flag) {                          // copies in flight land before the shared memory goes away
    const long long t0 = clock64();
    while (clock64() - t0 < 4000000) {
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_arrive();
  cluster_wait();                             // neither CTA leaves while the other may still reach into it
  if (warp == 1) dealloc2(tmem, kTmemCols);
}

// ---- host ----------------------------------------------------------------------------------------
// A bf16 (or fp32: f32) matrix in boxes of 128-byte rows x box_rows, 128-byte swizzle.
inline int make_map(CUtensorMap *m, const void *base, int64_t rows, int64_t cols, int64_t ld, int box_rows,
                    bool f32 = false) {
  EncodeTiledFn enc = encode_fn();
  if (!enc) return fb::set_error(FB_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  const int es = f32 ? 4 : 2;
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)(ld * es)};
  cuuint32_t box[2] = {(cuuint32_t)(128 / es), (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  const CUresult r = enc(m, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
                         const_cast<void *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fb::set_error(FB_ERR_ARG, "tensor map rejected (alignment or stride)");
  return FB_OK;
}

// The same for the three planes of a matrix, `rows` rows each.
inline int make_map3(CUtensorMap *m, const void *base, int64_t rows, int64_t cols, int64_t ld, int64_t plane,
                     int box_rows) {
  EncodeTiledFn enc = encode_fn();
  if (!enc) return fb::set_error(FB_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, 3};
  cuuint64_t strides[2] = {(cuuint64_t)(ld * 2), (cuuint64_t)(plane * 2)};
  cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(base), dims, strides, box, estr,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fb::set_error(FB_ERR_ARG, "tensor map rejected (alignment or stride)");
  return FB_OK;
}

// A product's operand in boxes of box_rows rows: bf16, or fp32 as planes.
inline int operand_map(CUtensorMap *m, const fbh::Mat &x, int64_t rows, int64_t cols, int box_rows) {
  return x.plane ? make_map3(m, x.p, rows, cols, x.ld, x.plane, box_rows) : make_map(m, x.p, rows, cols, x.ld, box_rows);
}

inline bool map_ok(const void *p, int64_t ld, int es) {
  return ((reinterpret_cast<uintptr_t>(p) | (uintptr_t)(ld * es)) & 15u) == 0;
}

// Clusters of two that fit on the device at once.
template <auto kernel> int pair_slots(int smem, int threads) {
  static int slots[64] = {0};
  int dev = 0;
  cudaGetDevice(&dev);
  int &s = slots[dev & 63];
  if (!s) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return 0;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(num_sms() / 2 * 2);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 2;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
      cudaGetLastError();
      n = 0;
    }
    s = n > 0 ? n : num_sms() / 2;
  }
  return s;
}

template <int EPI, int P = 1> int launch_pair(const PairArgs &a, cudaStream_t stream) {
  constexpr auto k = k_pair<EPI, P>;
  constexpr int smem = smem_bytes<EPI, P>();
  const int slots = pair_slots<k>(smem, threads_of<EPI>());
  if (!slots) return fb::cuda_error(cudaGetLastError(), "k_pair shared memory");
  const int tiles = a.tile0[a.n];
  if (tiles == 0) return FB_OK;
  FB_TRY_CUDA(fb::launch(k, 2 * (unsigned)std::min(tiles, slots), threads_of<EPI>(), smem, stream, a));
  FB_LAUNCHED("k_pair");
  return FB_OK;
}

inline int tiles_of(int64_t n, int t) { return (int)((n + t - 1) / t); }

// A launch of one product of M x N over kb stages, 256-column tiles of `tile` result columns, unsplit.
inline void one_product(PairArgs &a, int64_t M, int64_t N, int tile, int kb, int terms) {
  std::memset(&a, 0, sizeof(a));
  PairProb &b = a.p[0];
  a.n = 1;
  b.bn = 256;
  b.mt = tiles_of(M, 256);
  b.nt = tiles_of(N, tile);
  b.splits = 1;
  b.kb[0] = kb;
  b.kb[1] = terms > 1 ? kb : 0;
  b.kper = terms * kb;
  b.M = (int)M;
  b.N = (int)N;
  b.has_tc = 1;
  a.tile0[1] = b.mt * b.nt;
  a.err = err_word();
}

}  // namespace fbpair
