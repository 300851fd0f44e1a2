// chunk_tc.cuh - attention of a chunk on the 5th-generation tensor cores
// (tcgen05.mma kind::f16, accumulators in tensor memory), for fp16 and bf16
// queries over every cache format.
//
// Operands are fp16. A query row is scaled by a power of two that brings its
// largest magnitude to [2^14, 2^15), so bf16's range fits and its 8 bits are
// kept; the power goes into the row's softmax scale. f16 cache rows are taken
// as they are; int8 and int4 codes become rn(zero + scale * code) with one
// rounding. Softmax weights are rounded to fp16, their sum is kept in fp32 of
// the unrounded ones. Both products accumulate in fp32.
//
// Warp groups (of 128 threads; one block per SM):
//   0, 1   softmax, thread = row of a 128-row tile. TWO: each group has its own
//          row tile and both take every step of 128 tokens; else both have the
//          same rows and take steps in turn, each with its own output, as two
//          splits. Either way one group's softmax runs while the tensor cores
//          work for the other;
//   2, 3   quantized caches: converters, one for K and one for V. Raw half steps
//          (64 tokens) land in a ring of their own and become fp16 tiles of 128
//          tokens x 64 channels with the 128-byte swizzle. f16 caches: TMA writes
//          those tiles itself, and group 2 only clears what must not be seen;
//   last   two warps issue the MMAs (one lane each), one per softmax group, so that
//          neither waits on the other's weights: S = Q K^T into tensor memory, O += P V
//          with P read from tensor memory, where the softmax group writes it over its
//          scores, and V read MN-major. The other two are the producers of K and of V:
//          TMA boxes per page, none for tokens that nobody sees or for a block
//          without a page.
// A row's weights are taken against a reference 7 below its running maximum (log2),
// so that the largest is about 2^7: fp16 then holds weights down to 2^-32 of it, where
// against the maximum itself those below 2^-25 would be lost, and many small ones
// can outweigh one large one whose value is small. The reference is raised only when
// 64 weights add up to more than 2^15 (weights up to that fit fp16, and their sum
// fp32), so the output in tensor memory is rescaled rarely, a step's scores are
// read once, and their maximum is not needed before.
// Waits are bounded in time; tensor memory is released before exit.
#pragma once

#include "chunk.cuh"
#include "tc.cuh"

#include <cuda.h>

#include <cstddef>

namespace kvfb {

// A wait of chunk_tc_kernel ran out of time (reported as bit 0 of
// kvf_b200_device_errors).
__device__ unsigned g_kvfb_chunk_error;

namespace {

constexpr int kTcRows = 128;    // rows of a tile
constexpr int kTcStep = 128;    // tokens of a step
constexpr int kTcHalf = 64;     // tokens of a raw half step
constexpr float kTcTop = 7.f;          // log2 of a row's largest weight when its reference is raised
constexpr float kTcLazySum = 32768.f;  // most that 64 weights may add up to before that
// A reference of 2^24 and more (log2) is rounded so coarsely that the largest weight,
// 2^7 above it but for that, may come out as infinity or 0: from there on a row's
// reference is its largest score as it is, taken off before the scale.
constexpr float kTcFar = 16777216.f;

__host__ __device__ constexpr int cache_row_bytes(int fmt, int d) {
  return fmt == KVF_FMT_F16 ? 2 * d : fmt == KVF_FMT_INT8 ? d : d / 2;
}

// Shared memory of a variant: query tiles, then rings of fp16 tiles for K and
// for V, then rings of raw half steps with their metadata, as deep as fits.
template <int FMT, int D, bool TWO> struct TcLayout {
  static constexpr bool RAW = FMT != KVF_FMT_F16;
  static constexpr int GROUPS = RAW ? 5 : 4;                 // warp groups
  static constexpr int THREADS = 128 * GROUPS;
  // Registers per thread after the start: the block is launched with 96 (five
  // groups) or 128 (four), and the groups' shares add up to no more than that.
  static constexpr int SOFT_REGS = RAW ? 136 : 168, CONV_REGS = 72, LAST_REGS = RAW ? 64 : 96;
  static_assert(2 * SOFT_REGS + (RAW ? 2 : 1) * CONV_REGS + LAST_REGS <= (RAW ? 96 * 5 : 128 * 4), "registers");
  static constexpr uint32_t TILE = kTcStep * D * 2;
  static constexpr uint32_t QB = (TWO ? 2u : 1u) * TILE;
  // fp16 tiles per operand. Without TWO a tile belongs to one issuer, which must
  // meet every phase of its slots' barriers: an even number.
  static constexpr int SLOTS = RAW || TWO || D == 128 ? 2 : 4;
  static constexpr uint32_t RAWB = RAW ? kTcHalf * (uint32_t)cache_row_bytes(FMT, D) : 0u;
  static constexpr uint32_t METAB = RAW ? kTcHalf * (FMT == KVF_FMT_INT8 ? 8u : 16u) : 0u;
  static constexpr uint32_t FREE = 232448u - 1024u - QB - 2u * SLOTS * TILE;
  static constexpr int FIT = RAW ? (int)(FREE / (2u * (RAWB + METAB))) : 0;
  static constexpr int RSLOTS = FIT > 8 ? 8 : FIT;           // raw half steps per operand
  static constexpr uint32_t OFF_RING = QB;
  static constexpr uint32_t OFF_RAW = OFF_RING + 2u * SLOTS * TILE;
  static constexpr uint32_t OFF_META = OFF_RAW + 2u * RSLOTS * RAWB;
  static constexpr uint32_t OFF_MISC = OFF_META + 2u * RSLOTS * METAB;
  static constexpr uint32_t BYTES = OFF_MISC + 1024u;
  static_assert(!RAW || RSLOTS >= 2, "two raw half steps per operand");
  static_assert(BYTES <= 232448u, "shared memory");
};

struct TcShared {
  // Barriers, in the order of tc_bar_count.
  uint64_t kfull[4], vfull[4];                        // a tile is there
  uint64_t kempty[4], vempty[4];                      // its slot is free
  uint64_t sfull[2][2], pready[2][2], ofull[2][2];    // per group and half step: scores, weights, output
  uint64_t vraw[4], vfixed[4];                        // f16 V tiles on their way through group 2
  uint64_t qready, done;
  uint64_t rfull[2][8], rempty[2][8];                 // raw half steps of K, of V
  uint8_t qexp[2 * kTcRows];                          // 14 + exponent (biased) of the power of two a row was divided by
  uint32_t tmem;
  int abort_flag;
  int odd;            // a masked V tile held an infinity or NaN, taken as 0
};
constexpr int kTcBars = 16 + 12 + 8 + 2 + 32;
static_assert(offsetof(TcShared, qexp) == 8 * kTcBars, "barriers");

// Arrivals that complete a phase of barrier i of TcShared.
template <bool RAW, bool TWO> __device__ __forceinline__ uint32_t tc_bar_count(int i) {
  return i < 8    ? (RAW ? 4u : 1u)   // kfull, vfull: four converter warps, or TMA
         : i < 16 ? (TWO ? 2u : 1u)   // kempty, vempty: each issuer that uses the tile
         : i < 20 ? 1u                // sfull
         : i < 24 ? 4u                // pready: a group's warps
         : i < 28 ? 1u                // ofull
         : i < 32 ? 1u                // vraw
         : i < 36 ? 4u                // vfixed
         : i < 37 ? (TWO ? 8u : 4u)   // qready: the warps that load queries
         : i < 38 ? 2u                // done: both issuers
         : i < 54 ? 1u                // rfull: the boxes' bytes
                  : 4u;               // rempty: converter warps
}
static_assert(sizeof(TcShared) <= 1024, "misc area");

template <int N> __device__ __forceinline__ void regs_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N> __device__ __forceinline__ void regs_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// Waits (bounded) for a phase of a barrier; every lane of a warp may call it.
__device__ __forceinline__ bool tc_wait(uint32_t bar, uint32_t parity, volatile int *abort_flag) {
  if (ptx::mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = ptx::globaltimer_ns();
  for (uint32_t it = 1;; ++it) {
    if (ptx::mbar_try_wait(bar, parity)) return true;
    if ((it & 63u) == 0 && (*abort_flag || ptx::globaltimer_ns() - t0 > 2000000000ull)) return false;
  }
}
__device__ __forceinline__ bool tc_wait_warp(uint32_t bar, uint32_t parity, volatile int *abort_flag) {
  return __all_sync(0xffffffffu, tc_wait(bar, parity, abort_flag));
}

__device__ __forceinline__ float2 fma2f(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ float2 add2f(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "add.rn.f32x2 w, x, y;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// Weights 2^(s c - m) of 32 scores as fp16 pairs, and their sum; 0 for tokens
// from `seen` on. (Computing one pair in four, or in eight, with a polynomial on
// the FMA pipe instead of the special function unit was measured: 4096 tokens
// over 32768 int8 tokens 2.03 and 2.00 ms against 1.96, f16 prompts the same. The
// FMA pipe, which the converters use too, is the busier one.)
template <bool MASKED>
__device__ __forceinline__ float weigh(const uint32_t (&s)[32], float m, float c, int at, int seen, uint32_t *p) {
  const float ref = m == -INFINITY ? 0.f : m;
  const float2 c2 = make_float2(c, c), m2 = make_float2(-ref, -ref);
  float2 sum0 = make_float2(0.f, 0.f), sum1 = sum0;
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const float2 x = fma2f(make_float2(__uint_as_float(s[2 * k]), __uint_as_float(s[2 * k + 1])), c2, m2);
    float2 e = make_float2(ex2(x.x), ex2(x.y));
    if (MASKED) {
      e.x = at + 2 * k < seen ? e.x : 0.f;
      e.y = at + 2 * k + 1 < seen ? e.y : 0.f;
    }
    if (k & 1)
      sum1 = add2f(sum1, e);
    else
      sum0 = add2f(sum0, e);
    p[k] = narrow2<KVF_DT_F16>(e.x, e.y);
  }
  return (sum0.x + sum0.y) + (sum1.x + sum1.y);
}
__device__ __forceinline__ bool odd_f16x2(uint32_t w) {
  return (w & 0x7C00u) == 0x7C00u || (w & 0x7C000000u) == 0x7C000000u;
}
// A word with each infinity or NaN of it replaced by zero.
__device__ __forceinline__ uint32_t even_f16x2(uint32_t w) {
  if ((w & 0x7C00u) == 0x7C00u) w &= 0xffff0000u;
  if ((w & 0x7C000000u) == 0x7C000000u) w &= 0x0000ffffu;
  return w;
}

template <int FMT, int DT, int D, bool TWO>
__global__ void __launch_bounds__(TcLayout<FMT, D, TWO>::THREADS, 1)
chunk_tc_kernel(const ChunkArgs a, const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv) {
  using L = TcLayout<FMT, D, TWO>;
  constexpr int KB = D / 64;                       // 64-channel blocks of a tile
  constexpr uint32_t TILE = L::TILE;
  constexpr uint32_t BLK = TILE / KB;              // 128 rows x 128 bytes
  constexpr int RB = cache_row_bytes(FMT, D);
  constexpr int SLOTS = L::SLOTS, RSLOTS = L::RSLOTS;
  constexpr uint32_t S_COL = 0, O_COL = 256;       // tensor-memory columns: scores (2 x 128), outputs (2 x D)
  constexpr int LAST = 4 * (L::GROUPS - 1);        // first warp of the last group: MMA issue, then the producers

  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sbase = ptx::smem_u32(smem);
  const uint32_t sq = sbase, skr = sbase + L::OFF_RING, svr = skr + SLOTS * TILE;
  TcShared &sh = *reinterpret_cast<TcShared *>(smem + L::OFF_MISC);
  volatile int *abort_flag = &sh.abort_flag;
  auto bar = [&](const uint64_t *b) -> uint32_t { return ptx::smem_u32(b); };
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // known to be the same in all lanes

  ChunkWork w;
  const int nsplit = TWO ? a.splits : a.splits / 2;
  if (!chunk_work(a, nsplit, TWO ? 2 * kTcRows : kTcRows, kTcStep, w)) return;
  const int n = (w.t1 - w.t0 + kTcStep - 1) / kTcStep;

  // Steps of each softmax group.
  auto group_steps = [&](int g) -> int {
    if (!TWO) return (n + 1 - g) / 2;
    const int rows = min(w.rows - g * kTcRows, kTcRows);
    const int seen = rows > 0 ? chunk_seen(a, w, g * kTcRows + rows - 1) : 0;
    return seen > w.t0 ? min(n, (seen - w.t0 + kTcStep - 1) / kTcStep) : 0;
  };

  // First step that some row of the block does not see whole. From there on V
  // tiles must not carry infinities or NaN into such rows (0 * inf): zeros stand
  // in, and the rows that do see them get them at the end.
  const int first_masked = w.seen0 > w.t0 ? (w.seen0 - w.t0) / kTcStep : 0;

  if (tid < kTcBars) ptx::mbar_init(bar(&sh.kfull[0]) + 8u * tid, tc_bar_count<L::RAW, TWO>(tid));
  if (tid == 0) {
    sh.abort_flag = 0;
    sh.odd = 0;
  }
  ptx::fence_barrier_init();
  if (warp == LAST) {
    tc::alloc(ptx::smem_u32(&sh.tmem), 512u);
    tc::relinquish();
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tbase = sh.tmem;
  const int grp = warp >> 2;              // softmax group (warps 0-7)
  // Each group executes one setmaxnreg, all four warps the same one.
  if (warp < 8) {
    // ------------------------------------------------------------- softmax
    regs_up<L::SOFT_REGS>();
    const int row = (TWO ? grp * kTcRows : 0) + (tid & 127);
    const bool live = row < w.rows;

    // Query rows, scaled, into their tile: a warp takes its own 32 rows, each by
    // D / 8 lanes, all loads in flight at once. A bf16 row is scaled by 2^(14 -
    // exponent of its largest magnitude), or the largest power that fp32 holds for
    // rows below 2^-100; by 1 if that is zero, infinite or NaN.
    if (TWO || grp == 0) {
      constexpr int LPR = D / 8, RPW = 32 / LPR, N = 32 / RPW;
      const int li = lane % LPR, r0 = 32 * (warp & 3) + lane / LPR;
      uint4 raw[N];
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const int rt = r0 + k * RPW, rr = (TWO ? grp * kTcRows : 0) + rt;
        raw[k] = make_uint4(0u, 0u, 0u, 0u);
        if (rr < w.rows) {
          const uint8_t *src = chunk_row(a.q, a, w, rr) + 16 * li;
          if (a.q.vec) {
            raw[k] = __ldg(reinterpret_cast<const uint4 *>(src));
          } else {
            const uint16_t *e = reinterpret_cast<const uint16_t *>(src);
            raw[k] = make_uint4(e[0] | (uint32_t)e[1] << 16, e[2] | (uint32_t)e[3] << 16, e[4] | (uint32_t)e[5] << 16,
                                e[6] | (uint32_t)e[7] << 16);
          }
        }
      }
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const int rt = r0 + k * RPW;
        uint32_t x[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
        int ex = 127 + 14;
        if (DT == KVF_DT_BF16) {
          // magnitudes order as integers; bf16 bits and fp32's upper half are the same
          uint32_t mx = 0u;
#pragma unroll
          for (int q = 0; q < 4; ++q) mx = max(mx, max(x[q] & 0x7fffu, (x[q] >> 16) & 0x7fffu));
#pragma unroll
          for (int off = 1; off < LPR; off <<= 1) mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, off));
          float f = 1.f;
          if (mx > 0u && mx < 0x7f80u) {
            ex = max((int)(mx >> 7), 27);
            f = __uint_as_float((uint32_t)(127 + 14 + 127 - ex) << 23);
          }
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float2 e = widen2<KVF_DT_BF16>(x[q]);
            x[q] = narrow2<KVF_DT_F16>(e.x * f, e.y * f);
          }
        }
        const uint32_t ad = sq + (TWO ? grp * TILE : 0u) + (li >> 3) * BLK + rt * 128u + ((uint32_t)((li ^ rt) & 7) << 4);
        asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(ad), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]) : "memory");
        if (li == 0) sh.qexp[(TWO ? grp * kTcRows : 0) + rt] = (uint8_t)ex;
      }
      ptx::fence_proxy_async_smem();
      __syncwarp();
      ptx::mbar_arrive_if(bar(&sh.qready), lane == 0);
    }
    bool ok = tc_wait_warp(bar(&sh.qready), 0u, abort_flag);  // without TWO group 1 has group 0's rows
    const float c = a.scale_log2 * __uint_as_float((uint32_t)(sh.qexp[row] - 14) << 23);  // softmax scale of the row
    // a lane without a row goes along (its query is zero); a warp without one only signs off
    const int seen = live ? chunk_seen(a, w, row) : 0x7fffffff;
    const bool idle = __all_sync(0xffffffffu, !live);
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t ts = tbase + lanes + S_COL + 128u * grp, to = tbase + lanes + O_COL + (uint32_t)(D * grp);
    const int steps = group_steps(grp);
    // Reference (log2) of the row's weights and their sum; where the reference is
    // past kTcFar it is the raw score `base`, and m is NaN so that every half is raised.
    float m = -INFINITY, l = 0.f, base = 0.f;
    bool early = false;
    uint32_t sa[32], sb[32];                // scores of the half at hand, or (early) of the next
    for (int j = 0; j < steps && ok; ++j) {
      const int t = w.t0 + (TWO ? j : 2 * j + grp) * kTcStep;
      // Half a step at a time (64 tokens), each half with scores, weights and
      // barriers of its own: while one half is weighed, the tensor cores take the
      // other's value product and its next scores. Whole steps and steps that some
      // row does not see to the end are weighed by code of their own: the
      // comparisons would cost the first a third of its instructions.
      const bool masked = __any_sync(0xffffffffu, t + kTcStep > seen);
      auto half = [&](int h) {
        const int at = t + 64 * h;
        const uint32_t tsh = ts + 64u * h;
        uint32_t p[32];
        if (!early) {
          tc::ld32(tsh, sa);
          tc::ld32(tsh + 32u, sb);
        }
        tc::wait_ld32(sa);
        tc::wait_ld32(sb);
        float sum;
        if (masked) {
          sum = weigh<true>(sa, m, c, at, seen, p);
          sum += weigh<true>(sb, m, c, at + 32, seen, p + 16);
        } else {
          sum = weigh<false>(sa, m, c, at, seen, p);
          sum += weigh<false>(sb, m, c, at + 32, seen, p + 16);
        }
        // Weights are taken against the reference as it stands; only where their
        // sum is past kTcLazySum is it raised, the output so far rescaled, and
        // the scores of the half read and weighed again. The warp goes along, but
        // a row that need not be raised keeps its reference and so its weights: its
        // output does not depend on the rows beside it.
        const bool raise = !(sum <= kTcLazySum) || (m == -INFINITY && at < seen);
        if (__any_sync(0xffffffffu, raise)) {
          // scores times the sign of the scale, and its magnitude
          const float ac = fabsf(c);
          const uint32_t flip = __float_as_uint(c) & 0x80000000u;
          float mx = -INFINITY;
#pragma unroll 1
          for (int u = 0; u < 4; ++u) {
            uint32_t s[16];
            tc::ld16(tsh + 16u * u, s);
            tc::wait_ld16(s);
#pragma unroll
            for (int k = 0; k < 16; ++k)
              if (at + 16 * u + k < seen) mx = fmaxf(mx, __uint_as_float(s[k] ^ flip));
          }
          float f = 1.f;
          if (raise && m == m) {
            const float mn = fmaxf(m, fmaf(mx, ac, -kTcTop));
            if (fabsf(mn) >= kTcFar && mn != -INFINITY) {
              f = exp2f(kTcTop - fmaf(mx, ac, -m));
              base = mx;
              m = NAN;
            } else {
              f = m == mn ? 1.f : exp2f(m - mn);
              m = mn;
            }
          } else if (raise) {
            const float top = fmaxf(base, mx);
            f = base == top ? 1.f : exp2f((base - top) * ac);
            base = top;
          }
          l *= f;
          if (2 * j + h > 0 && __any_sync(0xffffffffu, f != 1.f)) {
            // the half before this one; those before it were done when the scores came
            if (!tc_wait_warp(bar(&sh.ofull[grp][h ^ 1]), (uint32_t)((h ? j : j - 1) & 1), abort_flag)) {
              ok = false;
              return;
            }
            tc::fence_after();
#pragma unroll 1
            for (int u = 0; u < D / 16; ++u) {
              uint32_t o[16];
              tc::ld16(to + 16u * u, o);
              tc::wait_ld16(o);
#pragma unroll
              for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
              tc::st16(to + 16u * u, o);
            }
          }
          sum = 0.f;
          if (__any_sync(0xffffffffu, m != m)) {
            // rows with a raw reference: it is taken off where the scores lie
#pragma unroll 1
            for (int u = 0; u < 4; ++u) {
              uint32_t s[16];
              tc::ld16(tsh + 16u * u, s);
              tc::wait_ld16(s);
#pragma unroll
              for (int k = 0; k < 16; ++k)
                if (m != m) s[k] = __float_as_uint(__uint_as_float(s[k] ^ flip) - base);
              tc::st16(tsh + 16u * u, s);
            }
            tc::wait_st();
          }
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            uint32_t s[32];
            tc::ld32(tsh + 32u * u, s);
            tc::wait_ld32(s);
            sum += weigh<true>(s, m != m ? -kTcTop : m, m != m ? ac : c, at + 32 * u, seen, p + 16 * u);
          }
        }
        l += sum;
        // The next half's scores, if they are there: read while this half's weights are stored.
        const int nj = j + h, nh = h ^ 1;
        early = nj < steps && __all_sync(0xffffffffu, ptx::mbar_test_wait(bar(&sh.sfull[grp][nh]), (uint32_t)(nj & 1)));
        if (early) {
          tc::fence_after();
          tc::ld32(ts + 64u * nh, sa);
          tc::ld32(ts + 64u * nh + 32u, sb);
        }
        tc::st32(tsh, p);
        tc::wait_st();
        tc::fence_before();
      };
#pragma unroll 1
      for (int h = 0; h < 2; ++h) {
        if (!early && !tc_wait_warp(bar(&sh.sfull[grp][h]), (uint32_t)(j & 1), abort_flag)) {
          ok = false;
          break;
        }
        if (!idle) {
          tc::fence_after();
          half(h);
          if (!ok) break;
          __syncwarp();
        }
        ptx::mbar_arrive_if(bar(&sh.pready[grp][h]), lane == 0);
      }
      if (!ok) break;
    }
    if (ok && steps > 0 && !tc_wait_warp(bar(&sh.ofull[grp][1]), (uint32_t)((steps - 1) & 1), abort_flag)) ok = false;
    tc::fence_after();
    if (!ok && lane == 0) {
      atomicOr(&g_kvfb_chunk_error, 1u);
      *abort_flag = 1;
    }
    // ------------------------------------------------------------ epilogue
    const bool none = m == -INFINITY && l == 0.f;
    if (m != m) m = fmaf(base, fabsf(c), -kTcTop);
    const bool odd = *reinterpret_cast<volatile int *>(&sh.odd) != 0;
    const long long at = live ? chunk_index(a, w, row) : 0;
    const long long part = at * a.splits + (TWO ? w.split : 2 * w.split + grp);
    const float inv = none ? 0.f : 1.f / l;
    if (live) {
      if (a.splits > 1)
        *reinterpret_cast<float2 *>(a.part_ml + 2 * part) = make_float2(m, l);
      else if (a.lse)
        a.lse[at] = none ? -INFINITY : m + log2f(l);
    }
    // 32 columns at a time through shared memory that no MMA reads any more and no
    // copy will fill: the warp's part of the group's own query tile, or, where both
    // groups share one, of a K slot that only this group's tiles use. Threads have
    // rows, stores take whole rows.
    const uint32_t stage = (TWO ? sq : skr) + grp * TILE + (uint32_t)(warp & 3) * 4096u;
#pragma unroll 1
    for (int q = 0; q < D / 32; ++q) {
      uint32_t o[32];
      if (steps > 0) {
        tc::ld32(to + 32u * q, o);
        tc::wait_ld32(o);
      }
      if (none || steps == 0) {
#pragma unroll
        for (int k = 0; k < 32; ++k) o[k] = 0u;
      }
      if (odd && live && !none) {
        // what the masked tiles left out, for a row that sees it
        for (int t = w.t0 + first_masked * kTcStep; t < min(seen, w.t1); ++t) {
          if (!TWO && (((t - w.t0) / kTcStep) & 1) != grp) continue;
          const long long rw = a.cache.row(w.b, w.h, t);
          if (rw < 0) continue;
          for (int i = 0; i < 4; ++i) {
            float x[8];
            cache8<FMT, D>(a.v, a.vm, a, rw, 4 * q + i, x);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const float h = __half2float(__float2half_rn(x[k]));
              if (!(fabsf(h) < INFINITY)) {
#pragma unroll
                for (int u = 0; u < 4; ++u)
                  if (u == i) o[8 * u + k] = __float_as_uint(__uint_as_float(o[8 * u + k]) + h);
              }
            }
          }
        }
      }
      __syncwarp();
      if (a.splits > 1) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(stage + lane * 128u + ((uint32_t)((k ^ lane) & 7) << 4)),
                       "r"(o[4 * k]), "r"(o[4 * k + 1]), "r"(o[4 * k + 2]), "r"(o[4 * k + 3])
                       : "memory");
        __syncwarp();
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int rw = 4 * k + (lane >> 3), rr = row - lane + rw;  // eight lanes a row
          uint32_t x[4];
          asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                       : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3])
                       : "r"(stage + rw * 128u + ((uint32_t)((lane ^ rw) & 7) << 4)));
          if (rr < w.rows) {
            const long long pr = chunk_index(a, w, rr) * a.splits + (TWO ? w.split : 2 * w.split + grp);
            *reinterpret_cast<uint4 *>(a.part_o + pr * D + 32 * q + 4 * (lane & 7)) = make_uint4(x[0], x[1], x[2], x[3]);
          }
        }
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t x[4];
#pragma unroll
          for (int u = 0; u < 4; ++u)
            x[u] = narrow2<DT>(__uint_as_float(o[8 * k + 2 * u]) * inv, __uint_as_float(o[8 * k + 2 * u + 1]) * inv);
          asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(stage + lane * 64u + ((uint32_t)((k ^ (lane >> 1)) & 3) << 4)),
                       "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3])
                       : "memory");
        }
        __syncwarp();
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int rw = 8 * k + (lane >> 2), rr = row - lane + rw;  // four lanes a row
          uint32_t x[4];
          asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                       : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3])
                       : "r"(stage + rw * 64u + ((uint32_t)((lane ^ (rw >> 1)) & 3) << 4)));
          if (rr < w.rows) {
            uint8_t *out = chunk_row(a.out, a, w, rr) + 64 * q + 16 * (lane & 3);
            if (a.out.vec) {
              *reinterpret_cast<uint4 *>(out) = make_uint4(x[0], x[1], x[2], x[3]);
            } else {
              uint16_t *e = reinterpret_cast<uint16_t *>(out);
#pragma unroll
              for (int u = 0; u < 4; ++u) {
                e[2 * u] = (uint16_t)x[u];
                e[2 * u + 1] = (uint16_t)(x[u] >> 16);
              }
            }
          }
        }
      }
    }
    tc::fence_before();
  } else if (warp < LAST) {
    // ---------------------------------------------------------- converters
    regs_down<L::CONV_REGS>();
    const int lt = tid & 127;
    bool ok = true, odd = false;
    if constexpr (L::RAW) {
      constexpr int CPR = RB / 16;                 // 16-byte pieces of a raw row
      constexpr int RPP = 128 / CPR;               // rows that the group takes at a time
      constexpr int P16 = 2 * D / RB;              // 16-byte pieces of the tile per raw piece: 2 (int8), 4 (int4)
      const int op = (warp >> 2) - 2;              // 0: K, 1: V
      const int ch = lt % CPR, r0 = lt / CPR;
      const int gword = (ch * (16 * D / RB)) >> a.group_shift;  // metadata word of the piece
      const uint32_t ring = op ? svr : skr;
      // Metadata rows: a warp fetches those of the 16 rows that it converts itself,
      // one to a lane, RSLOTS halves ahead (cp.async into its own part of the slot's
      // area), so nobody else has to be told. The page of the half after is looked
      // up one half earlier. Row numbers fit 32 bits: fewer rows fit a GPU.
      constexpr int WR = 32 / CPR;                 // adjacent rows of a warp
      const bool paged = a.cache.paged != 0;
      const int bts = paged ? a.cache.bt_shift : 30, bmask = (1 << bts) - 1;
      const unsigned heads = (unsigned)a.cache.Hkv, hd = (unsigned)w.h;
      const unsigned pstep = paged ? heads << bts : heads * (unsigned)a.cache.n;
      const unsigned tstep = a.cache.head_major ? 1u : heads;
      const unsigned hoff = !a.cache.head_major ? hd : paged ? hd << bts : hd * (unsigned)a.cache.n;
      const int *table = paged ? a.cache.table + (long long)w.b * a.cache.max_blocks : nullptr;
      const uint32_t *mcache = op ? a.vm : a.km;
      const int mrow = lane < 16 ? (lane / WR) * RPP + (lt >> 5) * WR + lane % WR : 0;  // row of the half
      auto page_of = [&](int i) -> int {
        const int t = w.t0 + i * kTcHalf + mrow;
        if (i >= 2 * n || t >= w.t1) return -1;
        return paged ? __ldg(table + (t >> bts)) : w.b;
      };
      auto fetch_meta = [&](int i, int page) {     // half i into its slot
        if (i < 2 * n && lane < 16) {
          const int t = w.t0 + i * kTcHalf + mrow;
          const bool there = page >= 0;            // else zeros
          const unsigned row = (unsigned)page * pstep + (unsigned)(t & bmask) * tstep + hoff;
          const uint32_t *src = there ? mcache + (size_t)row * a.gpr : mcache;
          const uint32_t d = sbase + L::OFF_META + (uint32_t)(op * RSLOTS + i % RSLOTS) * L::METAB + (uint32_t)(mrow * a.gpr * 4);
          if (a.gpr == 1)
            ptx::cp_async_4_zfill(d, src, there ? 4u : 0u);
          else if (a.gpr == 2)
            ptx::cp_async_8_zfill(d, src, there ? 8u : 0u);
          else
            ptx::cp_async_16_zfill(d, src, there ? 16u : 0u);
        }
        ptx::cp_async_commit();
      };
      for (int i = 0; i < RSLOTS; ++i) fetch_meta(i, page_of(i));
      int page = page_of(RSLOTS);
      for (int i = 0; i < 2 * n; ++i) {
        const int rs = i % RSLOTS, s = (i >> 1) % SLOTS, use = (i >> 1) / SLOTS;
        const bool masked = op && (i >> 1) >= first_masked;
        if (!tc_wait_warp(bar(&sh.rfull[op][rs]), (uint32_t)((i / RSLOTS) & 1), abort_flag) ||
            (!(i & 1) && use > 0 &&
             !tc_wait_warp(bar(op ? &sh.vempty[s] : &sh.kempty[s]), (uint32_t)((use - 1) & 1), abort_flag))) {
          ok = false;
          break;
        }
        const uint32_t raw = sbase + L::OFF_RAW + (uint32_t)(op * RSLOTS + rs) * L::RAWB;
        const uint32_t meta = sbase + L::OFF_META + (uint32_t)(op * RSLOTS + rs) * L::METAB;
        ptx::cp_async_wait<RSLOTS - 1>();
        __syncwarp();
        // All pieces of the half first, so that their loads overlap.
        constexpr int N = CPR / 2;
        uint32_t in[N][4], sz[N];
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const int rr = r0 + k * RPP;             // row of the half step
          // the raw tile has TMA's swizzle of its row width
          const int pc = RB == 128 ? ch ^ (rr & 7) : RB == 64 ? ch ^ ((rr >> 1) & 3) : ch ^ ((rr >> 2) & 1);
          asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                       : "=r"(in[k][0]), "=r"(in[k][1]), "=r"(in[k][2]), "=r"(in[k][3])
                       : "r"(raw + (uint32_t)(rr * RB + pc * 16)));
          asm volatile("ld.shared.u32 %0, [%1];" : "=r"(sz[k]) : "r"(meta + (uint32_t)((rr * a.gpr + gword) * 4)));
        }
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const int rr = r0 + k * RPP;
          // (a row that nobody sees has zero metadata: zeros, whatever its page holds)
          const uint32_t s2 = ptx::prmt(sz[k], sz[k], 0x1010), z2 = ptx::prmt(sz[k], sz[k], 0x3232);
          uint32_t o[4 * P16];
          if (FMT == KVF_FMT_INT8) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              // bytes under the exponent of 1024: half2 of 1024 + code, exact; less 1024, exact
              const uint32_t lo = ptx::prmt(in[k][q], 0x64646464u, 0x4140), hi = ptx::prmt(in[k][q], 0x64646464u, 0x4342);
              o[2 * q] = ptx::hfma2_u32(ptx::hsub2_u32(lo, 0x64006400u), s2, z2);
              o[2 * q + 1] = ptx::hfma2_u32(ptx::hsub2_u32(hi, 0x64006400u), s2, z2);
            }
          } else {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              uint32_t v[4];  // columns (0,4), (1,5), (2,6), (3,7) of the word's eight
#pragma unroll
              for (int u = 0; u < 4; ++u)
                v[u] = ptx::hfma2_u32(
                    ptx::hsub2_u32(ptx::lop3_and_or(in[k][q] >> (4 * u), 0x000F000Fu, 0x64006400u), 0x64006400u), s2, z2);
              o[4 * q] = ptx::prmt(v[0], v[1], 0x5410);
              o[4 * q + 1] = ptx::prmt(v[2], v[3], 0x5410);
              o[4 * q + 2] = ptx::prmt(v[0], v[1], 0x7632);
              o[4 * q + 3] = ptx::prmt(v[2], v[3], 0x7632);
            }
          }
          if (masked) {
#pragma unroll
            for (int q = 0; q < 4 * P16; ++q)
              if (odd_f16x2(o[q])) {
                odd = true;
                o[q] = even_f16x2(o[q]);
              }
          }
          // lanes that share a row start at different pieces, so that a
          // quarter of a warp stores to all banks
          const int turn = D == 64 ? 0 : FMT == KVF_FMT_INT8 ? ch >> 2 : (ch >> 1) << 1;
          const int tr = rr + (i & 1) * kTcHalf;   // row of the tile
          const uint32_t base = ring + s * TILE + tr * 128u;
#pragma unroll
          for (int q = 0; q < P16; ++q) {
            const int at = q ^ turn;
            const int ci = ch * P16 + at;          // 16-byte piece of the tile row
            uint32_t x0 = o[0], x1 = o[1], x2 = o[2], x3 = o[3];
#pragma unroll
            for (int u = 1; u < P16; ++u)
              if (at == u) {
                x0 = o[4 * u];
                x1 = o[4 * u + 1];
                x2 = o[4 * u + 2];
                x3 = o[4 * u + 3];
              }
            asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(base + (ci >> 3) * BLK +
                                                                     ((uint32_t)((ci ^ tr) & 7) << 4)),
                         "r"(x0), "r"(x1), "r"(x2), "r"(x3)
                         : "memory");
          }
        }
        const int next = page_of(i + RSLOTS + 1);
        if (i & 1) {
          if (odd) *reinterpret_cast<volatile int *>(&sh.odd) = 1;
          ptx::fence_proxy_async_smem();
        }
        __syncwarp();
        ptx::mbar_arrive_if(bar(&sh.rempty[op][rs]), lane == 0);
        if (i & 1) ptx::mbar_arrive_if(bar(op ? &sh.vfull[s] : &sh.kfull[s]), lane == 0);
        fetch_meta(i + RSLOTS, page);
        page = next;
      }
      ptx::cp_async_wait<0>();
    } else {
      for (int i = first_masked; i < n; ++i) {
        const int s = i % SLOTS;
        if (!tc_wait_warp(bar(&sh.vraw[s]), (uint32_t)(((i - first_masked) / SLOTS) & 1), abort_flag)) {
          ok = false;
          break;
        }
        const int ch = lt % (D / 8);
        for (int rr = lt / (D / 8); rr < kTcStep; rr += 128 / (D / 8)) {
          const uint32_t ad = svr + s * TILE + (ch >> 3) * BLK + rr * 128u + ((uint32_t)((ch ^ rr) & 7) << 4);
          const bool seen = w.t0 + i * kTcStep + rr < w.t1;
          uint32_t x[4];
          asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(ad));
          const bool bad = odd_f16x2(x[0]) || odd_f16x2(x[1]) || odd_f16x2(x[2]) || odd_f16x2(x[3]);
          if (seen && !bad) continue;
          if (seen) odd = true;
#pragma unroll
          for (int q = 0; q < 4; ++q) x[q] = seen ? even_f16x2(x[q]) : 0u;
          asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(ad), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3])
                       : "memory");
        }
        if (odd) *reinterpret_cast<volatile int *>(&sh.odd) = 1;
        ptx::fence_proxy_async_smem();
        __syncwarp();
        ptx::mbar_arrive_if(bar(&sh.vfixed[s]), lane == 0);
      }
    }
    if (!ok && lane == 0) {
      atomicOr(&g_kvfb_chunk_error, 1u);
      *abort_flag = 1;
    }
  } else {
    regs_down<L::LAST_REGS>();
    if (warp == LAST + 1 || warp == LAST + 2) {
      // ----------------------------------------------------------- producers
      const int op = warp - LAST - 1;  // 0: K, 1: V
      const CUtensorMap *map = op ? &tmv : &tmk;
      const uint64_t pol = ptx::policy_evict_last();
      const bool paged = a.cache.paged != 0;
      const int bts = paged ? a.cache.bt_shift : 30, bmask = (1 << bts) - 1;
      const int tbs = min(bts, 6);             // log2 of the tokens of a box
      const int span = L::RAW ? kTcHalf : kTcStep, boxes = span >> tbs;  // 1 to 8 boxes an item
      const int count = L::RAW ? 2 * n : n;
      const int box = lane & (boxes - 1);
      const int *table = paged ? a.cache.table + (long long)w.b * a.cache.max_blocks : nullptr;
      // Page (or sequence) of box `box` of item i; -1 where there is nothing to read.
      auto page_of = [&](int i) -> int {
        const int t = w.t0 + i * span + (box << tbs);
        int page = paged ? -1 : w.b;
        if (i >= count || t >= w.t1) return -1;
        if (paged) page = __ldg(table + (t >> bts));
        return page;
      };
      // One elected lane issues an item's boxes; coordinates come from the lanes
      // that hold them. A box with no page is not asked for. What its rows hold is
      // of no account where nobody sees them (scores are masked, values cleared),
      // nor in a quantized cache (codes of no scale and no zero); rows of an f16
      // cache that are seen all the same, in a block without a page, are zeros.
      auto fill = [&](uint32_t dst, uint32_t full, uint32_t bytes, int t, int page) {
        const uint32_t there = __ballot_sync(0xffffffffu, lane < boxes && page >= 0);
        if constexpr (!L::RAW) {
          uint32_t blank = __ballot_sync(0xffffffffu, lane < boxes && page < 0 && t + (lane << tbs) < w.t1);
          if (blank) {
            for (; blank; blank &= blank - 1) {
              const uint32_t at = dst + ((uint32_t)(__ffs(blank) - 1) << tbs) * 128u;
              for (int k = lane; k < KB * (8 << tbs); k += 32)
                asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(at + (uint32_t)(k / (8 << tbs)) * BLK +
                                                                         (uint32_t)(k % (8 << tbs)) * 16u),
                             "r"(0)
                             : "memory");
            }
            ptx::fence_proxy_async_smem();
            __syncwarp();
          }
        }
        bytes = bytes / (uint32_t)boxes * (uint32_t)__popc(there);
        if (tc::elect_one()) {
          if (bytes)
            ptx::mbar_arrive_expect_tx(full, bytes);
          else
            ptx::mbar_arrive(full);
        }
        __syncwarp();
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          if (there >> x & 1u) {
            const int pg = __shfl_sync(0xffffffffu, page, x);
            if (tc::elect_one()) {
              const int c1 = paged ? (t + (x << tbs)) & bmask : t + (x << tbs);
              if (L::RAW) {
                ptx::tma_g2s_4d(dst + ((uint32_t)x << tbs) * RB, map, 0, c1, w.h, pg, full, pol);
              } else {
#pragma unroll
                for (int blk = 0; blk < KB; ++blk)
                  ptx::tma_g2s_4d(dst + blk * BLK + ((uint32_t)x << tbs) * 128u, map, 128 * blk, c1, w.h, pg, full, pol);
              }
            }
            __syncwarp();
          }
        }
      };
      bool ok = true;
      int page = page_of(0), i = 0;
      for (; i < count; ++i) {
        const int t = w.t0 + i * span;
        if constexpr (L::RAW) {
          const int s = i % RSLOTS;
          if (i >= RSLOTS && !tc_wait_warp(bar(&sh.rempty[op][s]), (uint32_t)((i / RSLOTS - 1) & 1), abort_flag)) {
            ok = false;
            break;
          }
          fill(sbase + L::OFF_RAW + (uint32_t)(op * RSLOTS + s) * L::RAWB, bar(&sh.rfull[op][s]), L::RAWB, t, page);
        } else {
          const int s = i % SLOTS;
          if (i >= SLOTS && !tc_wait_warp(bar(op ? &sh.vempty[s] : &sh.kempty[s]), (uint32_t)((i / SLOTS - 1) & 1), abort_flag)) {
            ok = false;
            break;
          }
          fill((op ? svr : skr) + s * TILE, bar(!op ? &sh.kfull[s] : i < first_masked ? &sh.vfull[s] : &sh.vraw[s]), TILE, t,
               page);
        }
        page = page_of(i + 1);
      }
      if (!ok && lane == 0) {
        atomicOr(&g_kvfb_chunk_error, 1u);
        *abort_flag = 1;
      }
      // Never leave with copies in flight: the last item of each slot has landed.
      constexpr int RING = L::RAW ? RSLOTS : SLOTS;
      for (int k = max(0, i - RING); k < i; ++k) {
        const int s = k % RING;
        const bool fixed = !L::RAW && op && k >= first_masked;
        const uint32_t full = L::RAW ? bar(&sh.rfull[op][s]) : bar(!op ? &sh.kfull[s] : fixed ? &sh.vraw[s] : &sh.vfull[s]);
        if (!ptx::mbar_wait(full, (uint32_t)(((fixed ? k - first_masked : k) / RING) & 1)) && lane == 0) atomicOr(&g_kvfb_chunk_error, 1u);
      }
    } else {
      // --------------------------------------------------------- MMA issue
      const int g = warp == LAST ? 0 : 1;  // the softmax group that this warp issues for
      const int nw = group_steps(g);
      constexpr uint32_t ID_S = tc::idesc_f16(false, false, 128, 64), ID_O = tc::idesc_f16(false, true, 128, D);
      bool ok = true;
      // Waits for K or V tile i.
      auto take_k = [&](int i) -> bool {
        if (!tc_wait_warp(bar(&sh.kfull[i % SLOTS]), (uint32_t)((i / SLOTS) & 1), abort_flag)) return ok = false;
        tc::fence_after();
        return true;
      };
      auto take_v = [&](int i) -> bool {
        const bool fixed = !L::RAW && i >= first_masked;
        const int use = (fixed ? i - first_masked : i) / SLOTS;
        if (!tc_wait_warp(bar(fixed ? &sh.vfixed[i % SLOTS] : &sh.vfull[i % SLOTS]), (uint32_t)(use & 1), abort_flag))
          return ok = false;
        tc::fence_after();
        return true;
      };
      // S = Q K^T for half h of K tile i, and O += P V for half h of V tile i (the
      // group's step j) once the weights are there.
      auto scores = [&](int i, int h) {
        const uint32_t q = sq + (TWO ? (uint32_t)g * TILE : 0u), k = skr + (uint32_t)(i % SLOTS) * TILE + 8192u * h;
        const uint64_t dq = tc::smem_desc(q, 16u, 1024u, tc::kSwizzle128), dk = tc::smem_desc(k, 16u, 1024u, tc::kSwizzle128);
        if (tc::elect_one()) {
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks) {
            const uint32_t off = ((ks >> 2) * BLK + (ks & 3) * 32u) >> 4;  // descriptors count 16-byte units
            tc::mma_f16_ss(tbase + S_COL + 128u * g + 64u * h, dq + off, dk + off, ID_S, ks > 0);
          }
          tc::commit(bar(&sh.sfull[g][h]));
        }
        __syncwarp();
      };
      auto values = [&](int i, int j, int h) -> bool {
        const uint64_t dv = tc::smem_desc(svr + (uint32_t)(i % SLOTS) * TILE + 8192u * h, BLK, 1024u, tc::kSwizzle128);
        if (!tc_wait_warp(bar(&sh.pready[g][h]), (uint32_t)(j & 1), abort_flag)) return ok = false;
        tc::fence_after();
        if (tc::elect_one()) {
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            tc::mma_f16_ta(tbase + O_COL + (uint32_t)(D * g), tbase + S_COL + 128u * g + 64u * h + 8u * ks, dv + ks * (2048u >> 4),
                           ID_O, j > 0 || h > 0 || ks > 0);
          tc::commit(bar(&sh.ofull[g][h]));
        }
        __syncwarp();
        return true;
      };
      auto release = [&](const uint64_t *b) {
        if (tc::elect_one()) tc::commit(bar(b));
        __syncwarp();
      };
      // Tiles: every one (TWO; past the group's last step only to hand it back), or
      // every second.
      constexpr int STRIDE = TWO ? 1 : 2;
      int i = TWO ? 0 : g;
      ok = tc_wait_warp(bar(&sh.qready), 0u, abort_flag);
      if (ok && i < n && take_k(i)) {
        if (nw > 0)
          for (int h = 0; h < 2; ++h) scores(i, h);
        release(&sh.kempty[i % SLOTS]);
      }
      for (int j = 0; i < n && ok; ++j, i += STRIDE) {
        if (!take_v(i)) break;
        const int next = i + STRIDE;
        const bool more = next < n;
        // The first half's next scores go between the two products, unless the
        // K tile is late: the second product does not wait for it.
        if (j < nw && !values(i, j, 0)) break;
        const bool between = more && __all_sync(0xffffffffu, ptx::mbar_test_wait(bar(&sh.kfull[next % SLOTS]),
                                                                               (uint32_t)((next / SLOTS) & 1)));
        if (between) {
          tc::fence_after();
          if (j + 1 < nw) scores(next, 0);
        }
        if (j < nw && !values(i, j, 1)) break;
        release(&sh.vempty[i % SLOTS]);
        if (more && (between || take_k(next))) {
          if (j + 1 < nw) {
            if (!between) scores(next, 0);
            scores(next, 1);
          }
          release(&sh.kempty[next % SLOTS]);
        }
      }
      if (!ok && lane == 0) {
        atomicOr(&g_kvfb_chunk_error, 1u);
        *abort_flag = 1;
      }
      // tensor memory is freed below only after every MMA issued here completed
      release(&sh.done);
      if (!ptx::mbar_wait(bar(&sh.done), 0u, 1000000000ull) && lane == 0) atomicOr(&g_kvfb_chunk_error, 1u);
    }
    __syncwarp();
  }
  __syncthreads();
  if (warp == LAST) tc::dealloc(tbase, 512u);
}

} // namespace
} // namespace kvfb
