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
// Warp roles (416 threads, one block per SM):
//   warps 0-3, 4-7  two softmax groups, thread = row of a 128-row tile. TWO: each
//                   has its own row tile and both take every step of 128 tokens;
//                   else both have the same rows and take steps in turn, each
//                   with its own output, as two splits. Either way one group's
//                   softmax runs while the tensor cores work for the other;
//   warps 8-11      loaders: rows come by cp.async from wherever their pages lie,
//                   quantized ones into a staging area of the thread that also
//                   converts them, into tiles of 128 tokens x 64 channels with the
//                   128-byte swizzle; K and V tiles share a ring of four slots;
//   warp 12         one thread issues the MMAs: S = Q K^T into tensor memory,
//                   O += P V with P read from tensor memory, where the softmax
//                   group writes it over its scores, and V read MN-major.
// The running maximum a row's weights are taken against is raised only when a
// step exceeds it by more than 2^8 (weights up to 256 fit fp16, and their sum
// fp32), so the output in tensor memory is rescaled rarely and a step's scores
// are read once.
// Waits are bounded in time; tensor memory is released before exit.
#pragma once

#include "chunk.cuh"
#include "tc.cuh"

namespace kvfb {

// A wait of chunk_tc_kernel ran out of time (reported as bit 0 of
// kvf_b200_device_errors).
__device__ unsigned g_kvfb_chunk_error;

namespace {

constexpr int kTcRows = 128;    // rows of a tile
constexpr int kTcStep = 128;    // tokens of a step
constexpr int kTcThreads = 416;
constexpr int kTcLoadWarp = 8;  // to 11
constexpr int kTcMmaWarp = 12;
constexpr int kTcSlots = 4;
constexpr int kTcStages = 2;    // staged items of a quantized cache
constexpr float kTcLazy = 8.f;  // log2 of the most a weight may exceed 1 by

struct TcShared {
  uint64_t bars[16];  // full[4], empty[4], sfull[2], pready[2], ofull[2], done
  uint32_t tmem;
  int abort_flag;
  int odd;            // a masked V tile held an infinity or NaN, taken as 0
};

__host__ __device__ constexpr int cache_row_bytes(int fmt, int d) {
  return fmt == KVF_FMT_F16 ? 2 * d : fmt == KVF_FMT_INT8 ? d : d / 2;
}
__host__ __device__ constexpr uint32_t tc_tile_bytes(int d) { return (uint32_t)(kTcStep * d * 2); }
// One staged item: raw rows, then their metadata words.
__host__ __device__ constexpr uint32_t tc_stage_bytes(int fmt, int d) {
  return fmt == KVF_FMT_F16 ? 0u : (uint32_t)(kTcStep * cache_row_bytes(fmt, d) + kTcStep * (fmt == KVF_FMT_INT8 ? 8 : 16));
}
__host__ __device__ constexpr uint32_t tc_smem_bytes(int fmt, int d, bool two) {
  return (two ? 2u : 1u) * tc_tile_bytes(d) + kTcSlots * tc_tile_bytes(d) + kTcStages * tc_stage_bytes(fmt, d) +
         (uint32_t)sizeof(TcShared);
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
__device__ __forceinline__ float max3f(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
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

// Order in which K and V tiles are loaded and consumed: `lead` K tiles, then
// V0, K(lead), V1, ...
struct TcItems {
  int kn = 0, vn = 0;
  __device__ __forceinline__ bool next(int n, int lead, int &i) {  // true: a V tile
    if (kn < n && kn < vn + lead) {
      i = kn++;
      return false;
    }
    i = vn++;
    return true;
  }
};

template <int FMT, int DT, int D, bool TWO>
__global__ void __launch_bounds__(kTcThreads, 1) chunk_tc_kernel(const ChunkArgs a) {
  constexpr int KB = D / 64;                       // 64-channel blocks of a tile
  constexpr uint32_t TILE = tc_tile_bytes(D);
  constexpr uint32_t BLK = TILE / KB;              // 128 rows x 128 bytes
  constexpr int RB = cache_row_bytes(FMT, D);
  constexpr int CPR = RB / 16;                     // 16-byte pieces of a cache row
  constexpr int RPP = 128 / CPR;                   // rows that the 128 loader threads take at a time
  constexpr int LEAD = TWO ? 1 : 2;
  constexpr uint32_t S_COL = 0, O_COL = 256;       // tensor-memory columns: scores (2 x 128), outputs (2 x D)

  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sbase = ptx::smem_u32(smem);
  const uint32_t sq = sbase, sring = sq + (TWO ? 2u : 1u) * TILE, sstage = sring + kTcSlots * TILE;
  TcShared &sh = *reinterpret_cast<TcShared *>(smem + (sstage - sbase) + kTcStages * tc_stage_bytes(FMT, D));
  volatile int *abort_flag = &sh.abort_flag;
  const uint32_t bars = ptx::smem_u32(&sh.bars[0]);
  const uint32_t bar_full = bars, bar_empty = bars + 32, bar_sfull = bars + 64, bar_pready = bars + 80,
                 bar_ofull = bars + 96, bar_done = bars + 112;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  ChunkWork w;
  const int nsplit = TWO ? a.splits : a.splits / 2;
  if (!chunk_work(a, nsplit, TWO ? 2 * kTcRows : kTcRows, kTcStep, w)) return;
  const int n = (w.t1 - w.t0 + kTcStep - 1) / kTcStep;

  // Steps of each softmax group.
  int nw[2];
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    if (TWO) {
      const int rows = min(w.rows - g * kTcRows, kTcRows);
      const int seen = rows > 0 ? chunk_seen(a, w, w.row0 + g * kTcRows + rows - 1) : 0;
      nw[g] = seen > w.t0 ? min(n, (seen - w.t0 + kTcStep - 1) / kTcStep) : 0;
    } else {
      nw[g] = (n + 1 - g) / 2;
    }
  }

  if (tid == 0) {
    sh.abort_flag = 0;
    sh.odd = 0;
    for (int s = 0; s < kTcSlots; ++s) {
      ptx::mbar_init(bar_full + 8u * s, 4u);
      ptx::mbar_init(bar_empty + 8u * s, 1u);
    }
    for (int g = 0; g < 2; ++g) {
      ptx::mbar_init(bar_sfull + 8u * g, 1u);
      ptx::mbar_init(bar_pready + 8u * g, 4u);
      ptx::mbar_init(bar_ofull + 8u * g, 1u);
    }
    ptx::mbar_init(bar_done, 1u);
    ptx::fence_barrier_init();
  }
  if (warp == kTcMmaWarp) {
    tc::alloc(ptx::smem_u32(&sh.tmem), 512u);
    tc::relinquish();
  }

  // Query rows, scaled, into their tile: thread = row.
  const int grp = warp >> 2;              // softmax group (warps 0-7)
  const int r = tid & 127;                // row of the tile
  float c = a.scale_log2;                 // softmax scale of the row, log2 units
  const int row = (TWO ? grp * kTcRows : 0) + r;
  if (warp < 8) {
    float mx = 0.f;
    uint32_t e = 127u << 23;
    const bool live = row < w.rows;
    const uint8_t *src = a.q.p + (live ? chunk_row(a.q, a, w, row) : 0);
    if (DT == KVF_DT_BF16 && live) {
      for (int i = 0; i < D / 8; ++i) {
        float x[8];
        load8<DT>(src + 16 * i, a.q.vec, x);
#pragma unroll
        for (int k = 0; k < 8; ++k) mx = fmaxf(mx, fabsf(x[k]));
      }
      // 2^(14 - exponent of mx), within what fp32 holds; 1 for zero, infinities and NaN
      if (mx > 0.f && mx < INFINITY) {
        const int ex = min(max((int)(__float_as_uint(mx) >> 23), 27), 240);
        e = (uint32_t)(127 + 14 + 127 - ex) << 23;
        c *= __uint_as_float((uint32_t)(ex - 14) << 23);
      }
    }
    if (TWO || grp == 0) {
      const float f = __uint_as_float(e);
      for (int i = 0; i < D / 8; ++i) {
        float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (live) load8<DT>(src + 16 * i, a.q.vec, x);
        uint32_t p[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) p[k] = narrow2<KVF_DT_F16>(x[2 * k] * f, x[2 * k + 1] * f);
        const uint32_t ad = sq + (TWO ? grp * TILE : 0u) + (i >> 3) * BLK + r * 128u + ((uint32_t)((i ^ r) & 7) << 4);
        asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(ad), "r"(p[0]), "r"(p[1]), "r"(p[2]), "r"(p[3])
                     : "memory");
      }
    }
    ptx::fence_proxy_async_smem();
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tbase = sh.tmem;

  if (warp >= kTcLoadWarp && warp < kTcMmaWarp) {
    // ------------------------------------------------------------- loaders
    const int lt = tid - kTcLoadWarp * 32;
    const int ch = lt % CPR, r0 = lt / CPR;
    const int items = 2 * n;
    bool ok = true;
    TcItems gi, gc;
    const int gword = FMT == KVF_FMT_F16 ? 0 : (ch * (16 * D / RB)) >> a.group_shift;  // metadata word of the piece
    // Starts the copies of item `it` and closes their group.
    auto issue = [&](int it) {
      if (it < items && ok) {
        int i;
        const bool isv = gi.next(n, LEAD, i);
        const uint8_t *src = isv ? a.v : a.k;
        const uint32_t *meta = isv ? a.vm : a.km;
        const int t = w.t0 + i * kTcStep;
        uint32_t dst = sstage + (it % kTcStages) * tc_stage_bytes(FMT, D);
        const uint32_t mdst = dst + kTcStep * RB;
        if (FMT == KVF_FMT_F16) {
          const int s = it % kTcSlots;
          if (it >= kTcSlots && !tc_wait_warp(bar_empty + 8u * s, (uint32_t)((it / kTcSlots - 1) & 1), abort_flag)) ok = false;
          dst = sring + s * TILE;
        }
        if (ok) {
#pragma unroll
          for (int k = 0; k < CPR; ++k) {
            const int rr = r0 + k * RPP;
            const long long rw = t + rr < w.t1 ? a.cache.row(w.b, w.h, t + rr) : -1;
            const bool there = rw >= 0;
            const uint8_t *p = there ? src + rw * RB + ch * 16 : src;
            if (FMT == KVF_FMT_F16) {
              ptx::cp_async_16_zfill(dst + (ch >> 3) * BLK + rr * 128u + ((uint32_t)((ch ^ rr) & 7) << 4), p, there ? 16u : 0u);
            } else {
              ptx::cp_async_16_zfill(dst + (uint32_t)(k * 128 + lt) * 16u, p, there ? 16u : 0u);
              if (ch == 0) {
                const uint32_t *mp = there ? meta + rw * a.gpr : meta;
                const uint32_t md = mdst + (uint32_t)(rr * a.gpr * 4);
                if (a.gpr == 1)
                  ptx::cp_async_4_zfill(md, mp, there ? 4u : 0u);
                else if (a.gpr == 2)
                  ptx::cp_async_8_zfill(md, mp, there ? 8u : 0u);
                else
                  ptx::cp_async_16_zfill(md, mp, there ? 16u : 0u);
              }
            }
          }
        }
      }
      ptx::cp_async_commit();
    };
    constexpr int AHEAD = FMT == KVF_FMT_F16 ? kTcSlots - 1 : kTcStages;  // items in flight
    for (int it = 0; it < AHEAD; ++it) issue(it);
    for (int it = 0; it < items && ok; ++it) {
      int i;
      const bool isv = gc.next(n, LEAD, i);
      const int s = it % kTcSlots;
      const int t = w.t0 + i * kTcStep;
      // V tiles that some row of the block does not see whole must not carry
      // infinities or NaN into it (0 * inf): zeros stand in, and the rows that
      // do see them get them at the end.
      const bool masked = isv && t + kTcStep > w.seen0;
      bool odd = false;
      ptx::cp_async_wait<AHEAD - 1>();
      const uint32_t tile = sring + s * TILE;
      if (FMT == KVF_FMT_F16) {
        if (masked) {
#pragma unroll 4
          for (int k = 0; k < CPR; ++k) {
            const int rr = r0 + k * RPP;
            const uint32_t ad = tile + (ch >> 3) * BLK + rr * 128u + ((uint32_t)((ch ^ rr) & 7) << 4);
            uint32_t p[4];
            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(p[0]), "=r"(p[1]), "=r"(p[2]), "=r"(p[3]) : "r"(ad));
            if (odd_f16x2(p[0]) || odd_f16x2(p[1]) || odd_f16x2(p[2]) || odd_f16x2(p[3])) {
              odd = true;
              asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(ad), "r"(even_f16x2(p[0])),
                           "r"(even_f16x2(p[1])), "r"(even_f16x2(p[2])), "r"(even_f16x2(p[3]))
                           : "memory");
            }
          }
        }
      } else {
        __syncwarp();  // the row's metadata words came by its first lane
        if (it >= kTcSlots && !tc_wait_warp(bar_empty + 8u * s, (uint32_t)((it / kTcSlots - 1) & 1), abort_flag)) {
          ok = false;
          break;
        }
        const uint32_t stage = sstage + (it % kTcStages) * tc_stage_bytes(FMT, D);
        const uint32_t mstage = stage + kTcStep * RB;
#pragma unroll 4
        for (int k = 0; k < CPR; ++k) {
          const int rr = r0 + k * RPP;
          uint32_t raw[4], sz;
          asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                       : "=r"(raw[0]), "=r"(raw[1]), "=r"(raw[2]), "=r"(raw[3])
                       : "r"(stage + (uint32_t)(k * 128 + lt) * 16u));
          asm volatile("ld.shared.u32 %0, [%1];" : "=r"(sz) : "r"(mstage + (uint32_t)((rr * a.gpr + gword) * 4)));
          const uint32_t s2 = ptx::prmt(sz, sz, 0x1010), z2 = ptx::prmt(sz, sz, 0x3232);
          uint32_t o[16];
          if (FMT == KVF_FMT_INT8) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              // bytes under the exponent of 1024: half2 of 1024 + code, exact; less 1024, exact
              const uint32_t lo = ptx::prmt(raw[q], 0x64646464u, 0x4140), hi = ptx::prmt(raw[q], 0x64646464u, 0x4342);
              o[2 * q] = ptx::hfma2_u32(ptx::hsub2_u32(lo, 0x64006400u), s2, z2);
              o[2 * q + 1] = ptx::hfma2_u32(ptx::hsub2_u32(hi, 0x64006400u), s2, z2);
            }
          } else {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              uint32_t v[4];  // columns (0,4), (1,5), (2,6), (3,7) of the word's eight
#pragma unroll
              for (int u = 0; u < 4; ++u)
                v[u] = ptx::hfma2_u32(ptx::hsub2_u32(ptx::lop3_and_or(raw[q] >> (4 * u), 0x000F000Fu, 0x64006400u), 0x64006400u), s2, z2);
              o[4 * q] = ptx::prmt(v[0], v[1], 0x5410);
              o[4 * q + 1] = ptx::prmt(v[2], v[3], 0x5410);
              o[4 * q + 2] = ptx::prmt(v[0], v[1], 0x7632);
              o[4 * q + 3] = ptx::prmt(v[2], v[3], 0x7632);
            }
          }
          constexpr int P16 = 32 / (RB * 16 / D);  // 16-byte pieces out per piece in: 2 (int8), 4 (int4)
          static_assert(FMT == KVF_FMT_F16 || P16 == (FMT == KVF_FMT_INT8 ? 2 : 4), "pieces");
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
          const int turn = FMT == KVF_FMT_INT8 ? ch >> 2 : (ch >> 1) << 1;
#pragma unroll
          for (int q = 0; q < P16; ++q) {
            const int at = q ^ (D == 128 ? turn & (P16 - 1) : 0);
            const int ci = ch * P16 + at;  // 16-byte piece of the tile row
            uint32_t x0 = o[0], x1 = o[1], x2 = o[2], x3 = o[3];
#pragma unroll
            for (int u = 1; u < P16; ++u)
              if (at == u) {
                x0 = o[4 * u];
                x1 = o[4 * u + 1];
                x2 = o[4 * u + 2];
                x3 = o[4 * u + 3];
              }
            asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(tile + (ci >> 3) * BLK + rr * 128u +
                                                                     ((uint32_t)((ci ^ rr) & 7) << 4)),
                         "r"(x0), "r"(x1), "r"(x2), "r"(x3)
                         : "memory");
          }
        }
      }
      if (odd) *reinterpret_cast<volatile int *>(&sh.odd) = 1;
      ptx::fence_proxy_async_smem();
      __syncwarp();
      ptx::mbar_arrive_if(bar_full + 8u * s, lane == 0);
      issue(it + AHEAD);
    }
    if (!ok && lane == 0) {
      atomicOr(&g_kvfb_chunk_error, 1u);
      *abort_flag = 1;
    }
    ptx::cp_async_wait<0>();
  } else if (warp == kTcMmaWarp) {
    // ----------------------------------------------------------- MMA issue
    if (lane == 0) {
      constexpr uint32_t ID_S = tc::idesc_f16(false, false, 128, 128), ID_O = tc::idesc_f16(false, true, 128, D);
      bool ok = true;
      int it = 0;  // items consumed
      uint32_t kslot = 0;
      // Waits for the next item of the ring and returns its tile.
      auto take = [&](uint32_t &slot) -> bool {
        slot = (uint32_t)(it % kTcSlots);
        if (!tc_wait(bar_full + 8u * slot, (uint32_t)((it / kTcSlots) & 1), abort_flag)) return ok = false;
        ++it;
        tc::fence_after();
        return true;
      };
      auto scores = [&](int g, uint32_t slot) {
        const uint32_t q = sq + (TWO ? (uint32_t)g * TILE : 0u), k = sring + slot * TILE;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          const uint32_t off = (ks >> 2) * BLK + (ks & 3) * 32u;
          tc::mma_f16_ss(tbase + S_COL + 128u * g, tc::smem_desc(q + off, 16u, 1024u, tc::kSwizzle128),
                         tc::smem_desc(k + off, 16u, 1024u, tc::kSwizzle128), ID_S, ks > 0);
        }
        tc::commit(bar_sfull + 8u * g);
      };
      auto values = [&](int g, uint32_t slot, bool acc) {
        const uint32_t v = sring + slot * TILE;
#pragma unroll
        for (int ks = 0; ks < kTcStep / 16; ++ks)
          tc::mma_f16_ta(tbase + O_COL + (uint32_t)(D * g), tbase + S_COL + 128u * g + 8u * ks,
                         tc::smem_desc(v + ks * 2048u, BLK, 1024u, tc::kSwizzle128), ID_O, acc || ks > 0);
        tc::commit(bar_ofull + 8u * g);
      };
      if (TWO) {
        if (n > 0 && take(kslot)) {
          for (int g = 0; g < 2; ++g)
            if (nw[g] > 0) scores(g, kslot);
          tc::commit(bar_empty + 8u * kslot);
        }
        for (int i = 0; i < n && ok; ++i) {
          uint32_t vslot;
          if (!take(vslot)) break;
          bool have = false;
          const int last = i < nw[1] ? 1 : 0;
          for (int g = 0; g < 2 && ok; ++g) {
            if (i < nw[g]) {
              if (!tc_wait(bar_pready + 8u * g, (uint32_t)(i & 1), abort_flag)) {
                ok = false;
                break;
              }
              tc::fence_after();
              values(g, vslot, i > 0);
            }
            if (g == last) tc::commit(bar_empty + 8u * vslot);
            if (i + 1 < nw[g]) {
              if (!have && !take(kslot)) break;
              have = true;
              scores(g, kslot);
            }
          }
          if (ok && i + 1 < n) {
            if (!have && !take(kslot)) break;
            tc::commit(bar_empty + 8u * kslot);
          }
        }
      } else {
        for (int g = 0; g < 2 && g < n && ok; ++g)
          if (take(kslot)) {
            scores(g, kslot);
            tc::commit(bar_empty + 8u * kslot);
          }
        for (int i = 0; i < n && ok; ++i) {
          const int g = i & 1, j = i >> 1;
          uint32_t vslot;
          if (!take(vslot)) break;
          if (!tc_wait(bar_pready + 8u * g, (uint32_t)(j & 1), abort_flag)) {
            ok = false;
            break;
          }
          tc::fence_after();
          values(g, vslot, j > 0);
          tc::commit(bar_empty + 8u * vslot);
          if (i + 2 < n && take(kslot)) {
            scores(g, kslot);
            tc::commit(bar_empty + 8u * kslot);
          }
        }
      }
      if (!ok) {
        atomicOr(&g_kvfb_chunk_error, 1u);
        *abort_flag = 1;
      }
      // tensor memory is freed below only after every MMA issued here completed
      tc::commit(bar_done);
      if (!ptx::mbar_wait(bar_done, 0u, 1000000000ull)) atomicOr(&g_kvfb_chunk_error, 1u);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------- softmax
    const bool live = row < w.rows;
    const int seen = live ? chunk_seen(a, w, w.row0 + row) : 0;
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t ts = tbase + lanes + S_COL + 128u * grp, to = tbase + lanes + O_COL + (uint32_t)(D * grp);
    const int steps = nw[grp];
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int j = 0; j < steps; ++j) {
      const int t = w.t0 + (TWO ? j : 2 * j + grp) * kTcStep;
      if (!tc_wait_warp(bar_sfull + 8u * grp, (uint32_t)(j & 1), abort_flag)) {
        ok = false;
        break;
      }
      tc::fence_after();
      uint32_t p[64];
      bool done = false;
      // Every row sees the whole step and has a maximum: scores are read once.
      if (__all_sync(0xffffffffu, !live || (t + kTcStep <= seen && m > -INFINITY))) {
        const float ref = live ? m : 0.f;
        const float2 c2 = make_float2(c, c), m2 = make_float2(-ref, -ref);
        float2 sum = make_float2(0.f, 0.f);
        float over = -INFINITY;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t s[32];
          tc::ld32(ts + 32u * q, s);
          tc::wait_ld32(s);
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const float2 x = fma2f(make_float2(__uint_as_float(s[2 * k]), __uint_as_float(s[2 * k + 1])), c2, m2);
            over = max3f(over, x.x, x.y);
            const float2 e = make_float2(ex2(x.x), ex2(x.y));
            sum = add2f(sum, e);
            p[16 * q + k] = narrow2<KVF_DT_F16>(e.x, e.y);
          }
        }
        if (__all_sync(0xffffffffu, !live || over <= kTcLazy)) {
          l += sum.x + sum.y;
          done = true;
        }
      }
      if (!done) {
        float mx = -INFINITY;
#pragma unroll 1
        for (int q = 0; q < 4; ++q) {
          uint32_t s[32];
          tc::ld32(ts + 32u * q, s);
          tc::wait_ld32(s);
#pragma unroll
          for (int k = 0; k < 32; ++k)
            if (t + 32 * q + k < seen) mx = fmaxf(mx, __uint_as_float(s[k]) * c);
        }
        const float mn = fmaxf(m, mx), ref = mn == -INFINITY ? 0.f : mn;
        const float f = exp2f(m - ref);
        m = mn;
        l *= f;
        if (j > 0 && __any_sync(0xffffffffu, f != 1.f)) {
          if (!tc_wait_warp(bar_ofull + 8u * grp, (uint32_t)((j - 1) & 1), abort_flag)) {
            ok = false;
            break;
          }
          tc::fence_after();
#pragma unroll 1
          for (int q = 0; q < D / 32; ++q) {
            uint32_t o[32];
            tc::ld32(to + 32u * q, o);
            tc::wait_ld32(o);
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
            tc::st32(to + 32u * q, o);
          }
        }
        float sum = 0.f;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t s[32];
          tc::ld32(ts + 32u * q, s);
          tc::wait_ld32(s);
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const int at = t + 32 * q + 2 * k;
            const float e0 = at < seen ? ex2(fmaf(__uint_as_float(s[2 * k]), c, -ref)) : 0.f;
            const float e1 = at + 1 < seen ? ex2(fmaf(__uint_as_float(s[2 * k + 1]), c, -ref)) : 0.f;
            sum += e0 + e1;
            p[16 * q + k] = narrow2<KVF_DT_F16>(e0, e1);
          }
        }
        l += sum;
      }
      {
        uint32_t x[32];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int k = 0; k < 32; ++k) x[k] = p[32 * h + k];
          tc::st32(ts + 32u * h, x);
        }
      }
      tc::wait_st();
      tc::fence_before();
      __syncwarp();
      ptx::mbar_arrive_if(bar_pready + 8u * grp, lane == 0);
    }
    if (ok && steps > 0 && !tc_wait_warp(bar_ofull + 8u * grp, (uint32_t)((steps - 1) & 1), abort_flag)) ok = false;
    tc::fence_after();
    if (!ok && lane == 0) {
      atomicOr(&g_kvfb_chunk_error, 1u);
      *abort_flag = 1;
    }
    // ------------------------------------------------------------ epilogue
    const bool none = m == -INFINITY && l == 0.f;
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
    uint8_t *out = a.out.p + (live ? chunk_row(a.out, a, w, row) : 0);
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
        const int first = w.seen0 >= w.t0 + kTcStep ? (w.seen0 - w.t0) / kTcStep : 0;
        for (int t = w.t0 + first * kTcStep; t < min(seen, w.t1); ++t) {
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
      if (!live) continue;
      if (a.splits > 1) {
        float4 *po = reinterpret_cast<float4 *>(a.part_o + part * D + 32 * q);
#pragma unroll
        for (int k = 0; k < 8; ++k)
          po[k] = make_float4(__uint_as_float(o[4 * k]), __uint_as_float(o[4 * k + 1]), __uint_as_float(o[4 * k + 2]),
                              __uint_as_float(o[4 * k + 3]));
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float x[8];
#pragma unroll
          for (int u = 0; u < 8; ++u) x[u] = __uint_as_float(o[8 * k + u]) * inv;
          store8<DT>(out + (32 * q + 8 * k) * 2, a.out.vec, x);
        }
      }
    }
    tc::fence_before();
  }
  __syncthreads();
  if (warp == kTcMmaWarp) tc::dealloc(tbase, 512u);
}

} // namespace
} // namespace kvfb
