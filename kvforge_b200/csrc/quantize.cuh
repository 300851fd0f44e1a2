// quantize.cuh - device pieces of the KV quantizer shared by the kernels that
// write quantized rows: codes and their (scale, zero) words, a row spread over
// lanes of eight channels, and the physical row of a cache token. The rules
// that make the result bit-exact with kvf::quantize
// (runtime/kvf_host.h:72-120) are all here.
#pragma once

#include "kvforge_b200.h"

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstdint>

namespace kvfb {
namespace {

__device__ __forceinline__ uint16_t h_bits(__half h) { return __half_as_ushort(h); }

// Physical row of token t of (sequence b, KV head h) in a cache of n tokens
// per sequence (runtime/kvf_kernels.cuh:51-64, kvf_host.h:124-135). -1 for a
// token outside the cache or in a block that the table does not hold or maps
// to a negative page.
struct CacheRows {
  const int *table;
  int Hkv, n, head_major, paged, bt_shift, max_blocks;
  __device__ __forceinline__ long long row(int b, int h, long long t) const {
    if (t < 0 || t >= n) return -1;
    if (!paged) return head_major ? ((long long)b * Hkv + h) * n + t : ((long long)b * n + t) * Hkv + h;
    const int blk = (int)(t >> bt_shift);
    if (blk >= max_blocks) return -1;
    const int page = table[(long long)b * max_blocks + blk];
    if (page < 0) return -1;
    const long long bt = 1ll << bt_shift, tl = t & (bt - 1);
    const long long base = (long long)page * Hkv * bt;
    return head_major ? base + (long long)h * bt + tl : base + tl * Hkv + h;
  }
};

// clamp(lround((x - zero) / sc), 0, levels) with the host's behaviour at the
// edges: lround of a NaN, an infinity or a value of magnitude >= 2^63 yields
// LONG_MIN on x86-64, which the clamp turns into 0 (this happens when a group
// exceeds the fp16 range and zero becomes -inf).
__device__ __forceinline__ int code(float x, float zero, float sc, int levels) {
  const float t = __fdiv_rn(__fsub_rn(x, zero), sc);
  if (!(t < 9.223372036854775808e18f && t > -9.223372036854775808e18f)) return 0;
  const long long q = llroundf(t);
  return q < 0 ? 0 : (q > levels ? levels : (int)q);
}

// One group of a row held as eight channels per lane (group / 8 adjacent
// lanes, a power of two): its (scale, zero) word and their fp32 values.
struct GroupScale {
  uint32_t word;
  float zero, sc, rsc;
};

// Range of lane li's group by the host loop's comparisons (first-wins), combined
// across the group's lanes with shuffles (every lane of the warp takes part). A
// lane that does not hold the group's first element folds its values into +inf /
// -inf (NaNs never replace a running value in the host loop, which starts from
// the first element), the first lane starts from that element (a NaN there stays
// NaN), and two adjacent ranges combine as the loop would have met them, earlier
// range first (ties keep the earlier value).
__device__ __noinline__ float2 group_range8_exact(float e0, float e1, float e2, float e3, float e4, float e5, float e6,
                                                  float e7, int li, int lpg) {
  const float e[8] = {e0, e1, e2, e3, e4, e5, e6, e7};
  const bool first = (li & (lpg - 1)) == 0;
  float lo = first ? e[0] : INFINITY, hi = first ? e[0] : -INFINITY;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    if (k == 0 && first) continue;
    lo = (e[k] < lo) ? e[k] : lo;
    hi = (hi < e[k]) ? e[k] : hi;
  }
  for (int off = 1; off < lpg; off <<= 1) {
    const float plo = __shfl_xor_sync(0xffffffffu, lo, off);
    const float phi = __shfl_xor_sync(0xffffffffu, hi, off);
    const bool earlier = (li & off) == 0;
    const float alo = earlier ? lo : plo, blo = earlier ? plo : lo;
    const float ahi = earlier ? hi : phi, bhi = earlier ? phi : hi;
    lo = (blo < alo) ? blo : alo;
    hi = (ahi < bhi) ? bhi : ahi;
  }
  return make_float2(lo, hi);
}

__device__ __forceinline__ float min3f(float a, float b, float c) {
  float r;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float max3f(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Scale and zero of lane li's group, bit for bit the host loop's. The hardware's
// minimum and maximum give its range except where the group starts with a NaN
// (which the host keeps and they drop) or where its least value is a zero and one of
// its zeros negative: the host takes the sign from the first one. Those go by
// group_range8_exact.
__device__ __forceinline__ GroupScale group_scale8(const float (&e)[8], int li, int group, int levels) {
  const int lpg = group >> 3;  // lanes per group
  float lo = fminf(min3f(min3f(min3f(e[0], e[1], e[2]), e[3], e[4]), e[5], e[6]), e[7]);
  float hi = fmaxf(max3f(max3f(max3f(e[0], e[1], e[2]), e[3], e[4]), e[5], e[6]), e[7]);
  for (int off = 1; off < lpg; off <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, off));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, off));
  }
  if (__any_sync(0xffffffffu, !(lo != 0.f && lo == lo) || e[0] != e[0])) {
    // Where a least value of zero meets no negative zero it is the positive one
    // (2^20 rows of 128 values from zero up into int8: 176 us, 222 where each goes
    // through the loop; rows of zeros 168 and 215).
    uint32_t bits = 0u;
#pragma unroll
    for (int k = 0; k < 8; ++k) bits |= __float_as_uint(e[k]);
    if (__any_sync(0xffffffffu, lo != lo || e[0] != e[0] || (lo == 0.f && (int)bits < 0))) {
      const float2 r = group_range8_exact(e[0], e[1], e[2], e[3], e[4], e[5], e[6], e[7], li, lpg);
      lo = r.x;
      hi = r.y;
    }
  }
  const __half zero_h = __float2half_rn(lo);
  float scale = __fdiv_rn(__fsub_rn(hi, lo), (float)levels);
  if (scale <= 0.f) scale = 1.f;
  const __half scale_h = __float2half_rn(scale);
  GroupScale g;
  g.word = (uint32_t)h_bits(scale_h) | ((uint32_t)h_bits(zero_h) << 16);
  g.zero = __half2float(zero_h);
  g.sc = __half2float(scale_h);
  g.rsc = __frcp_rn(g.sc);
  return g;
}

// code() of eight values. Without the division in the common case: with a = x -
// zero (fp32, as the host computes it) and r = 1/sc rounded to nearest, t = a * r
// is within 3 * 2^-24 |t| of the host's a / sc (both correctly rounded), so for
// |t| < 1024 the two differ by less than 2^-12. Where t clamped to [0, levels] is
// further than that from every half-integer, the nearest integer is the host's
// code (clamping and rounding to nearest commute: the ends are integers). Otherwise
// (and for |t| >= 1024, infinities and a zero scale) the exact code() decides;
// a NaN is code 0 either way. Adding 1.5 * 2^23 leaves the integer in the low bits.
__device__ __noinline__ uint2 codes8_exact(float x0, float x1, float x2, float x3, float x4, float x5, float x6, float x7,
                                           float zero, float sc, int levels) {
  return make_uint2((uint32_t)code(x0, zero, sc, levels) | (uint32_t)code(x1, zero, sc, levels) << 8 |
                        (uint32_t)code(x2, zero, sc, levels) << 16 | (uint32_t)code(x3, zero, sc, levels) << 24,
                    (uint32_t)code(x4, zero, sc, levels) | (uint32_t)code(x5, zero, sc, levels) << 8 |
                        (uint32_t)code(x6, zero, sc, levels) << 16 | (uint32_t)code(x7, zero, sc, levels) << 24);
}
// The payload's bytes: eight codes (int8), or four bytes of two codes, the odd
// channel's above, in x (int4).
template <int FMT> __device__ __forceinline__ uint2 codes8(const float (&e)[8], const GroupScale &g) {
  constexpr int levels = FMT == KVF_FMT_INT8 ? 255 : 15;
  const float top = (float)levels, big = 12582912.f;
  float far = 0.f, off = 0.f;
  uint32_t y[8];
#pragma unroll
  for (int k = 0; k < 8; k += 2) {
    const float t0 = __fmul_rn(__fsub_rn(e[k], g.zero), g.rsc), t1 = __fmul_rn(__fsub_rn(e[k + 1], g.zero), g.rsc);
    far = max3f(far, fabsf(t0), fabsf(t1));
    const float c0 = fminf(fmaxf(t0, 0.f), top), c1 = fminf(fmaxf(t1, 0.f), top);
    const float y0 = __fadd_rn(c0, big), y1 = __fadd_rn(c1, big);
    off = max3f(off, fabsf(__fsub_rn(c0, __fsub_rn(y0, big))), fabsf(__fsub_rn(c1, __fsub_rn(y1, big))));
    y[k] = __float_as_uint(y0);
    y[k + 1] = __float_as_uint(y1);
  }
  uint2 c;
  if (FMT == KVF_FMT_INT8)
    c = make_uint2(__byte_perm(__byte_perm(y[0], y[1], 0x0040), __byte_perm(y[2], y[3], 0x0040), 0x5410),
                   __byte_perm(__byte_perm(y[4], y[5], 0x0040), __byte_perm(y[6], y[7], 0x0040), 0x5410));
  else
    c = make_uint2(__byte_perm(__byte_perm(y[0] + (y[1] << 4), y[2] + (y[3] << 4), 0x0040),
                               __byte_perm(y[4] + (y[5] << 4), y[6] + (y[7] << 4), 0x0040), 0x5410),
                   0u);
  if (!(far < 1024.f && off < 0.5f - 0x1p-12f)) {
    c = codes8_exact(e[0], e[1], e[2], e[3], e[4], e[5], e[6], e[7], g.zero, g.sc, levels);
    if (FMT == KVF_FMT_INT4) c.x = __byte_perm(c.x | c.x >> 4, c.y | c.y >> 4, 0x6420);
  }
  return c;
}

// Lane li's eight codes of a row whose payload starts at `row` (8-byte aligned
// for int8, 4-byte for int4).
template <int FMT>
__device__ __forceinline__ void store_codes8(const float (&e)[8], const GroupScale &g, uint8_t *row, int li) {
  const uint2 c = codes8<FMT>(e, g);
  if (FMT == KVF_FMT_INT8)
    reinterpret_cast<uint2 *>(row)[li] = c;
  else
    reinterpret_cast<uint32_t *>(row)[li] = c.x;
}

} // namespace
} // namespace kvfb
