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

// code() without the division in the common case. With a = x - zero (fp32,
// as the host computes it) and r = 1/sc rounded to nearest, t' = a * r is
// within 3 * 2^-24 |t| of the host's t = a / sc (both correctly rounded), so
// for |t'| < 1024 the two differ by less than 2^-12. When t' is further than
// that from every half-integer, t lies strictly between the same two
// half-integers as t', and round-half-away(t) = rint(t'); otherwise (and for
// |t'| >= 1024, NaN or infinities, including sc = 0) the exact code() decides.
__device__ __forceinline__ int code_fast(float x, float zero, float sc, float rsc, int levels) {
  const float a = __fsub_rn(x, zero);
  const float t = __fmul_rn(a, rsc);
  if (fabsf(t) < 1024.f) {
    const float q = rintf(t);
    if (fabsf(__fsub_rn(t, q)) < 0.5f - 0x1p-12f) {
      const int qi = (int)q;
      return qi < 0 ? 0 : (qi > levels ? levels : qi);
    }
  }
  return code(x, zero, sc, levels);
}

// One group of a row held as eight channels per lane (group / 8 adjacent
// lanes, a power of two): its (scale, zero) word and their fp32 values.
struct GroupScale {
  uint32_t word;
  float zero, sc, rsc;
};

// Scale and zero of lane li's group, combined across the group's lanes with
// shuffles (every lane of the warp takes part). The combination keeps the
// host loop's results bit for bit: a lane that does not hold the group's first
// element folds its values into +inf / -inf (NaNs never replace a running
// value in the host loop, which starts from the first element), the first lane
// starts from that element (a NaN there stays NaN), and two adjacent ranges
// combine as the loop would have met them, earlier range first (ties keep the
// earlier value).
__device__ __forceinline__ GroupScale group_scale8(const float (&e)[8], int li, int group, int levels) {
  const int lpg = group >> 3;  // lanes per group
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

// Lane li's eight codes of a row whose payload starts at `row` (8-byte aligned
// for int8, 4-byte for int4).
template <int FMT>
__device__ __forceinline__ void store_codes8(const float (&e)[8], const GroupScale &g, uint8_t *row, int li) {
  const int levels = FMT == KVF_FMT_INT8 ? 255 : 15;
  uint32_t c[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) c[k] = (uint32_t)code_fast(e[k], g.zero, g.sc, g.rsc, levels);
  if (FMT == KVF_FMT_INT8) {
    const uint2 w = make_uint2(c[0] | (c[1] << 8) | (c[2] << 16) | (c[3] << 24),
                               c[4] | (c[5] << 8) | (c[6] << 16) | (c[7] << 24));
    reinterpret_cast<uint2 *>(row)[li] = w;
  } else {
    reinterpret_cast<uint32_t *>(row)[li] =
        c[0] | (c[1] << 4) | (c[2] << 8) | (c[3] << 12) | (c[4] << 16) | (c[5] << 20) | (c[6] << 24) | (c[7] << 28);
  }
}

} // namespace
} // namespace kvfb
