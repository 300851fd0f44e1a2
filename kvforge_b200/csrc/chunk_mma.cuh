// chunk_mma.cuh - attention of a chunk on mma.sync in fp32 accuracy, for fp32
// queries: every cache format, both head widths.
//
// Each operand x is split into two tf32 numbers, hi = tf32(x) and lo = x - hi
// (11 significant bits each, the exponent range of fp32, so nothing has to be
// scaled), and a product is hi*hi + lo*hi + hi*lo accumulated in fp32: relative
// error about 2^-21 per product. f16 caches need no lo for K and V, whose 11
// bits tf32 holds. The tensor cores' own sums are short (32 channels of a score,
// one step of an output): they round towards zero, and what they leave is added
// in fp32 to nearest.
//
// Infinities and NaN cannot go through halves (lo * inf is NaN where lo is 0 or of
// the other sign, and 0 * inf would reach rows that do not see the token), so zeros
// stand in for those of a K or V tile, and the tokens that held them are noted: their
// scores are then worked out in fp32 from the cache, for the rows that see them,
// and their infinite or NaN values added channel by channel.
//
// Four warps of 16 rows share tiles of 64 tokens, dequantised to fp32 in shared
// memory. Scores stay in registers: the fragment that the score product leaves
// (rows x two adjacent tokens) is taken as it is for the operand of the value
// product, whose k index then runs over tokens 2t and 2t + 1 instead of t and
// t + 4, and V's rows are fetched in the same order.
#pragma once

#include "chunk.cuh"

namespace kvfb {
namespace {

constexpr int kChunkRows = 64;    // rows of a tile
constexpr int kChunkTokens = 64;  // tokens per step
constexpr int kChunkThreads = 128;

__host__ __device__ constexpr int chunk_mma_smem(int d) {
  // q and k rows of d + 8 floats (conflict-free 8-byte reads), v rows of d + 4
  // and two masks of 64 tokens
  return (kChunkRows * (d + 8) + kChunkTokens * (d + 8) + kChunkTokens * (d + 4)) * 4 + 16;
}

// x = hi + lo: hi is x rounded to tf32's 11 bits, lo the exact rest, of which the
// tensor cores take the upper 11 bits (off by at most 2^-23 of x).
__device__ __forceinline__ void split(float x, uint32_t &hi, uint32_t &lo) {
  hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
  lo = __float_as_uint(__fsub_rn(x, __uint_as_float(hi)));
}
// K and V of an f16 cache are tf32 numbers as they are.
template <bool LO> __device__ __forceinline__ void split_if(float x, uint32_t &hi, uint32_t &lo) {
  if (LO) {
    split(x, hi, lo);
  } else {
    hi = __float_as_uint(x);
    lo = 0u;
  }
}

__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}

__device__ __forceinline__ void put8(float *p, const float (&x)[8]) {
  reinterpret_cast<float4 *>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4 *>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}

// Infinities and NaN of the step's tiles, seldom there: out of line, so that the
// loops around them stay as they are without.

// Zeros for those that this thread stored, their tokens into `odd`: K's in words 0
// and 1, V's in 2 and 3.
template <int D> __device__ __noinline__ void odd_tokens(float *sk, float *sv, unsigned *odd) {
  constexpr int KS = D + 8, VS = D + 4;
  for (int i = threadIdx.x; i < kChunkTokens * (D / 8); i += kChunkThreads) {
    const int r = i / (D / 8), li = i % (D / 8);
    for (int k = 0; k < 16; ++k) {
      float *x = k < 8 ? sk + r * KS + 8 * li + k : sv + r * VS + 8 * li + k - 8;
      if (fabsf(*x) < INFINITY) continue;
      *x = 0.f;
      atomicOr(odd + (k < 8 ? 0 : 2) + (r >> 5), 1u << (r & 31));
    }
  }
}
// Products of two query rows with the K row of a token.
template <int FMT, int D>
__device__ __noinline__ float2 odd_scores(const ChunkArgs &a, long long row, const float *q_lo, const float *q_hi) {
  float2 s = make_float2(0.f, 0.f);
  for (int li = 0; li < D / 8; ++li) {
    float x[8];
    cache8<FMT, D>(a.k, a.km, a, row, li, x);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      s.x = fmaf(q_lo[8 * li + k], x[k], s.x);
      s.y = fmaf(q_hi[8 * li + k], x[k], s.y);
    }
  }
  return s;
}
// Channels 8 n + 2 t4 and the next of the V row of a token.
template <int FMT, int D> __device__ __noinline__ float2 odd_values(const ChunkArgs &a, long long row, int n, int t4) {
  float x[8];
  cache8<FMT, D>(a.v, a.vm, a, row, n, x);
  return t4 == 0   ? make_float2(x[0], x[1])
         : t4 == 1 ? make_float2(x[2], x[3])
         : t4 == 2 ? make_float2(x[4], x[5])
                   : make_float2(x[6], x[7]);
}

template <int FMT, int D>
__global__ void __launch_bounds__(kChunkThreads) chunk_mma_kernel(const __grid_constant__ ChunkArgs a) {
  constexpr int QS = D + 8, KS = D + 8, VS = D + 4;
  constexpr bool LO = FMT != KVF_FMT_F16;  // K and V need their lo halves
  extern __shared__ __align__(16) float sm[];
  float *sq = sm, *sk = sq + kChunkRows * QS, *sv = sk + kChunkTokens * KS;
  // Tokens of the step whose K (words 0, 1) or V (2, 3) rows hold an infinity or NaN.
  unsigned *odd = reinterpret_cast<unsigned *>(sv + kChunkTokens * VS);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g4 = lane >> 2, t4 = lane & 3;

  ChunkWork w;
  if (!chunk_work(a, a.splits, kChunkRows, kChunkTokens, w)) return;

  for (int i = tid; i < kChunkRows * (D / 8); i += kChunkThreads) {
    const int r = i / (D / 8), li = i % (D / 8);
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (r < w.rows) load8<KVF_DT_F32>(chunk_row(a.q, a, w, r) + 32 * li, a.q.vec, x);
    // halved, and the scale doubled: rounding to 11 bits cannot make the greatest numbers infinite
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] *= 0.5f;
    put8(sq + r * QS + 8 * li, x);
  }

  const float scale = 2.f * a.scale_log2;
  const int r_lo = warp * 16 + g4, r_hi = r_lo + 8;
  const int seen_lo = r_lo < w.rows ? chunk_seen(a, w, r_lo) : 0;
  const int seen_hi = r_hi < w.rows ? chunk_seen(a, w, r_hi) : 0;
  float m_lo = -INFINITY, m_hi = -INFINITY, l_lo = 0.f, l_hi = 0.f;
  float o[D / 8][4];
#pragma unroll
  for (int n = 0; n < D / 8; ++n)
#pragma unroll
    for (int k = 0; k < 4; ++k) o[n][k] = 0.f;

  for (int t = w.t0; t < w.t1; t += kChunkTokens) {
    __syncthreads();
    if (tid < 4) odd[tid] = 0u;
    uint32_t any = 0u;
    __syncthreads();
#pragma unroll 4
    for (int i = tid; i < kChunkTokens * (D / 8); i += kChunkThreads) {
      const int r = i / (D / 8), li = i % (D / 8);
      float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      // rows past the last that anyone sees are zero, whatever the cache holds there
      const long long row = t + r < w.t1 ? a.cache.row(w.b, w.h, t + r) : -1;
      if (row >= 0) {
        any |= cache8<FMT, D>(a.k, a.km, a, row, li, x) | cache8<FMT, D>(a.v, a.vm, a, row, li, y);
      }
      put8(sk + r * KS + 8 * li, x);
      put8(sv + r * VS + 8 * li, y);
    }
    if (any) odd_tokens<D>(sk, sv, odd);
    __syncthreads();
    unsigned long long odd_k = odd[0] | (unsigned long long)odd[1] << 32, odd_v = odd[2] | (unsigned long long)odd[3] << 32;

    float s[kChunkTokens / 8][4];
#pragma unroll
    for (int n = 0; n < kChunkTokens / 8; ++n)
#pragma unroll
      for (int k = 0; k < 4; ++k) s[n][k] = 0.f;
#pragma unroll 1
    for (int c0 = 0; c0 < D; c0 += 32) {
      uint32_t qh[4][4], ql[4][4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 q0 = *reinterpret_cast<const float2 *>(sq + r_lo * QS + c0 + 8 * k + 2 * t4);
        const float2 q1 = *reinterpret_cast<const float2 *>(sq + r_hi * QS + c0 + 8 * k + 2 * t4);
        split(q0.x, qh[k][0], ql[k][0]);
        split(q1.x, qh[k][1], ql[k][1]);
        split(q0.y, qh[k][2], ql[k][2]);
        split(q1.y, qh[k][3], ql[k][3]);
      }
#pragma unroll
      for (int n = 0; n < kChunkTokens / 8; ++n) {
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 k2 = *reinterpret_cast<const float2 *>(sk + (8 * n + g4) * KS + c0 + 8 * k + 2 * t4);
          uint32_t kh[2], kl[2];
          split_if<LO>(k2.x, kh[0], kl[0]);
          split_if<LO>(k2.y, kh[1], kl[1]);
          mma_tf32(acc, ql[k], kh);
          if (LO) mma_tf32(acc, qh[k], kl);
          mma_tf32(acc, qh[k], kh);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) s[n][k] += acc[k];
      }
    }

#pragma unroll 1
    for (; odd_k; odd_k &= odd_k - 1) {
      const int u = __ffsll(odd_k) - 1;
      // the token's score for this thread's rows, if the thread holds it
      const float2 x = odd_scores<FMT, D>(a, a.cache.row(w.b, w.h, t + u), sq + r_lo * QS, sq + r_hi * QS);
#pragma unroll
      for (int n = 0; n < kChunkTokens / 8; ++n)
#pragma unroll
        for (int k = 0; k < 2; ++k)
          if (8 * n + 2 * t4 + k == u) {
            s[n][k] = x.x;
            s[n][2 + k] = x.y;
          }
    }

    float mx_lo = -INFINITY, mx_hi = -INFINITY;
#pragma unroll
    for (int n = 0; n < kChunkTokens / 8; ++n)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int tok = t + 8 * n + 2 * t4 + k;
        s[n][k] = tok < seen_lo ? s[n][k] * scale : -INFINITY;
        s[n][2 + k] = tok < seen_hi ? s[n][2 + k] * scale : -INFINITY;
        mx_lo = fmaxf(mx_lo, s[n][k]);
        mx_hi = fmaxf(mx_hi, s[n][2 + k]);
      }
#pragma unroll
    for (int off = 1; off < 4; off <<= 1) {
      mx_lo = fmaxf(mx_lo, __shfl_xor_sync(0xffffffffu, mx_lo, off));
      mx_hi = fmaxf(mx_hi, __shfl_xor_sync(0xffffffffu, mx_hi, off));
    }
    // a row that has seen nothing keeps -inf; 0 stands in for it in the exponents
    const float n_lo = fmaxf(m_lo, mx_lo), n_hi = fmaxf(m_hi, mx_hi);
    const float b_lo = n_lo == -INFINITY ? 0.f : n_lo, b_hi = n_hi == -INFINITY ? 0.f : n_hi;
    const float f_lo = exp2f(m_lo - b_lo), f_hi = exp2f(m_hi - b_hi);
    m_lo = n_lo;
    m_hi = n_hi;
    l_lo *= f_lo;
    l_hi *= f_hi;
#pragma unroll
    for (int n = 0; n < kChunkTokens / 8; ++n)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        s[n][k] = exp2f(s[n][k] - b_lo);
        s[n][2 + k] = exp2f(s[n][2 + k] - b_hi);
        l_lo += s[n][k];
        l_hi += s[n][2 + k];
      }
    // Rows that see such a value are rescaled before it is added; the others as ever.
    float g_lo = f_lo, g_hi = f_hi;
    if (odd_v) {
      const int first = t + __ffsll(odd_v) - 1;
      if (first < seen_lo) g_lo = 1.f;
      if (first < seen_hi) g_hi = 1.f;
#pragma unroll
      for (int n = 0; n < D / 8; ++n)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          if (first < seen_lo) o[n][k] *= f_lo;
          if (first < seen_hi) o[n][2 + k] *= f_hi;
        }
    }
#pragma unroll 1
    for (; odd_v; odd_v &= odd_v - 1) {
      const int u = __ffsll(odd_v) - 1;
      // the token's weights, from the lanes that hold them
      float p_lo = 0.f, p_hi = 0.f;
      const int src = (lane & ~3) + ((u & 7) >> 1);
#pragma unroll
      for (int n = 0; n < kChunkTokens / 8; ++n) {
        const float x0 = __shfl_sync(0xffffffffu, (u & 1) ? s[n][1] : s[n][0], src);
        const float x1 = __shfl_sync(0xffffffffu, (u & 1) ? s[n][3] : s[n][2], src);
        if (n == (u >> 3)) {
          p_lo = x0;
          p_hi = x1;
        }
      }
      const long long row = a.cache.row(w.b, w.h, t + u);
#pragma unroll
      for (int n = 0; n < D / 8; ++n) {
        const float2 x = odd_values<FMT, D>(a, row, n, t4);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float v = k ? x.y : x.x;
          if (fabsf(v) < INFINITY) continue;
          if (t + u < seen_lo) o[n][k] = fmaf(p_lo, v, o[n][k]);
          if (t + u < seen_hi) o[n][2 + k] = fmaf(p_hi, v, o[n][2 + k]);
        }
      }
    }
    uint32_t ph[kChunkTokens / 8][4], pl[kChunkTokens / 8][4];
#pragma unroll
    for (int u = 0; u < kChunkTokens / 8; ++u) {
      split(s[u][0], ph[u][0], pl[u][0]);
      split(s[u][2], ph[u][1], pl[u][1]);
      split(s[u][1], ph[u][2], pl[u][2]);
      split(s[u][3], ph[u][3], pl[u][3]);
    }
    const float *v0 = sv + 2 * t4 * VS + g4;
#pragma unroll
    for (int n = 0; n < D / 8; ++n) {
      float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int u = 0; u < kChunkTokens / 8; ++u) {
        uint32_t vh[2], vl[2];
        split_if<LO>(v0[8 * u * VS + 8 * n], vh[0], vl[0]);
        split_if<LO>(v0[(8 * u + 1) * VS + 8 * n], vh[1], vl[1]);
        mma_tf32(acc, pl[u], vh);
        if (LO) mma_tf32(acc, ph[u], vl);
        mma_tf32(acc, ph[u], vh);
      }
      o[n][0] = fmaf(o[n][0], g_lo, acc[0]);
      o[n][1] = fmaf(o[n][1], g_lo, acc[1]);
      o[n][2] = fmaf(o[n][2], g_hi, acc[2]);
      o[n][3] = fmaf(o[n][3], g_hi, acc[3]);
    }
  }

#pragma unroll
  for (int off = 1; off < 4; off <<= 1) {
    l_lo += __shfl_xor_sync(0xffffffffu, l_lo, off);
    l_hi += __shfl_xor_sync(0xffffffffu, l_hi, off);
  }
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int r = half ? r_hi : r_lo;
    if (r >= w.rows) continue;
    const float m = half ? m_hi : m_lo, l = half ? l_hi : l_lo;
    const long long at = chunk_index(a, w, r);
    if (a.splits > 1) {
      const long long part = at * a.splits + w.split;
      float *po = a.part_o + part * D;
      if (t4 == 0) *reinterpret_cast<float2 *>(a.part_ml + 2 * part) = make_float2(m, l);
#pragma unroll
      for (int n = 0; n < D / 8; ++n)
        *reinterpret_cast<float2 *>(po + 8 * n + 2 * t4) = make_float2(o[n][2 * half], o[n][2 * half + 1]);
      continue;
    }
    // a row that sees nothing: zeros and -inf (NaN scores leave m at -inf too, but not l at 0)
    const bool none = m == -INFINITY && l == 0.f;
    const float inv = none ? 0.f : 1.f / l;
    if (a.lse && t4 == 0) a.lse[at] = none ? -INFINITY : m + log2f(l);
    float *out = reinterpret_cast<float *>(chunk_row(a.out, a, w, r));
#pragma unroll
    for (int n = 0; n < D / 8; ++n) {
      out[8 * n + 2 * t4] = o[n][2 * half] * inv;
      out[8 * n + 2 * t4 + 1] = o[n][2 * half + 1] * inv;
    }
  }
}

} // namespace
} // namespace kvfb
