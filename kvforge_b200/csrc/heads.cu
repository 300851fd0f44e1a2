// heads.cu - what lies between a model's projections and its KV cache, and back:
// RMS norm and rotation of head vectors, the append of rotated keys and of
// values to the cache, and rows of the cache read back as values.
//
//   norm    y = x * (1 / sqrt(mean(x^2) + eps)) * w        over the D channels of a head
//   rotate  (a, b) -> (a cos - b sin, a sin + b cos)       for pairs (c, c + rot/2) or (2c, 2c + 1)
//   store   the rounding of the cache's format (quantize.cuh), at the token's physical row
//   read    zero + scale * code
//
// All of it is fp32, every operation rounded to nearest and none contracted,
// and the squares are added in a fixed tree (channels 2i and 2i + 1, then
// pairs of those, ...), so the result is the same however the work is spread
// and what lands in a quantized cache is, bit for bit, kvf_b200_quantize of
// the rotated row.
#include "heads.cuh"
#include "quantize.cuh"

#include <algorithm>

namespace kvfb {

// A token of a call in this file fell outside the cache or the rotation table
// (reported as bit 2 of kvf_b200_device_errors).
__device__ unsigned g_kvfb_heads_error;

int device_sm_count();  // decode.cu

namespace {

struct Rows {
  uint8_t *p;
  long long sb, st, sh;  // strides in bytes
  int heads;
  int vec;               // rows start on 16-byte boundaries
};

struct Norm {
  const void *w;
  int dtype;
  float eps;
};

struct HeadsArgs {
  Rows q, q_out, k, v;   // heads = 0: not part of the call
  Norm qn, kn;           // w = NULL: no norm
  const float *cos, *sin;
  int rot, positions, interleaved;
  const int *pos, *lens;
  int B, T;
  int q_units, k_units, units;  // warps per token: of its query heads, of its keys and of its values
  CacheRows cache;
  uint8_t *kd, *vd;
  void *km, *vm;
  int fmt, group;
  int paired;            // queries go by paired_rows
};

__device__ __forceinline__ void load_weight8(const Norm &n, int li, float (&w)[8]) {
  const bool vec = (reinterpret_cast<uintptr_t>(n.w) & 15u) == 0;
  const uint8_t *p = reinterpret_cast<const uint8_t *>(n.w) + 8 * li * dtype_bytes(n.dtype);
  if (n.dtype == KVF_DT_F32)
    load8<KVF_DT_F32>(p, vec, w);
  else if (n.dtype == KVF_DT_F16)
    load8<KVF_DT_F16>(p, vec, w);
  else
    load8<KVF_DT_BF16>(p, vec, w);
}

// Four channels as they lie in memory (8- or 16-byte aligned), and their values.
template <int DT> struct Raw4 {
  uint32_t a[DT == KVF_DT_F32 ? 4 : 2];
};
template <int DT> __device__ __forceinline__ Raw4<DT> load_raw4(const void *p) {
  Raw4<DT> r;
  if constexpr (DT == KVF_DT_F32) {
    const uint4 x = __ldcs(reinterpret_cast<const uint4 *>(p));
    r.a[0] = x.x; r.a[1] = x.y; r.a[2] = x.z; r.a[3] = x.w;
  } else {
    const uint2 x = __ldcs(reinterpret_cast<const uint2 *>(p));
    r.a[0] = x.x; r.a[1] = x.y;
  }
  return r;
}
template <int DT> __device__ __forceinline__ void values4(const Raw4<DT> &r, float *e) {
  if constexpr (DT == KVF_DT_F32) {
#pragma unroll
    for (int k = 0; k < 4; ++k) e[k] = __uint_as_float(r.a[k]);
  } else {
    const float2 x = widen2<DT>(r.a[0]), y = widen2<DT>(r.a[1]);
    e[0] = x.x; e[1] = x.y; e[2] = y.x; e[3] = y.y;
  }
}
template <int DT> __device__ __forceinline__ void store4(void *p, const float *e) {
  if constexpr (DT == KVF_DT_F32)
    *reinterpret_cast<float4 *>(p) = make_float4(e[0], e[1], e[2], e[3]);
  else
    *reinterpret_cast<uint2 *>(p) = make_uint2(narrow2<DT>(e[0], e[1]), narrow2<DT>(e[2], e[3]));
}

// Query rows whose whole width turns in half-split pairs: a lane holds channels
// 4 li .. 4 li + 3 of both halves, so that a pair is one lane's and the rotation
// needs no shuffles (of which the other layout has eight a row, and the
// shared-memory pipe that carries them was as busy as the schedulers: 4 x 4001
// tokens of 64 heads 127 us with them, 98 us without, 81 us at the copy peak). The sum of squares keeps its tree: four
// channels in the lane, neighbours by lane, the halves last.
template <int DT, int D, int R>
__device__ __forceinline__ void paired_rows(const HeadsArgs &a, int b, int j, long long t, int r0, int li) {
  constexpr int LPR = D / 8, RPW = 32 / LPR, E = DT == KVF_DT_F32 ? 4 : 2;
  const int lane = threadIdx.x & 31;
  Raw4<DT> lo[R], hi[R];
  const uint8_t *in = a.q.p + b * a.q.sb + j * a.q.st + 4 * li * E;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const uint8_t *p = in + min(r0 + i * RPW, a.q.heads - 1) * a.q.sh;
    lo[i] = load_raw4<DT>(p);
    hi[i] = load_raw4<DT>(p + (D / 2) * E);
  }
  const float4 c4 = *reinterpret_cast<const float4 *>(a.cos + t * (D / 2) + 4 * li);
  const float4 s4 = *reinterpret_cast<const float4 *>(a.sin + t * (D / 2) + 4 * li);
  const float cs[4] = {c4.x, c4.y, c4.z, c4.w}, sn[4] = {s4.x, s4.y, s4.z, s4.w};
  const bool normed = a.qn.w != nullptr;
  float root = 0.f, w[8];
  if (normed) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int c = (k >> 2) * (D / 2) + 4 * li + (k & 3);
      w[k] = a.qn.dtype == KVF_DT_F32   ? __ldg(reinterpret_cast<const float *>(a.qn.w) + c)
             : a.qn.dtype == KVF_DT_F16 ? __half2float(__ldg(reinterpret_cast<const __half *>(a.qn.w) + c))
                                        : __bfloat162float(__ldg(reinterpret_cast<const __nv_bfloat16 *>(a.qn.w) + c));
    }
    const bool odd = li & 1;
    float mine = 0.f;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      float s[8];
      values4<DT>(lo[i], s);
      values4<DT>(hi[i], s + 4);
#pragma unroll
      for (int k = 0; k < 8; k += 2) mul2(s[k], s[k + 1], s[k], s[k + 1], s[k], s[k + 1]);
      const float x = __fadd_rn(__fadd_rn(s[0], s[1]), __fadd_rn(s[2], s[3]));
      const float y = __fadd_rn(__fadd_rn(s[4], s[5]), __fadd_rn(s[6], s[7]));
      // even lanes go on with the lower half's sum, odd ones with the upper's
      float sum = __fadd_rn(odd ? y : x, __shfl_xor_sync(0xffffffffu, odd ? x : y, 1));
#pragma unroll
      for (int off = 2; off < LPR; off <<= 1) sum = __fadd_rn(sum, __shfl_xor_sync(0xffffffffu, sum, off));
      sum = __fadd_rn(sum, __shfl_xor_sync(0xffffffffu, sum, 1));
      mine = i == 0 || li % R == i ? sum : mine;
    }
    root = __fdiv_rn(1.f, __fsqrt_rn(__fadd_rn(__fmul_rn(mine, 1.f / D), a.qn.eps)));
  }
  uint8_t *out = a.q_out.p + b * a.q_out.sb + j * a.q_out.st + 4 * li * E;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = r0 + i * RPW;
    float x[4], y[4], u[4], v[4];
    values4<DT>(lo[i], x);
    values4<DT>(hi[i], y);
    if (normed) {
      const float inv = R == 1 ? root : __shfl_sync(0xffffffffu, root, (lane & ~(LPR - 1)) + i);
#pragma unroll
      for (int k = 0; k < 4; k += 2) {
        mul2(x[k], x[k + 1], x[k], x[k + 1], inv, inv);
        mul2(x[k], x[k + 1], x[k], x[k + 1], w[k], w[k + 1]);
        mul2(y[k], y[k + 1], y[k], y[k + 1], inv, inv);
        mul2(y[k], y[k + 1], y[k], y[k + 1], w[4 + k], w[5 + k]);
      }
    }
#pragma unroll
    for (int k = 0; k < 4; k += 2) {
      // scalar sums: a packed one may be contracted with its products
      float p0, p1, q0, q1;
      mul2(p0, p1, x[k], x[k + 1], cs[k], cs[k + 1]);
      mul2(q0, q1, y[k], y[k + 1], sn[k], sn[k + 1]);
      u[k] = __fsub_rn(p0, q0);
      u[k + 1] = __fsub_rn(p1, q1);
      mul2(p0, p1, x[k], x[k + 1], sn[k], sn[k + 1]);
      mul2(q0, q1, y[k], y[k + 1], cs[k], cs[k + 1]);
      v[k] = __fadd_rn(p0, q0);
      v[k + 1] = __fadd_rn(p1, q1);
    }
    if (r < a.q.heads) {
      store4<DT>(out + r * a.q_out.sh, u);
      store4<DT>(out + r * a.q_out.sh + (D / 2) * E, v);
    }
  }
}

// One warp takes up to R * (32 / (D / 8)) head vectors of one token and of one
// kind (queries, keys or values), R per group of D / 8 lanes: its weight and the
// token's angles are read once for R rows, R loads are in flight per lane, and
// the R roots are taken by R lanes at once. CACHE: keys and values are part of
// the call.
template <int DT, int D, int R, bool CACHE>
__global__ void __launch_bounds__(256, CACHE ? 5 : 3) heads_kernel(const HeadsArgs a) {
  constexpr int LPR = D / 8;     // lanes per row
  constexpr int RPW = 32 / LPR;  // rows per warp at a time
  const int lane = threadIdx.x & 31;
  const int li = lane % LPR;
  const unsigned wid = blockIdx.x * 8u + (threadIdx.x >> 5);
  const unsigned token = wid / (unsigned)a.units;
  const unsigned bu = token / (unsigned)a.T;
  if (bu >= (unsigned)a.B) return;
  const int b = (int)bu, j = (int)(token - bu * (unsigned)a.T);
  if (a.lens && j >= a.lens[b]) return;
  int unit = (int)(wid - token * (unsigned)a.units), kind = 0;
  if (CACHE && unit >= a.q_units) {
    unit -= a.q_units;
    kind = 1;
    if (unit >= a.k_units) {
      unit -= a.k_units;
      kind = 2;
    }
  }
  const Rows &src = kind == 0 ? a.q : kind == 1 ? a.k : a.v;
  const int r0 = unit * (R * RPW) + lane / LPR;
  const long long t = a.pos ? (long long)a.pos[b] + j : j;
  const bool bad_pos = t < 0 || (a.rot && t >= a.positions);
  if (a.paired && kind == 0) {
    if (!bad_pos)
      paired_rows<DT, D, R>(a, b, j, t, r0, li);
    else if (lane == 0)
      atomicOr(&g_kvfb_heads_error, 1u);
    return;
  }

  // Rows stay as they lie in memory until they are worked on: R of them in
  // flight take 4 R registers (8 R for fp32).
  Raw8<DT> raw[R];
  const uint8_t *in = src.p + b * src.sb + j * src.st + 8 * li * dtype_bytes(DT);
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = min(r0 + i * RPW, src.heads - 1);
    raw[i] = load_raw8<DT>(in + r * src.sh, src.vec);
  }

  const bool turning = kind < 2 && a.rot && !bad_pos;  // the same for the whole warp
  float cs[8], sn[8];
  const int half = a.rot >> 1;
  const bool turns = turning && 8 * li < a.rot, low = 8 * li < half;
  if (turns) {
    // Angles of this lane's channels. Half-split pairs: channel c < rot/2 turns
    // with c + rot/2, rot/16 lanes further; both halves use angle c mod rot/2, and
    // the lower one the sine's negative.
    const float *c = a.cos + t * half, *s = a.sin + t * half;
    if (a.interleaved) {
      const float4 c4 = *reinterpret_cast<const float4 *>(c + 4 * li), s4 = *reinterpret_cast<const float4 *>(s + 4 * li);
      cs[0] = c4.x; cs[1] = c4.y; cs[2] = c4.z; cs[3] = c4.w;
      sn[0] = s4.x; sn[1] = s4.y; sn[2] = s4.z; sn[3] = s4.w;
    } else {
      const int at = low ? 8 * li : 8 * li - half;
#pragma unroll
      for (int k = 0; k < 8; k += 4) {
        const float4 c4 = *reinterpret_cast<const float4 *>(c + at + k), s4 = *reinterpret_cast<const float4 *>(s + at + k);
        cs[k] = c4.x; cs[k + 1] = c4.y; cs[k + 2] = c4.z; cs[k + 3] = c4.w;
        sn[k] = s4.x; sn[k + 1] = s4.y; sn[k + 2] = s4.z; sn[k + 3] = s4.w;
      }
      if (low)
#pragma unroll
        for (int k = 0; k < 8; ++k) sn[k] = -sn[k];
    }
  }

  const Norm &nm = kind == 0 ? a.qn : a.kn;
  const bool normed = kind < 2 && nm.w;
  float root = 0.f, w[8];
  if (normed) {
    load_weight8(nm, li, w);
    float mine = 0.f;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      float s[8];
      values8<DT>(raw[i], s);
#pragma unroll
      for (int k = 0; k < 8; k += 2) mul2(s[k], s[k + 1], s[k], s[k + 1], s[k], s[k + 1]);
      float sum = __fadd_rn(__fadd_rn(__fadd_rn(s[0], s[1]), __fadd_rn(s[2], s[3])),
                            __fadd_rn(__fadd_rn(s[4], s[5]), __fadd_rn(s[6], s[7])));
#pragma unroll
      for (int off = 1; off < LPR; off <<= 1) sum = __fadd_rn(sum, __shfl_xor_sync(0xffffffffu, sum, off));
      mine = i == 0 || li % R == i ? sum : mine;
    }
    root = __fdiv_rn(1.f, __fsqrt_rn(__fadd_rn(__fmul_rn(mine, 1.f / D), nm.eps)));
  }
  const int partner = (lane & ~(LPR - 1)) + (turns ? (low ? li + (a.rot >> 4) : li - (a.rot >> 4)) : li);

  uint8_t *out = nullptr, *data = nullptr;
  uint32_t *meta = nullptr;
  long long row0 = 0, hstep = 0;
  if (!CACHE || kind == 0) {
    if (bad_pos) {
      if (lane == 0) atomicOr(&g_kvfb_heads_error, 1u);
      return;
    }
    out = a.q_out.p + b * a.q_out.sb + j * a.q_out.st + 8 * li * dtype_bytes(DT);
  } else {
    // Heads of a token lie one row apart (token-major) or a whole sequence or page apart.
    row0 = bad_pos ? -1 : a.cache.row(b, 0, t);
    if (row0 < 0) {
      if (lane == 0) atomicOr(&g_kvfb_heads_error, 1u);
      return;
    }
    hstep = !a.cache.head_major ? 1 : a.cache.paged ? 1ll << a.cache.bt_shift : a.cache.n;
    data = kind == 1 ? a.kd : a.vd;
    meta = reinterpret_cast<uint32_t *>(kind == 1 ? a.km : a.vm);
  }

#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = r0 + i * RPW;
    if (__all_sync(0xffffffffu, r >= src.heads)) return;
    const bool live = r < src.heads;
    float e[8];
    values8<DT>(raw[i], e);
    if (normed) {
      const float inv = R == 1 ? root : __shfl_sync(0xffffffffu, root, (lane & ~(LPR - 1)) + i);
#pragma unroll
      for (int k = 0; k < 8; k += 2) {
        mul2(e[k], e[k + 1], e[k], e[k + 1], inv, inv);
        mul2(e[k], e[k + 1], e[k], e[k + 1], w[k], w[k + 1]);
      }
    }
    if (turning) {
      if (a.interleaved) {
        if (turns) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float x = e[2 * k], y = e[2 * k + 1];
            e[2 * k] = __fsub_rn(__fmul_rn(x, cs[k]), __fmul_rn(y, sn[k]));
            e[2 * k + 1] = __fadd_rn(__fmul_rn(x, sn[k]), __fmul_rn(y, cs[k]));
          }
        }
      } else {
        float o[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] = __shfl_sync(0xffffffffu, e[k], partner);
        if (turns) {
#pragma unroll
          for (int k = 0; k < 8; k += 2) {
            mul2(e[k], e[k + 1], e[k], e[k + 1], cs[k], cs[k + 1]);
            mul2(o[k], o[k + 1], o[k], o[k + 1], sn[k], sn[k + 1]);
            // scalar sums: a packed one may be contracted with its products
            e[k] = __fadd_rn(e[k], o[k]);
            e[k + 1] = __fadd_rn(e[k + 1], o[k + 1]);
          }
        }
      }
    }
    if (!CACHE || kind == 0) {
      if (live) store8<DT>(out + r * a.q_out.sh, a.q_out.vec, e);
      continue;
    }
    const long long dr = row0 + r * hstep;
    if (a.fmt == KVF_FMT_F16) {
      if (live) store8<KVF_DT_F16>(data + (dr * D + 8 * li) * 2, true, e);
      continue;
    }
    const GroupScale g = group_scale8(e, li, a.group, a.fmt == KVF_FMT_INT8 ? 255 : 15);
    if (!live) continue;
    if ((li & ((a.group >> 3) - 1)) == 0) meta[(dr * D + 8 * li) >> __popc(a.group - 1)] = g.word;  // group: a power of two
    if (a.fmt == KVF_FMT_INT8)
      store_codes8<KVF_FMT_INT8>(e, g, data + dr * D, li);
    else
      store_codes8<KVF_FMT_INT4>(e, g, data + dr * (D / 2), li);
  }
}

template <int DT, int D>
cudaError_t launch_heads(HeadsArgs a, cudaStream_t st) {
  constexpr int RPW = 32 / (D / 8);
  const long long tokens = (long long)a.B * a.T;
  a.paired = a.q.heads && a.rot == D && !a.interleaved && a.q.vec && a.q_out.vec;
  // Rows per lane group. One in short calls, whose time is that of one row; more
  // where that still gives every SM some 32 warps. Queries alone: eight (four of
  // fp32), if a token's heads fill three quarters of such units (4 x 4001 tokens of
  // 64 heads: 98 us with eight, 113 with four, 132 with two). With keys and values
  // the quantizer needs the registers: two (8 ragged chunks of 2048 tokens into
  // int8: 111 us with two, 123 with four, 148 with eight).
  constexpr int BIG = DT == KVF_DT_F32 ? 4 : 8;
  const bool cache = a.k.heads > 0;
  auto units = [](int heads, int r) { return (heads + r * RPW - 1) / (r * RPW); };
  const long long pairs = units(a.q.heads, 1) + units(a.k.heads, 1) + units(a.v.heads, 1);
  const long long filled = 32LL * device_sm_count();
  int r = tokens * pairs >= 2 * filled ? 2 : 1;
  if (!cache && tokens * pairs >= BIG * filled && 4 * a.q.heads >= 3 * units(a.q.heads, BIG) * BIG * RPW) r = BIG;
  a.q_units = units(a.q.heads, r);
  a.k_units = units(a.k.heads, r);
  a.units = a.q_units + a.k_units + units(a.v.heads, r);
  const long long warps = tokens * a.units;
  if (warps > 0xffffffffLL - 8) return cudaErrorInvalidValue;
  const unsigned blocks = (unsigned)((warps + 7) / 8);
  if (cache && r == 2)
    heads_kernel<DT, D, 2, true><<<blocks, 256, 0, st>>>(a);
  else if (cache)
    heads_kernel<DT, D, 1, true><<<blocks, 256, 0, st>>>(a);
  else if (r == BIG)
    heads_kernel<DT, D, BIG, false><<<blocks, 256, 0, st>>>(a);
  else if (r == 2)
    heads_kernel<DT, D, 2, false><<<blocks, 256, 0, st>>>(a);
  else
    heads_kernel<DT, D, 1, false><<<blocks, 256, 0, st>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_heads(const HeadsArgs &a, int dtype, int d, cudaStream_t st) {
  if (d == 128)
    return dtype == KVF_DT_F32   ? launch_heads<KVF_DT_F32, 128>(a, st)
           : dtype == KVF_DT_F16 ? launch_heads<KVF_DT_F16, 128>(a, st)
                                 : launch_heads<KVF_DT_BF16, 128>(a, st);
  return dtype == KVF_DT_F32   ? launch_heads<KVF_DT_F32, 64>(a, st)
         : dtype == KVF_DT_F16 ? launch_heads<KVF_DT_F16, 64>(a, st)
                               : launch_heads<KVF_DT_BF16, 64>(a, st);
}

Rows rows_of(const kvf_heads *r) {
  if (!r) return Rows{nullptr, 0, 0, 0, 0, 0};
  const long long e = dtype_bytes(r->dtype);
  return Rows{reinterpret_cast<uint8_t *>(r->p), r->stride_b * e, r->stride_t * e, r->stride_h * e, r->heads,
              rows_aligned(*r) ? 1 : 0};
}

cudaError_t check_norm(const kvf_norm *n, Norm &out) {
  out = Norm{nullptr, 0, 0.f};
  if (!n) return cudaSuccess;
  if (!n->weight || n->dtype < KVF_DT_F32 || n->dtype > KVF_DT_BF16 || !(n->eps >= 0.f)) return cudaErrorInvalidValue;
  if (reinterpret_cast<uintptr_t>(n->weight) & (uintptr_t)(dtype_bytes(n->dtype) - 1)) return cudaErrorMisalignedAddress;
  out = Norm{n->weight, n->dtype, n->eps};
  return cudaSuccess;
}

cudaError_t check_rope(const kvf_rope *r, int d, HeadsArgs &a) {
  if (!r) return cudaSuccess;
  if (!r->cos || !r->sin || r->positions <= 0 || r->rot <= 0 || r->rot > d || r->rot % 16 ||
      (r->interleaved != 0 && r->interleaved != 1))
    return cudaErrorInvalidValue;
  if ((reinterpret_cast<uintptr_t>(r->cos) | reinterpret_cast<uintptr_t>(r->sin)) & 15u)
    return cudaErrorMisalignedAddress;
  a.cos = r->cos;
  a.sin = r->sin;
  a.rot = r->rot;
  a.positions = r->positions;
  a.interleaved = r->interleaved;
  return cudaSuccess;
}

// ------------------------------------------------------------------ read back
struct GatherArgs {
  Rows k, v;
  const int *pos, *lens, *seq_lens;
  int B, T, units;
  CacheRows cache;
  const uint8_t *kd, *vd;
  const uint32_t *km, *vm;
  int gpr, group_shift;
};

// One warp takes R * RPW rows of one token, KV heads of k and then of v.
template <int FMT, int DT, int D, int R>
__global__ void __launch_bounds__(256) gather_kernel(const GatherArgs a) {
  constexpr int LPR = D / 8;
  constexpr int RPW = 32 / LPR;
  const int lane = threadIdx.x & 31;
  const int li = lane % LPR;
  const unsigned wid = blockIdx.x * 8u + (threadIdx.x >> 5);
  const unsigned token = wid / (unsigned)a.units;
  const unsigned bu = token / (unsigned)a.T;
  if (bu >= (unsigned)a.B) return;
  const int b = (int)bu, j = (int)(token - bu * (unsigned)a.T);
  if (a.lens && j >= a.lens[b]) return;
  const long long t = a.pos ? (long long)a.pos[b] + j : j;
  if (a.seq_lens && t >= a.seq_lens[b]) return;
  const int Hkv = a.k.heads;
  const long long row0 = a.cache.row(b, 0, t);
  if (row0 < 0) {
    if (lane == 0) atomicOr(&g_kvfb_heads_error, 1u);
    return;
  }
  // Heads of a token lie one row apart (token-major) or a whole sequence or page apart.
  const long long hstep = !a.cache.head_major ? 1 : a.cache.paged ? 1ll << a.cache.bt_shift : a.cache.n;
  const int r0 = (int)(wid - token * (unsigned)a.units) * (R * RPW) + lane / LPR;
  uint4 raw[R];
  uint32_t mw[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = r0 + i * RPW;
    if (r >= 2 * Hkv) continue;
    const bool isv = r >= Hkv;
    const long long row = row0 + (isv ? r - Hkv : r) * hstep;
    const uint8_t *data = isv ? a.vd : a.kd;
    if (FMT == KVF_FMT_F16) {
      raw[i] = __ldcs(reinterpret_cast<const uint4 *>(data + row * (2 * D)) + li);
    } else {
      if (FMT == KVF_FMT_INT8) {
        const uint2 w = __ldcs(reinterpret_cast<const uint2 *>(data + row * D) + li);
        raw[i].x = w.x;
        raw[i].y = w.y;
      } else {
        raw[i].x = __ldcs(reinterpret_cast<const uint32_t *>(data + row * (D / 2)) + li);
      }
      mw[i] = (isv ? a.vm : a.km)[row * a.gpr + ((8 * li) >> a.group_shift)];
    }
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = r0 + i * RPW;
    if (r >= 2 * Hkv) continue;
    const bool isv = r >= Hkv;
    float x[8];
    if (FMT == KVF_FMT_F16) {
      const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 f = widen2<KVF_DT_F16>(w[k]);
        x[2 * k] = f.x;
        x[2 * k + 1] = f.y;
      }
    } else {
      const __half2 m = *reinterpret_cast<const __half2 *>(&mw[i]);
      const float sc = __low2float(m), zero = __high2float(m);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t c = FMT == KVF_FMT_INT8 ? ((k < 4 ? raw[i].x : raw[i].y) >> (8 * (k & 3))) & 255u
                                               : (raw[i].x >> (4 * k)) & 15u;
        // the product is exact in fp32 (11 + 8 bits), so fused or not is the same
        x[k] = __fmaf_rn((float)c, sc, zero);
      }
    }
    const Rows &o = isv ? a.v : a.k;
    store8<DT>(o.p + b * o.sb + j * o.st + (isv ? r - Hkv : r) * o.sh + 8 * li * dtype_bytes(DT), o.vec, x);
  }
}

template <int FMT, int DT, int D>
cudaError_t launch_gather(GatherArgs a, cudaStream_t st) {
  // Rows per lane group: as many as keep three quarters of the lanes busy, four,
  // or eight of the short int4 rows (65536 tokens of 8 heads: 75 us with eight,
  // 80 with four; a ragged f16 batch 64 us with four, 67 with eight).
  constexpr int RPW = 32 / (D / 8), BIG = FMT == KVF_FMT_INT4 ? 8 : 4;
  const int rows = 2 * a.k.heads;
  auto units = [&](int r) { return (rows + r * RPW - 1) / (r * RPW); };
  auto full = [&](int r) { return 4 * rows >= 3 * units(r) * r * RPW; };
  const int r = full(BIG) ? BIG : full(2) ? 2 : 1;
  a.units = units(r);
  const long long warps = (long long)a.B * a.T * a.units;
  if (warps > 0xffffffffLL - 8) return cudaErrorInvalidValue;
  const unsigned blocks = (unsigned)((warps + 7) / 8);
  if (r == BIG)
    gather_kernel<FMT, DT, D, BIG><<<blocks, 256, 0, st>>>(a);
  else if (r == 2)
    gather_kernel<FMT, DT, D, 2><<<blocks, 256, 0, st>>>(a);
  else
    gather_kernel<FMT, DT, D, 1><<<blocks, 256, 0, st>>>(a);
  return cudaGetLastError();
}

template <int FMT>
cudaError_t launch_gather(const GatherArgs &a, int dtype, int d, cudaStream_t st) {
  if (d == 128)
    return dtype == KVF_DT_F32   ? launch_gather<FMT, KVF_DT_F32, 128>(a, st)
           : dtype == KVF_DT_F16 ? launch_gather<FMT, KVF_DT_F16, 128>(a, st)
                                 : launch_gather<FMT, KVF_DT_BF16, 128>(a, st);
  return dtype == KVF_DT_F32   ? launch_gather<FMT, KVF_DT_F32, 64>(a, st)
         : dtype == KVF_DT_F16 ? launch_gather<FMT, KVF_DT_F16, 64>(a, st)
                               : launch_gather<FMT, KVF_DT_BF16, 64>(a, st);
}

} // namespace

// Nonzero if a token fell outside since the last call (then cleared).
unsigned take_heads_errors() {
  unsigned v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_kvfb_heads_error, sizeof(v)) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  if (v) cudaMemcpyToSymbol(g_kvfb_heads_error, &zero, sizeof(zero));
  return v;
}

} // namespace kvfb

using namespace kvfb;

extern "C" cudaError_t kvf_b200_norm_rope(const kvf_heads *x, const kvf_heads *out, int B, int T, int d,
                                          const kvf_rope *rope, const kvf_norm *norm, const int *pos, const int *lens,
                                          cudaStream_t stream) {
  if (B < 0 || T < 0 || (d != 64 && d != 128) || (!rope && !norm)) return cudaErrorInvalidValue;
  if (B == 0 || T == 0) return cudaSuccess;
  if (rope && !pos) return cudaErrorInvalidValue;
  cudaError_t e;
  if ((e = check_heads(x)) != cudaSuccess || (e = check_heads(out)) != cudaSuccess) return e;
  if (x->dtype != out->dtype || x->heads != out->heads) return cudaErrorInvalidValue;
  HeadsArgs a{};
  if ((e = check_rope(rope, d, a)) != cudaSuccess || (e = check_norm(norm, a.qn)) != cudaSuccess) return e;
  a.q = rows_of(x);
  a.q_out = rows_of(out);
  a.k = a.v = rows_of(nullptr);
  a.pos = rope ? pos : nullptr;
  a.lens = lens;
  a.B = B;
  a.T = T;
  return launch_heads(a, x->dtype, d, stream);
}

extern "C" cudaError_t kvf_b200_append_rope(const kvf_args *args, int fmt, int d, int ord, int paged,
                                            const kvf_heads *k, const kvf_heads *v, int T, const kvf_rope *rope,
                                            const kvf_norm *k_norm, const int *pos, const int *lens,
                                            const kvf_heads *q, const kvf_heads *q_out, const kvf_norm *q_norm,
                                            cudaStream_t stream) {
  HeadsArgs a{};
  cudaError_t e;
  if (T < 0) return cudaErrorInvalidValue;
  if ((e = check_cache(args, fmt, d, ord, paged, a.cache, a.group)) != cudaSuccess) return e;
  if (args->B == 0 || T == 0) return cudaSuccess;
  if ((e = check_heads(k)) != cudaSuccess || (e = check_heads(v)) != cudaSuccess) return e;
  if (!pos || k->heads != args->Hkv || v->heads != args->Hkv || k->dtype != v->dtype) return cudaErrorInvalidValue;
  if ((q == nullptr) != (q_out == nullptr) || (!q && q_norm)) return cudaErrorInvalidValue;
  if (q) {
    if ((e = check_heads(q)) != cudaSuccess || (e = check_heads(q_out)) != cudaSuccess) return e;
    if (q->dtype != k->dtype || q_out->dtype != q->dtype || q_out->heads != q->heads) return cudaErrorInvalidValue;
  }
  if ((e = check_rope(rope, d, a)) != cudaSuccess || (e = check_norm(k_norm, a.kn)) != cudaSuccess ||
      (e = check_norm(q_norm, a.qn)) != cudaSuccess)
    return e;
  a.q = rows_of(q);
  a.q_out = rows_of(q_out);
  a.k = rows_of(k);
  a.v = rows_of(v);
  a.pos = pos;
  a.lens = lens;
  a.B = args->B;
  a.T = T;
  a.fmt = fmt;
  a.kd = const_cast<uint8_t *>(args->k);
  a.vd = const_cast<uint8_t *>(args->v);
  a.km = const_cast<void *>(args->k_meta);
  a.vm = const_cast<void *>(args->v_meta);
  return launch_heads(a, k->dtype, d, stream);
}

extern "C" cudaError_t kvf_b200_gather(const kvf_args *args, int fmt, int d, int ord, int paged, int T, const int *pos,
                                       const int *lens, const kvf_heads *k_out, const kvf_heads *v_out,
                                       cudaStream_t stream) {
  GatherArgs a{};
  cudaError_t e;
  int group = 0;
  if (T < 0) return cudaErrorInvalidValue;
  if ((e = check_cache(args, fmt, d, ord, paged, a.cache, group)) != cudaSuccess) return e;
  if (args->B == 0 || T == 0) return cudaSuccess;
  if ((e = check_heads(k_out)) != cudaSuccess || (e = check_heads(v_out)) != cudaSuccess) return e;
  if (k_out->heads != args->Hkv || v_out->heads != args->Hkv || k_out->dtype != v_out->dtype)
    return cudaErrorInvalidValue;
  a.k = rows_of(k_out);
  a.v = rows_of(v_out);
  a.pos = pos;
  a.lens = lens;
  a.seq_lens = args->seq_lens;
  a.B = args->B;
  a.T = T;
  a.kd = args->k;
  a.vd = args->v;
  a.km = reinterpret_cast<const uint32_t *>(args->k_meta);
  a.vm = reinterpret_cast<const uint32_t *>(args->v_meta);
  a.gpr = group ? d / group : 0;
  a.group_shift = group ? args->group_shift : 0;
  return fmt == KVF_FMT_F16    ? launch_gather<KVF_FMT_F16>(a, k_out->dtype, d, stream)
         : fmt == KVF_FMT_INT8 ? launch_gather<KVF_FMT_INT8>(a, k_out->dtype, d, stream)
                               : launch_gather<KVF_FMT_INT4>(a, k_out->dtype, d, stream);
}
