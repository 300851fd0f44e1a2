// heads.cuh - head vectors of a model's activations (kvf_heads): element types,
// strides, and eight channels of a row at a time; checks of the arguments that
// the calls around the cache share.
#pragma once

#include "quantize.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstdint>

namespace kvfb {
namespace {

__host__ __device__ constexpr int dtype_bytes(int dt) { return dt == KVF_DT_F32 ? 4 : 2; }

template <int DT> struct Elem;
template <> struct Elem<KVF_DT_F32> {
  using T = float;
  static __device__ __forceinline__ float to(float x) { return x; }
  static __device__ __forceinline__ float from(float x) { return x; }
};
template <> struct Elem<KVF_DT_F16> {
  using T = __half;
  static __device__ __forceinline__ float to(__half x) { return __half2float(x); }
  static __device__ __forceinline__ __half from(float x) { return __float2half_rn(x); }
};
template <> struct Elem<KVF_DT_BF16> {
  using T = __nv_bfloat16;
  static __device__ __forceinline__ float to(__nv_bfloat16 x) { return __bfloat162float(x); }
  static __device__ __forceinline__ __nv_bfloat16 from(float x) { return __float2bfloat16_rn(x); }
};

// Two 16-bit values of a word as fp32, and back (round to nearest even).
template <int DT> __device__ __forceinline__ float2 widen2(uint32_t w) {
  if (DT == KVF_DT_BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  const __half2 h = *reinterpret_cast<const __half2 *>(&w);
  return __half22float2(h);
}
template <int DT> __device__ __forceinline__ uint32_t narrow2(float a, float b) {
  uint32_t w;
  if (DT == KVF_DT_BF16)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(b), "f"(a));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(b), "f"(a));
  return w;
}

// Eight consecutive channels at p; `vec`: p is 16-byte aligned.
template <int DT> __device__ __forceinline__ void load8(const void *p, bool vec, float (&e)[8]) {
  using T = typename Elem<DT>::T;
  if (!vec) {
#pragma unroll
    for (int k = 0; k < 8; ++k) e[k] = Elem<DT>::to(reinterpret_cast<const T *>(p)[k]);
  } else if (DT == KVF_DT_F32) {
    const float4 a = __ldcs(reinterpret_cast<const float4 *>(p)), b = __ldcs(reinterpret_cast<const float4 *>(p) + 1);
    e[0] = a.x; e[1] = a.y; e[2] = a.z; e[3] = a.w;
    e[4] = b.x; e[5] = b.y; e[6] = b.z; e[7] = b.w;
  } else {
    const uint4 a = __ldcs(reinterpret_cast<const uint4 *>(p));
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 f = widen2<DT>(w[k]);
      e[2 * k] = f.x;
      e[2 * k + 1] = f.y;
    }
  }
}

// Eight channels as they lie in memory, and their values.
template <int DT> struct Raw8 {
  uint4 a[DT == KVF_DT_F32 ? 2 : 1];
};
template <int DT> __device__ __forceinline__ Raw8<DT> load_raw8(const void *p, bool vec) {
  Raw8<DT> r;
  if (vec) {
#pragma unroll
    for (int k = 0; k < (DT == KVF_DT_F32 ? 2 : 1); ++k) r.a[k] = __ldcs(reinterpret_cast<const uint4 *>(p) + k);
  } else if (DT == KVF_DT_F32) {
    const uint32_t *e = reinterpret_cast<const uint32_t *>(p);
#pragma unroll
    for (int k = 0; k < (DT == KVF_DT_F32 ? 2 : 1); ++k) r.a[k] = make_uint4(e[4 * k], e[4 * k + 1], e[4 * k + 2], e[4 * k + 3]);
  } else {
    const uint16_t *e = reinterpret_cast<const uint16_t *>(p);
    r.a[0] = make_uint4(e[0] | (uint32_t)e[1] << 16, e[2] | (uint32_t)e[3] << 16, e[4] | (uint32_t)e[5] << 16,
                        e[6] | (uint32_t)e[7] << 16);
  }
  return r;
}
template <int DT> __device__ __forceinline__ void values8(const Raw8<DT> &r, float (&e)[8]) {
  if (DT == KVF_DT_F32) {
#pragma unroll
    for (int k = 0; k < (DT == KVF_DT_F32 ? 2 : 1); ++k) {
      e[4 * k] = __uint_as_float(r.a[k].x);
      e[4 * k + 1] = __uint_as_float(r.a[k].y);
      e[4 * k + 2] = __uint_as_float(r.a[k].z);
      e[4 * k + 3] = __uint_as_float(r.a[k].w);
    }
  } else {
    const uint32_t w[4] = {r.a[0].x, r.a[0].y, r.a[0].z, r.a[0].w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 f = widen2<DT>(w[k]);
      e[2 * k] = f.x;
      e[2 * k + 1] = f.y;
    }
  }
}

// Two products, each rounded to nearest, in one instruction.
__device__ __forceinline__ void mul2(float &x, float &y, float a, float b, float c, float d) {
  asm("{\n\t.reg .b64 u, v, w;\n\tmov.b64 u, {%2, %3};\n\tmov.b64 v, {%4, %5};\n\tmul.rn.f32x2 w, u, v;\n\t"
      "mov.b64 {%0, %1}, w;\n\t}"
      : "=f"(x), "=f"(y)
      : "f"(a), "f"(b), "f"(c), "f"(d));
}
template <int DT> __device__ __forceinline__ void store8(void *p, bool vec, const float (&e)[8]) {
  using T = typename Elem<DT>::T;
  if (!vec) {
#pragma unroll
    for (int k = 0; k < 8; ++k) reinterpret_cast<T *>(p)[k] = Elem<DT>::from(e[k]);
  } else if (DT == KVF_DT_F32) {
    reinterpret_cast<float4 *>(p)[0] = make_float4(e[0], e[1], e[2], e[3]);
    reinterpret_cast<float4 *>(p)[1] = make_float4(e[4], e[5], e[6], e[7]);
  } else {
    uint4 a;
    a.x = narrow2<DT>(e[0], e[1]);
    a.y = narrow2<DT>(e[2], e[3]);
    a.z = narrow2<DT>(e[4], e[5]);
    a.w = narrow2<DT>(e[6], e[7]);
    *reinterpret_cast<uint4 *>(p) = a;
  }
}

// Whether every row of `r` starts on a 16-byte boundary.
inline bool rows_aligned(const kvf_heads &r) {
  const long long e = dtype_bytes(r.dtype);
  return ((reinterpret_cast<uintptr_t>(r.p) | (uintptr_t)(r.stride_b * e) | (uintptr_t)(r.stride_t * e) |
           (uintptr_t)(r.stride_h * e)) & 15u) == 0;
}

// Whether `r` names rows of a known type on their natural alignment.
inline cudaError_t check_heads(const kvf_heads *r) {
  if (!r || !r->p || r->dtype < KVF_DT_F32 || r->dtype > KVF_DT_BF16 || r->heads <= 0) return cudaErrorInvalidValue;
  if (reinterpret_cast<uintptr_t>(r->p) & (uintptr_t)(dtype_bytes(r->dtype) - 1)) return cudaErrorMisalignedAddress;
  return cudaSuccess;
}

// The cache half of a call's arguments: placement, payload and metadata, in
// the formats that kvf_b200_decode reads.
inline cudaError_t check_cache(const kvf_args *a, int fmt, int d, int ord, int paged, CacheRows &rows, int &group) {
  if (!a || (d != 64 && d != 128) || fmt < 0 || fmt > 2 || (ord != KVF_ORD_HEAD && ord != KVF_ORD_TOKEN) ||
      (paged != 0 && paged != 1) || a->B < 0 || a->Hkv <= 0 || a->n <= 0)
    return cudaErrorInvalidValue;
  group = 0;
  if (fmt != KVF_FMT_F16) {
    if (a->group_shift < 5 || a->group_shift > 7) return cudaErrorInvalidValue;
    group = 1 << a->group_shift;
    if (group > d || (fmt == KVF_FMT_INT8 && group < 64)) return cudaErrorInvalidValue;
  }
  if (paged && (a->block_shift < 0 || a->block_shift > 20 || a->max_blocks <= 0)) return cudaErrorInvalidValue;
  if (a->B == 0) return cudaSuccess;
  if (!a->k || !a->v || (group && (!a->k_meta || !a->v_meta)) || (paged && !a->block_table))
    return cudaErrorInvalidValue;
  if ((reinterpret_cast<uintptr_t>(a->k) | reinterpret_cast<uintptr_t>(a->v)) & 15u) return cudaErrorMisalignedAddress;
  if (group && ((reinterpret_cast<uintptr_t>(a->k_meta) | reinterpret_cast<uintptr_t>(a->v_meta)) & 3u))
    return cudaErrorMisalignedAddress;
  rows = CacheRows{a->block_table, a->Hkv, a->n, ord == KVF_ORD_HEAD ? 1 : 0, paged, paged ? a->block_shift : 0,
                   paged ? a->max_blocks : 0};
  return cudaSuccess;
}

} // namespace
} // namespace kvfb
