// chunk.cu - attention of a chunk of new tokens over the cache
// (kvf_b200_chunk_attention): checks, the choice of kernel and splits, launches
// and the merge of splits. The kernels are in chunk_tc.cuh (fp16 and bf16
// queries) and chunk_mma.cuh (fp32 queries).
#include "chunk_mma.cuh"
#include "chunk_tc.cuh"

#include <algorithm>
#include <cstdlib>

namespace kvfb {

cudaError_t ensure_kernel_smem(void *fn, uint32_t smem);  // decode.cu
int device_sm_count();                                    // decode.cu
cudaError_t encode_cache_maps(const kvf_args *a, int fmt, int d, int ord, int paged, int tbox, CUtensorMap &k,
                              CUtensorMap &v);            // decode.cu

namespace {

// One warp per (token, query head): out = sum_s o_s 2^(m_s - M) / sum_s l_s 2^(m_s - M).
// Splits that saw nothing have m = -inf and no output.
template <int DT, int D>
__global__ void __launch_bounds__(128) chunk_merge(const ChunkArgs a) {
  const int lane = threadIdx.x & 31;
  const long long at = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (at >= (long long)a.B * a.T * a.H) return;
  const int h = (int)(at % a.H);
  const long long bt = at / a.H;
  const int j = (int)(bt % a.T), b = (int)(bt / a.T);
  if (a.q_lens && j >= a.q_lens[b]) return;
  const float2 *ml = reinterpret_cast<const float2 *>(a.part_ml) + at * a.splits;
  const float *po = a.part_o + at * a.splits * D;
  float m = -INFINITY;
  for (int s = lane; s < a.splits; s += 32) m = fmaxf(m, ml[s].x);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
  float acc[D / 32], l = 0.f;
#pragma unroll
  for (int k = 0; k < D / 32; ++k) acc[k] = 0.f;
  for (int s = 0; s < a.splits; ++s) {
    const float2 x = ml[s];
    if (x.x == -INFINITY && !(x.y != x.y)) continue;
    const float f = exp2f(x.x - (m == -INFINITY ? 0.f : m));
    l = fmaf(x.y, f, l);
#pragma unroll
    for (int k = 0; k < D / 32; ++k) acc[k] = fmaf(po[s * D + lane + 32 * k], f, acc[k]);
  }
  const bool none = m == -INFINITY && l == 0.f;
  const float inv = none ? 0.f : 1.f / l;
  if (a.lse && lane == 0) a.lse[at] = none ? -INFINITY : m + log2f(l);
  using E = Elem<DT>;
  typename E::T *out = reinterpret_cast<typename E::T *>(a.out.p + b * a.out.sb + (long long)j * a.out.st + (long long)h * a.out.sh);
#pragma unroll
  for (int k = 0; k < D / 32; ++k) out[lane + 32 * k] = E::from(acc[k] * inv);
}

template <int DT, int D> void *merge_fn() { return reinterpret_cast<void *>(&chunk_merge<DT, D>); }

template <int FMT> void *mma_fn(int d) {
  return d == 128 ? reinterpret_cast<void *>(&chunk_mma_kernel<FMT, 128>)
                  : reinterpret_cast<void *>(&chunk_mma_kernel<FMT, 64>);
}
struct TcVariant {
  void *fn;
  int threads;
  uint32_t smem;
};
template <int FMT, int DT, int D, bool TWO> TcVariant tc_variant() {
  using L = TcLayout<FMT, D, TWO>;
  return {reinterpret_cast<void *>(&chunk_tc_kernel<FMT, DT, D, TWO>), L::THREADS, L::BYTES};
}
template <int FMT, int DT> TcVariant tc_variant(int d, bool two) {
  if (d == 128) return two ? tc_variant<FMT, DT, 128, true>() : tc_variant<FMT, DT, 128, false>();
  return two ? tc_variant<FMT, DT, 64, true>() : tc_variant<FMT, DT, 64, false>();
}
template <int FMT> TcVariant tc_variant(int dtype, int d, bool two) {
  return dtype == KVF_DT_F16 ? tc_variant<FMT, KVF_DT_F16>(d, two) : tc_variant<FMT, KVF_DT_BF16>(d, two);
}

// Whether the two softmax groups of a tensor-core block take the steps of one
// row tile in turn (as two splits) or a tile each. One tile has no second one
// to hide its softmax behind.
bool one_tile(long long rows, int splits) { return rows <= kTcRows && splits % 2 == 0; }

// Launches fn(a) or fn(a, maps[0], maps[1]).
cudaError_t launch(void *fn, long long blocks, int threads, uint32_t smem, const ChunkArgs &a, CUtensorMap *maps,
                   cudaStream_t st) {
  if (blocks <= 0) return cudaSuccess;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)blocks, 1, 1);
  cfg.blockDim = dim3((unsigned)threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  void *params[] = {const_cast<ChunkArgs *>(&a), maps, maps ? maps + 1 : nullptr};
  return cudaLaunchKernelExC(&cfg, fn, params);
}

ChunkRows chunk_rows(const kvf_heads &r) {
  const long long e = dtype_bytes(r.dtype);
  return ChunkRows{reinterpret_cast<uint8_t *>(r.p), r.stride_b * e, (int)(r.stride_t * e), (int)(r.stride_h * e),
                   rows_aligned(r) ? 1 : 0};
}

// Splits of each tile's tokens. Tensor-core kernel: the blocks run one per SM, and
// a block costs its steps and about six more to start and end. Splits cost a merge,
// about sixteen steps for its launch and one for each 8 MB of partials written or
// read. One row tile without splits leaves a softmax group idle: its steps take
// 1.15 times as long. The count that makes the whole shortest, the least of equals,
// with at most kPartialBytes of partials. Measured against the neighbouring counts
// (int8, 128 channels): 64 x 4 tokens of 64 heads over 16384: 768 us with 4,
// 886 with 1, 816 with 2, 831 with 6; 512 x 16 over 1024: 774 with 1, 962 with 2;
// 64 x 512 over 65536: 74.9 ms with 1, 76.0 with 2; 1 x 2048 tokens of 32 heads
// over 131072: 4.28 ms with 4, 4.57 with 1.
constexpr double kPartialBytes = 512.0 * (1 << 20);
int pick_splits(int B, int T, int H, int Hkv, int n, int d, int dtype) {
  const long long rows = (long long)T * (H / Hkv);
  const int sms = device_sm_count();
  if (dtype == KVF_DT_F32) {
    // two waves of blocks (two per SM), at least four steps of tokens in each
    const long long blocks = (rows + kChunkRows - 1) / kChunkRows * B * Hkv;
    const long long want = (4LL * sms + blocks - 1) / blocks;
    return (int)std::max(1LL, std::min({want, (long long)n / (4 * kChunkTokens), 64LL}));
  }
  const bool one = rows <= kTcRows;
  const long long blocks = (rows + 2 * kTcRows - 1) / (2 * kTcRows) * B * Hkv;
  const int steps = (n + kTcStep - 1) / kTcStep;
  auto waves = [&](int k) { return (double)((blocks * k + sms - 1) / sms); };
  int best = 1;
  double cost = waves(1) * (one ? 1.15 * steps + 6 : steps + 6.0);
  for (int k = 1; k <= std::min(64, std::max(1, steps / 2)); ++k) {
    const int s = one ? 2 * k : k;
    const double bytes = (double)B * T * H * s * (d + 2) * 4;
    if (s == 1 || bytes > kPartialBytes) continue;
    const double x = waves(k) * ((steps + k - 1) / k + 6) + 16 + 2 * bytes / 8e6;
    if (x < cost) {
      cost = x;
      best = s;
    }
  }
  return best;
}

} // namespace

// Nonzero if a bounded wait ran out since the last call (then cleared).
unsigned take_chunk_errors() {
  unsigned v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_kvfb_chunk_error, sizeof(v)) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  if (v) cudaMemcpyToSymbol(g_kvfb_chunk_error, &zero, sizeof(zero));
  return v;
}

} // namespace kvfb

using namespace kvfb;

extern "C" int kvf_b200_chunk_splits(int B, int T, int H, int Hkv, int n, int fmt, int d, int dtype) {
  if (B <= 0 || T <= 0 || H <= 0 || Hkv <= 0 || H % Hkv || n <= 0 || fmt < 0 || fmt > 2 || (d != 64 && d != 128) ||
      dtype < KVF_DT_F32 || dtype > KVF_DT_BF16)
    return 1;
  return pick_splits(B, T, H, Hkv, n, d, dtype);
}

extern "C" cudaError_t kvf_b200_chunk_attention(const kvf_args *args, int fmt, int d, int ord, int paged,
                                                const kvf_heads *q, const kvf_heads *out, int T, const int *q_lens,
                                                int causal, cudaStream_t stream) {
  ChunkArgs a{};
  cudaError_t e;
  int group = 0;
  if (T < 0 || (causal != 0 && causal != 1)) return cudaErrorInvalidValue;
  if ((e = check_cache(args, fmt, d, ord, paged, a.cache, group)) != cudaSuccess) return e;
  if (args->H <= 0 || args->H % args->Hkv || args->splits < 1) return cudaErrorInvalidValue;
  if (args->B == 0 || T == 0) return cudaSuccess;
  if ((e = check_heads(q)) != cudaSuccess || (e = check_heads(out)) != cudaSuccess) return e;
  if (q->heads != args->H || out->heads != args->H || q->dtype != out->dtype) return cudaErrorInvalidValue;
  // 16-bit queries: a row's metadata is copied as one piece (fp32 queries read words)
  if (group && q->dtype != KVF_DT_F32 &&
      ((reinterpret_cast<uintptr_t>(args->k_meta) | reinterpret_cast<uintptr_t>(args->v_meta)) &
       (uintptr_t)(4 * (d / group) - 1)))
    return cudaErrorMisalignedAddress;
  if (paged && (args->block_shift < 4 || args->block_shift > 7 ||
                (long long)args->max_blocks << args->block_shift < args->n))
    return cudaErrorInvalidValue;
  if (args->splits > 1 && (!args->part_o || !args->part_ml)) return cudaErrorInvalidValue;
  if (args->splits > 1 && ((reinterpret_cast<uintptr_t>(args->part_o) & 15u) ||
                           (reinterpret_cast<uintptr_t>(args->part_ml) & 7u)))
    return cudaErrorMisalignedAddress;
  for (const kvf_heads *x : {q, out})
    if (std::llabs(x->stride_t) > 0x1fffffffLL || std::llabs(x->stride_h) > 0x1fffffffLL) return cudaErrorInvalidValue;
  a.q = chunk_rows(*q);
  a.out = chunk_rows(*out);
  a.B = args->B;
  a.T = T;
  a.H = args->H;
  a.g = args->H / args->Hkv;
  if (a.g > 32768) return cudaErrorInvalidValue;
  a.gmul = ((1ull << 32) + a.g - 1) / a.g;
  a.k = args->k;
  a.v = args->v;
  a.km = reinterpret_cast<const uint32_t *>(args->k_meta);
  a.vm = reinterpret_cast<const uint32_t *>(args->v_meta);
  a.gpr = group ? d / group : 0;
  a.group_shift = group ? args->group_shift : 0;
  a.seq_lens = args->seq_lens;
  a.q_lens = q_lens;
  a.causal = causal;
  a.scale_log2 = args->scale_log2;
  a.lse = args->lse;
  a.splits = args->splits;
  a.part_o = args->part_o;
  a.part_ml = args->part_ml;
  if ((long long)T * a.g > (1LL << 30) || args->n > (1 << 30)) return cudaErrorInvalidValue;
  if (q->dtype == KVF_DT_F32) {
    void *fn = fmt == KVF_FMT_F16    ? mma_fn<KVF_FMT_F16>(d)
               : fmt == KVF_FMT_INT8 ? mma_fn<KVF_FMT_INT8>(d)
                                     : mma_fn<KVF_FMT_INT4>(d);
    const uint32_t smem = (uint32_t)chunk_mma_smem(d);
    a.tiles = (T * a.g + kChunkRows - 1) / kChunkRows;
    if ((e = ensure_kernel_smem(fn, smem)) != cudaSuccess) return e;
    e = launch(fn, (long long)a.tiles * a.B * a.cache.Hkv * a.splits, kChunkThreads, smem, a, nullptr, stream);
  } else {
    const bool two = !one_tile((long long)T * a.g, a.splits);
    const TcVariant x = fmt == KVF_FMT_F16    ? tc_variant<KVF_FMT_F16>(q->dtype, d, two)
                        : fmt == KVF_FMT_INT8 ? tc_variant<KVF_FMT_INT8>(q->dtype, d, two)
                                              : tc_variant<KVF_FMT_INT4>(q->dtype, d, two);
    a.tiles = (T * a.g + 2 * kTcRows - 1) / (2 * kTcRows);
    CUtensorMap maps[2];
    const int tbox = paged ? std::min(kTcHalf, 1 << args->block_shift) : kTcHalf;
    if ((e = encode_cache_maps(args, fmt, d, ord, paged, tbox, maps[0], maps[1])) != cudaSuccess) return e;
    if ((e = ensure_kernel_smem(x.fn, x.smem)) != cudaSuccess) return e;
    e = launch(x.fn, (long long)a.tiles * a.B * a.cache.Hkv * (two ? a.splits : a.splits / 2), x.threads, x.smem, a, maps,
               stream);
  }
  if (e != cudaSuccess || a.splits == 1) return e;
  void *mf = d == 128 ? (q->dtype == KVF_DT_F32   ? merge_fn<KVF_DT_F32, 128>()
                         : q->dtype == KVF_DT_F16 ? merge_fn<KVF_DT_F16, 128>()
                                                  : merge_fn<KVF_DT_BF16, 128>())
                      : (q->dtype == KVF_DT_F32   ? merge_fn<KVF_DT_F32, 64>()
                         : q->dtype == KVF_DT_F16 ? merge_fn<KVF_DT_F16, 64>()
                                                  : merge_fn<KVF_DT_BF16, 64>());
  return launch(mf, ((long long)a.B * T * a.H + 3) / 4, 128, 0, a, nullptr, stream);
}
