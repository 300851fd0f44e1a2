// chunk.cuh - attention of a chunk of new tokens over the cache: arguments,
// lengths, masks and cache rows shared by its kernels.
//
//   s[r][t] = scale * q_r . k_t                 t < seen(r)
//   out[r]  = sum_t softmax(s[r])_t v_t         0 where seen(r) = 0
//   lse[r]  = log2 sum_t 2^(s[r][t] log2 e)
//
// A block takes a tile of rows of one (sequence, KV head): row r is query head
// r mod g of new token r / g (g query heads share the KV head, so a tile's K
// and V rows are read once for all of them). With kv tokens stored and ql new
// ones, token j is token kv - ql + j of its sequence: seen = kv - ql + j + 1
// (causal) or kv. Few tiles over a long cache are split along the tokens; the
// splits' unnormalised outputs, maxima and sums are combined by chunk_merge.
#pragma once

#include "heads.cuh"
#include "ptx.cuh"
#include "quantize.cuh"

namespace kvfb {
namespace {

struct ChunkRows {
  uint8_t *p;
  long long sb;          // strides in bytes
  int st, sh;
  int vec;               // rows start on 16-byte boundaries
};

struct ChunkArgs {
  ChunkRows q, out;
  int B, T, H, g;
  unsigned long long gmul;  // ceil(2^32 / g): x / g = x * gmul >> 32 for x < 2^16, g < 2^16
  CacheRows cache;       // Hkv, n
  const uint8_t *k, *v;
  const uint32_t *km, *vm;
  int gpr, group_shift;
  const int *seq_lens, *q_lens;
  int causal;
  float scale_log2;
  float *lse;            // [B][T][H] or null
  int splits, tiles;     // tiles: row tiles of a sequence's T tokens
  float *part_o;         // [B][T][H][splits][D]
  float *part_ml;        // [B][T][H][splits][2]
};

// What a block works on: sequence, KV head, first row, lengths, and its range
// of tokens [t0, t1).
struct ChunkWork {
  int b, h, row0, rows;  // rows: valid rows from row0 on (<= tile height)
  int ql, kv, split;
  int t0, t1;
  int seen0;             // tokens that row0 sees
  int j0, g0;            // token and query head (within the group) of row0
};

// Token (from w.j0 on) and query head of row r of the tile.
__device__ __forceinline__ void chunk_at(const ChunkArgs &a, const ChunkWork &w, int r, int &j, int &head) {
  const unsigned x = (unsigned)(w.g0 + r);
  j = (int)(x * a.gmul >> 32);
  head = (int)x - j * a.g;
}

// Tokens that row r of the tile sees.
__device__ __forceinline__ int chunk_seen(const ChunkArgs &a, const ChunkWork &w, int r) {
  if (!a.causal) return w.kv;
  int j, head;
  chunk_at(a, w, r, j, head);
  return max(0, w.kv - w.ql + w.j0 + j + 1);
}

// False if the block has no rows. Longest rows first: the tiles of a sequence
// are taken from its end, where a causal tile sees most. A tile's tokens are
// shared evenly among `splits` blocks in whole steps of `step` tokens.
__device__ __forceinline__ bool chunk_work(const ChunkArgs &a, int splits, int height, int step, ChunkWork &w) {
  unsigned i = blockIdx.x;
  w.split = (int)(i % (unsigned)splits);
  i /= (unsigned)splits;
  w.h = (int)(i % (unsigned)a.cache.Hkv);
  i /= (unsigned)a.cache.Hkv;
  w.b = (int)(i % (unsigned)a.B);
  const int tile = a.tiles - 1 - (int)(i / (unsigned)a.B);
  w.ql = a.q_lens ? min(max(a.q_lens[w.b], 0), a.T) : a.T;
  w.kv = a.seq_lens ? min(max(a.seq_lens[w.b], 0), a.cache.n) : a.cache.n;
  w.row0 = tile * height;
  w.rows = min(height, w.ql * a.g - w.row0);
  if (w.rows <= 0) return false;
  w.j0 = w.row0 / a.g;
  w.g0 = w.row0 - w.j0 * a.g;
  const int seen = chunk_seen(a, w, w.rows - 1);
  const int steps = (seen + step - 1) / step;
  const int each = (steps + splits - 1) / splits;
  w.t0 = (int)min((long long)w.split * each * step, (long long)seen);
  w.t1 = (int)min((long long)w.t0 + (long long)each * step, (long long)seen);
  w.seen0 = chunk_seen(a, w, 0);
  return true;
}

// Row r of the tile in q or out. Strides between tokens and heads fit 32 bits.
__device__ __forceinline__ uint8_t *chunk_row(const ChunkRows &x, const ChunkArgs &a, const ChunkWork &w, int r) {
  int j, head;
  chunk_at(a, w, r, j, head);
  uint8_t *base = x.p + w.b * x.sb + (long long)w.j0 * x.st + (long long)(w.h * a.g) * x.sh;
  return base + (long long)j * x.st + (long long)head * x.sh;
}

// Index of row r in lse and in the split partials.
__device__ __forceinline__ long long chunk_index(const ChunkArgs &a, const ChunkWork &w, int r) {
  int j, head;
  chunk_at(a, w, r, j, head);
  return ((long long)w.b * a.T + w.j0) * a.H + w.h * a.g + (long long)j * a.H + head;
}

// Whether one of a word's two fp16 numbers is infinite or NaN: an exponent of ones
// carries into the sign's place.
__device__ __forceinline__ uint32_t odd_halves(uint32_t w) { return ((w & 0x7C007C00u) + 0x04000400u) & 0x80008000u; }

// Eight channels of cache row `row` (from channel 8 * li) as fp32. Nonzero if one
// of them can be infinite or NaN (of a quantized cache: its scale or zero is).
template <int FMT, int D>
__device__ __forceinline__ uint32_t cache8(const uint8_t *data, const uint32_t *meta, const ChunkArgs &a, long long row,
                                           int li, float (&x)[8]) {
  if (FMT == KVF_FMT_F16) {
    const uint4 r = __ldg(reinterpret_cast<const uint4 *>(data + row * (2 * D)) + li);
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 f = widen2<KVF_DT_F16>(w[k]);
      x[2 * k] = f.x;
      x[2 * k + 1] = f.y;
    }
    return odd_halves(w[0]) | odd_halves(w[1]) | odd_halves(w[2]) | odd_halves(w[3]);
  }
  uint2 r;
  if (FMT == KVF_FMT_INT8) {
    r = __ldg(reinterpret_cast<const uint2 *>(data + row * D) + li);
  } else {
    r.x = __ldg(reinterpret_cast<const uint32_t *>(data + row * (D / 2)) + li);
    r.y = 0;
  }
  const uint32_t m = __ldg(meta + row * a.gpr + ((8 * li) >> a.group_shift));
  const __half2 sz = *reinterpret_cast<const __half2 *>(&m);
  const float sc = __low2float(sz), zero = __high2float(sz);
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const uint32_t c = FMT == KVF_FMT_INT8 ? ((k < 4 ? r.x : r.y) >> (8 * (k & 3))) & 255u : (r.x >> (4 * k)) & 15u;
    x[k] = __fmaf_rn((float)c, sc, zero);
  }
  return odd_halves(m);
}

} // namespace
} // namespace kvfb
