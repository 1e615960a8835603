// Internal interface of the context attention: what its kernels (context_attn.cu, context_rows.cu) share.
#pragma once
#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

namespace hb {

// Division of n < 2^31 by a fixed d >= 1: q = umulhi(n, ceil(2^p / d)) >> (p - 32) with p = 31 + ceil(log2 d), exact
// there (the rounded-up reciprocal is off by less than 2^(p - 31) / d parts). d = 1 has p = 31: n itself.
struct FastDiv {
  uint32_t mul;
  int shift;  // p - 32; -1 for d = 1
  __host__ __device__ __forceinline__ int div(int n) const {
#ifdef __CUDA_ARCH__
    return shift < 0 ? n : static_cast<int>(__umulhi(static_cast<uint32_t>(n), mul) >> shift);
#else
    return shift < 0 ? n : static_cast<int>((static_cast<uint64_t>(n) * mul) >> (32 + shift));
#endif
  }
};
inline FastDiv fast_div(int d) {
  int log2 = 0;
  while ((1ll << log2) < d) ++log2;
  if (log2 == 0) return {0u, -1};
  const int p = 31 + log2;
  return {static_cast<uint32_t>(((1ull << p) + d - 1) / d), p - 32};
}

// One kind of work item: the rows of one kv head (query token x query head of its group, token-major) in tiles,
// against a list of keys cut into `splits` parts. Pooled items take the rows of every batch element at once and
// only the shared keys, so those are read once for the whole batch.
struct CtxPart {
  int splits;        // parts of the key list
  int direct;        // 1: the item writes `out`; 0: each part writes its slot of partial results
  int slot0;         // first of them
  int row_tiles;     // tiles of rows of a kv head
  int item0;         // the part's items begin here ((batch element * kv_heads + kv head) * row_tiles + row tile)
  int count;         // work units: items * splits
  int pooled;        // rows of all batch elements
  int use_shared;    // the item's key list holds the shared keys ...
  int use_own;       // ... and the batch element's own
  FastDiv by_splits, by_row_tiles;
};

struct CtxParams {
  const uint16_t* q;      // [batch, q_len, heads * D] by strides (elements)
  int64_t q_bs, q_rs;
  const uint16_t* kv;     // [batch, kv_len, k | v], kv_heads * D each
  int64_t kv_bs, kv_rs;
  int kv_inter;           // batch elements interleaved row by row (kv_bs < kv_rs)
  const uint16_t* skv;    // [shared_len, k | v]
  int64_t skv_rs;
  const int32_t* lens;    // [batch] or null: keys at and past lens[b] are not read
  const uint8_t* mask;    // [batch, kv_len] (row stride mask_bs bytes) or null: keys with 0 are not read
  int64_t mask_bs;
  const uint8_t* smask;   // [shared_len] or null
  const float* q_w;       // [D] or null: RMSNorm weight of the queries
  float eps;
  float scale_log2;       // softmax scale * log2(e)
  uint16_t* out;
  int64_t o_bs, o_rs;
  int out_wide;           // every output row begins on a 32-byte boundary
  int B, Lq, H, Hkv, G, Lkv, Ls;
  FastDiv by_lq, by_g, by_h, by_hkv;
  CtxPart part[2];        // either's `count` may be 0
  // Partial results, merged by the combine kernel: per slot one row for every query token and head, or, where only
  // the last items of part[1] are cut (`tail_rows` > 0 rows per tile), for the rows of those items' tiles.
  int slots, prows, tail_rows;
  float* o_part;          // [slots][prows][D]: sum of p * v
  float2* ml_part;        // [slots][prows]: the exponent that p is relative to (log2; -inf: no key), sum of p
};

// A work unit: tile `rt` of the rows of kv head g (batch element b; all of them where pooled), keys
// [split / splits, (split + 1) / splits) of its list.
struct CtxUnit {
  int split, rt, g, b, item, rows;
};
__device__ __forceinline__ CtxUnit ctx_unit(const CtxParams& p, const CtxPart& part, int u) {
  CtxUnit x;
  const int i = part.by_splits.div(u);
  x.split = u - i * part.splits;
  x.item = part.item0 + i;
  const int bg = part.by_row_tiles.div(x.item);
  x.rt = x.item - bg * part.row_tiles;
  x.b = p.by_hkv.div(bg);
  x.g = bg - x.b * p.Hkv;
  x.rows = (part.pooled ? p.B : 1) * p.Lq * p.G;
  return x;
}

// Where row r of a unit lies: the query's (and the output's) batch element and token, the query head.
struct CtxRow {
  int bq, i, hq;
};
__device__ __forceinline__ CtxRow ctx_row(const CtxParams& p, int r, int g, int b, int pooled) {
  const int tk = p.by_g.div(r);
  CtxRow x;
  x.hq = g * p.G + (r - tk * p.G);
  x.bq = pooled ? p.by_lq.div(tk) : b;
  x.i = pooled ? tk - x.bq * p.Lq : tk;
  return x;
}
// Its row of the partial results; lr: the row within the unit's tile.
__device__ __forceinline__ int64_t ctx_prow(const CtxParams& p, const CtxPart& part, const CtxUnit& u, const CtxRow& x,
                                            int lr) {
  const int row = p.tail_rows ? (u.item - part.item0) * p.tail_rows + lr : (x.bq * p.Lq + x.i) * p.H + x.hq;
  return (int64_t)(part.slot0 + u.split) * p.prows + row;
}

// Own keys of batch element b that may be valid: [0, n).
__device__ __forceinline__ int ctx_own_len(const CtxParams& p, int b) {
  return p.lens ? max(0, min(p.lens[b], p.Lkv)) : p.Lkv;
}

constexpr int kCtxSms = 148;
constexpr int kCtxRowCtas = 2 * kCtxSms;  // CTAs of the few-rows kernel that run at once
// The tcgen05 kernel: keys of a tile, and CTAs that run at once (as many per SM as TMEM holds their S and O for).
constexpr int kCtxTileKeys = 64;
constexpr int ctx_tile_ctas(int D) { return (D == 64 ? 4 : 2) * kCtxSms; }
// Mask bits of a unit's keys are kept in shared memory, for at most this many tiles.
constexpr int kCtxMaskTiles = 256;

// Launchers of the parts whose `count` is not 0: a CUDA error (or a kernel that cannot be launched) returns
// HB_ERR_LAUNCH. The few-rows kernel (context_rows.cu; rows_per_tile 16, or 32 at D 64), the tcgen05 kernel on
// 128-row tiles (context_tiles.cu; `mask_tiles`: the most key tiles of a unit where there is a mask), and the merge
// of partial results (context_rows.cu). `beside`: the few-rows kernel was launched just before.
int launch_ctx_rows(const CtxParams& p, int D, bool fp16, int rows_per_tile, cudaStream_t stream);
int launch_ctx_tiles(const CtxParams& p, int D, bool fp16, int mask_tiles, bool beside, cudaStream_t stream);
int launch_ctx_combine(const CtxParams& p, int D, bool fp16, cudaStream_t stream);

// Read (and clear, when set) the status word of the tcgen05 kernel's translation unit on the current device.
int ctx_tiles_take_status(unsigned int* status);

}  // namespace hb
