// Internal interface of the context attention: what its kernels (context_attn.cu, context_rows.cu) share.
#pragma once
#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

namespace hb {

// One kind of work item: the rows of one kv head (query token x query head of its group, token-major) in tiles,
// against a list of keys cut into `splits` parts. Pooled items take the rows of every batch element at once and
// only the shared keys, so those are read once for the whole batch.
struct CtxPart {
  int splits;       // parts of the key list; each writes its own slot of partial results
  int slot0;        // first of them
  int row_tiles;    // tiles of rows of an item
  int ctas;         // (pooled ? 1 : batch) * kv_heads * row_tiles * splits
  int pooled;       // rows of all batch elements
  int use_shared;   // the item's key list holds the shared keys ...
  int use_own;      // ... and the batch element's own
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
  int B, Lq, H, Hkv, G, Lkv, Ls;
  CtxPart part[2];        // the second's `ctas` may be 0
  int slots;              // 1: the kernel writes `out`; more: partial results, merged by the combine kernel
  float* o_part;          // [slots][B * Lq * H][D], each normalised by nothing: sum of p * v
  float2* ml_part;        // [slots][B * Lq * H]: running maximum (log2 units), sum of p
};

// Own keys of batch element b that may be valid: [0, n).
__device__ __forceinline__ int ctx_own_len(const CtxParams& p, int b) {
  return p.lens ? max(0, min(p.lens[b], p.Lkv)) : p.Lkv;
}

// Mask bits of a CTA's keys are kept in its shared memory, 16 bytes per 128 keys, for at most this many tiles.
constexpr int kCtxMaskTiles = 512;

// Launchers of the parts whose `ctas` is not 0: a CUDA error (or a kernel that cannot be launched) returns
// HB_ERR_LAUNCH. The few-rows kernel (context_rows.cu; rows_per_tile 16, or 32 at D 64), the tcgen05 kernel on
// 128-row tiles (context_tiles.cu; `mask_tiles`: the most key tiles of a CTA where there is a mask), and the merge
// of partial results (context_rows.cu).
int launch_ctx_rows(const CtxParams& p, int D, bool fp16, int rows_per_tile, cudaStream_t stream);
int launch_ctx_tiles(const CtxParams& p, int D, bool fp16, int mask_tiles, cudaStream_t stream);
int launch_ctx_combine(const CtxParams& p, int D, bool fp16, cudaStream_t stream);

// Read (and clear, when set) the status word of the tcgen05 kernel's translation unit on the current device.
int ctx_tiles_take_status(unsigned int* status);

}  // namespace hb
