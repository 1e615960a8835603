// C entry points of the context attention: argument checks, how a call is cut into work items, and its launches.
#include <algorithm>
#include <cmath>
#include <cuda_runtime.h>

#include "../../include/hb_b200.h"
#include "abi_common.h"
#include "context_attn.h"

namespace hb {
namespace {

constexpr int kMaxSplits = 128;        // of a part, where nothing forces more
constexpr int kMaxKeys = 1 << 24;
constexpr int kRowsKernelMax = 32;     // rows of an item up to which it goes to the few-rows kernel

struct Shape {
  int B, Lq, Lkv, Ls, H, Hkv, D, masked;
};

struct Plan {
  CtxPart part[2];
  bool tiles[2];       // the part runs on the tcgen05 kernel
  int rows_per_tile;   // of the few-rows kernel
  int mask_tiles;      // most key tiles of a unit of the tcgen05 kernel
  int slots, prows, tail_rows;
  size_t bytes;        // partial results
};

bool shape_ok(const Shape& s) {
  if (s.B < 1 || s.Lq < 1 || s.Lkv < 0 || s.Ls < 0 || s.H < 1 || s.Hkv < 1 || s.H % s.Hkv) return false;
  if ((s.D != 64 && s.D != 128) || (s.masked != 0 && s.masked != 1)) return false;
  // a kv head's rows over the whole batch, and the items of a call, are counted in 32 bits
  return s.Lkv <= kMaxKeys && s.Ls <= kMaxKeys && s.H < (1 << 16) && s.B <= (1 << 28) / s.H &&
         (int64_t)s.B * s.Lq * s.H < (1ll << 28);
}

int ceil_div(int64_t a, int64_t b) { return static_cast<int>((a + b - 1) / b); }

// Into how many parts the key lists (n tiles each) of the units that a last, partly filled round of CTAs would take
// are cut: the parts' rounds, at 1.5 tiles of fixed cost a unit, and for any cut the merge, about 5 tiles' time
// (a tile: 0.8 us).
int tail_splits(int units, int n, int ctas) {
  int best = 1;
  double best_cost = n + 1.5;
  for (int k = 2; k <= 16 && n / k >= 4; ++k) {
    const double cost = ceil_div((int64_t)units * k, ctas) * (ceil_div(n, k) + 1.5) + 5;
    if (cost < best_cost) {
      best = k;
      best_cost = cost;
    }
  }
  return best;
}

Plan make_plan(const Shape& s) {
  Plan p{};
  const int G = s.H / s.Hkv;
  const int rows = s.Lq * G;
  // One pass over the shared keys for all batch elements pays where an element's rows would leave most of a
  // 128-row tile empty; otherwise each element walks them in the same pass as its own.
  const bool pooled = s.Ls > 0 && s.B > 1 && rows < 128;
  const int rows0 = pooled ? rows * s.B : rows;
  p.rows_per_tile = s.D == 64 && (rows0 <= kRowsKernelMax ? rows0 : rows) > 16 ? 32 : 16;
  auto fill = [&](int i, bool pool, bool sh, bool own, int part_rows) {
    CtxPart& part = p.part[i];
    const bool tiles = p.tiles[i] = part_rows > kRowsKernelMax;
    part.pooled = pool;
    part.use_shared = sh;
    part.use_own = own;
    part.row_tiles = ceil_div(part_rows, tiles ? 128 : p.rows_per_tile);
    const int64_t items = (int64_t)(pool ? 1 : s.B) * s.Hkv * part.row_tiles;
    const int keys = tiles ? ctx_tile_keys(s.D) : 2048 / s.D, ctas = tiles ? ctx_tile_ctas(s.D) : kCtxRowCtas;
    const int chunks = (sh ? ceil_div(s.Ls, keys) : 0) + (own ? ceil_div(s.Lkv, keys) : 0);
    // Few items: the key list is cut so that one round of CTAs fills the GPU, down to 256 keys (or two chunks
    // for each of the four warps) per CTA; the merge then costs less than the idle SMs.
    part.splits = std::max(1, std::min({static_cast<int>(ctas / items), chunks / (tiles ? 256 / keys : 8), kMaxSplits}));
    if (tiles && s.masked) part.splits = std::max(part.splits, ceil_div(chunks, kCtxMaskTiles));
    part.count = static_cast<int>(items * part.splits);
    part.slot0 = p.slots;
    p.slots += part.splits;
    if (tiles && !pooled && part.splits == 1 && items > ctas && items % ctas) {
      // Many items, and a last round that leaves CTAs idle: its items alone are cut.
      const int tail = static_cast<int>(items % ctas), k = tail_splits(tail, chunks, ctas);
      if (k > 1) {
        CtxPart& last = p.part[1] = part;
        part.count = static_cast<int>(items - tail);
        last.item0 = part.count;
        last.splits = k;
        last.count = tail * k;
        p.tiles[1] = true;
        p.tail_rows = 128;
        p.slots = k;
      }
    }
    if (tiles && s.masked) p.mask_tiles = std::max(p.mask_tiles, ceil_div(chunks, part.splits));
  };
  if (pooled) {
    fill(0, true, true, false, rows0);
    if (s.Lkv > 0) fill(1, false, false, true, rows);
  } else {
    fill(0, false, s.Ls > 0, true, rows);
  }
  for (CtxPart& part : p.part) {
    if (part.count == 0) part.splits = part.row_tiles = 1;
    part.by_splits = fast_div(part.splits);
    part.by_row_tiles = fast_div(part.row_tiles);
    part.direct = p.slots == 1 || (p.tail_rows && &part == &p.part[0]);
  }
  if (p.slots > 1) {
    p.prows = p.tail_rows ? p.part[1].count / p.part[1].splits * p.tail_rows : s.B * s.Lq * s.H;
    p.bytes = (size_t)p.slots * p.prows * (s.D + 2) * 4;
  }
  return p;
}

}  // namespace
}  // namespace hb

using namespace hb;

extern "C" int hb_context_workspace_bytes(int batch, int q_len, int kv_len, int shared_len, int num_heads,
                                          int kv_heads, int head_dim, int masked, size_t* bytes) {
  if (!bytes) return HB_ERR_NULL;
  const Shape s{batch, q_len, kv_len, shared_len, num_heads, kv_heads, head_dim, masked};
  if (!shape_ok(s)) return HB_ERR_SHAPE;
  *bytes = make_plan(s).bytes;
  return HB_OK;
}

extern "C" int hb_context_attn(const void* q, int64_t q_batch_stride, int64_t q_row_stride, const void* kv,
                               int64_t kv_batch_stride, int64_t kv_row_stride, const void* shared_kv,
                               int64_t shared_row_stride, const int32_t* lens, const uint8_t* mask,
                               int64_t mask_batch_stride, const uint8_t* shared_mask, const float* q_weight, float eps,
                               float scale, void* out, int64_t out_batch_stride, int64_t out_row_stride, int batch,
                               int q_len, int kv_len, int shared_len, int num_heads, int kv_heads, int head_dim,
                               int dtype, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  if (!q || !out || (kv_len > 0 && !kv) || (shared_len > 0 && !shared_kv)) return HB_ERR_NULL;
  const Shape s{batch, q_len, kv_len, shared_len, num_heads, kv_heads, head_dim, mask || shared_mask ? 1 : 0};
  if (!shape_ok(s) || (dtype != HB_BF16 && dtype != HB_FP16)) return HB_ERR_SHAPE;
  if (!(scale > 0.f) || !std::isfinite(scale) || (q_weight && !(eps >= 0.f))) return HB_ERR_SHAPE;
  const int64_t qw = (int64_t)num_heads * head_dim, kw = 2ll * kv_heads * head_dim;
  if (q_row_stride < qw || out_row_stride < qw || (kv_len > 1 && kv_row_stride < kw) ||
      (shared_len > 1 && shared_row_stride < kw) || q_batch_stride < 0 || kv_batch_stride < 0 ||
      (mask && mask_batch_stride < 0))
    return HB_ERR_SHAPE;
  constexpr int64_t kMaxStride = (1ll << 39) - 1;  // a tensor map's: below 2^40 bytes
  if (kv_batch_stride > kMaxStride || kv_row_stride > kMaxStride || shared_row_stride > kMaxStride) return HB_ERR_SHAPE;
  // no two rows of the output share memory: batch elements one after the other, or interleaved row by row
  if (batch > 1 && out_batch_stride < (q_len - 1) * out_row_stride + qw &&
      (out_batch_stride < qw || out_row_stride < (batch - 1) * out_batch_stride + qw))
    return HB_ERR_SHAPE;
  const void* ptrs[] = {q, kv_len > 0 ? kv : nullptr, shared_len > 0 ? shared_kv : nullptr, out, workspace};
  for (const void* pp : ptrs)
    if (pp && !aligned16(pp)) return HB_ERR_ALIGN;
  if (reinterpret_cast<uintptr_t>(workspace) % 32) return HB_ERR_ALIGN;
  if (q_batch_stride % 8 || q_row_stride % 8 || kv_batch_stride % 8 || kv_row_stride % 8 || shared_row_stride % 8 ||
      out_batch_stride % 8 || out_row_stride % 8)
    return HB_ERR_ALIGN;
  if ((reinterpret_cast<uintptr_t>(lens) & 3u) || (reinterpret_cast<uintptr_t>(q_weight) & 15u)) return HB_ERR_ALIGN;
  // What a tensor map describes: rows of at least their width; batch elements one after the other or interleaved
  // row by row, the larger stride a multiple of the smaller (or all of them the same rows: stride 0).
  const bool inter = batch > 1 && kv_len > 1 && kv_batch_stride > 0 && kv_batch_stride < kv_row_stride;
  if (batch > 1 && kv_len > 0 && kv_batch_stride > 0) {
    if (kv_batch_stride < kw) return HB_ERR_SHAPE;
    if (kv_len > 1 && (inter ? kv_row_stride % kv_batch_stride : kv_batch_stride % kv_row_stride)) return HB_ERR_ALIGN;
  }
  const Plan plan = make_plan(s);
  if (plan.bytes && (!workspace || workspace_bytes < plan.bytes)) return HB_ERR_WORKSPACE;
  const int st = check_device();
  if (st != HB_OK) return st;

  CtxParams p{};
  p.q = static_cast<const uint16_t*>(q);
  p.q_bs = q_batch_stride;
  p.q_rs = q_row_stride;
  p.kv = static_cast<const uint16_t*>(kv);
  p.kv_bs = kv_batch_stride;
  p.kv_rs = kv_len > 1 ? kv_row_stride : std::max(kv_row_stride, kw);
  if (kv_len == 1 && batch > 1 && kv_batch_stride > 0) p.kv_rs = kv_batch_stride;
  p.kv_inter = inter;
  p.skv = static_cast<const uint16_t*>(shared_kv);
  p.skv_rs = shared_len > 1 ? shared_row_stride : std::max(shared_row_stride, kw);
  p.lens = lens;
  p.mask = mask;
  p.mask_bs = mask_batch_stride;
  p.smask = shared_mask;
  p.q_w = q_weight;
  p.eps = eps;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.out = static_cast<uint16_t*>(out);
  p.o_bs = out_batch_stride;
  p.o_rs = out_row_stride;
  p.out_wide = reinterpret_cast<uintptr_t>(out) % 32 == 0 && out_row_stride % 16 == 0 && out_batch_stride % 16 == 0;
  p.B = batch;
  p.Lq = q_len;
  p.H = num_heads;
  p.Hkv = kv_heads;
  p.G = num_heads / kv_heads;
  p.Lkv = kv_len;
  p.Ls = shared_len;
  p.by_lq = fast_div(q_len);
  p.by_g = fast_div(p.G);
  p.by_h = fast_div(num_heads);
  p.by_hkv = fast_div(kv_heads);
  p.slots = plan.slots;
  p.prows = plan.prows;
  p.tail_rows = plan.tail_rows;
  p.o_part = static_cast<float*>(workspace);
  if (plan.bytes) p.ml_part = reinterpret_cast<float2*>(p.o_part + (size_t)plan.slots * plan.prows * head_dim);
  const bool fp16 = dtype == HB_FP16;
  for (int kernel = 0; kernel < 2; ++kernel) {  // the parts of the few-rows kernel, then those of the tcgen05 one
    for (int i = 0; i < 2; ++i) {
      p.part[i] = plan.part[i];
      if (plan.tiles[i] != (kernel == 1)) p.part[i].count = 0;
    }
    if (p.part[0].count + p.part[1].count == 0) continue;
    const int rc = kernel ? launch_ctx_tiles(p, head_dim, fp16, plan.mask_tiles, stream)
                          : launch_ctx_rows(p, head_dim, fp16, plan.rows_per_tile, stream);
    if (rc != HB_OK) return rc;
  }
  p.part[1] = plan.part[1];
  return plan.slots > 1 ? launch_ctx_combine(p, head_dim, fp16, stream) : HB_OK;
}
