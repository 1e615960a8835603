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
  bool too_large;      // work units do not fit 32 bits
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
  // 128-row tile empty and the passes saved weigh more than the launches and the merge that it takes (about 10 us, in
  // which 32 MiB of keys come out of L2 again); otherwise each element walks them in the same pass as its own.
  const bool pooled = s.B > 1 && rows < 128 && (int64_t)(s.B - 1) * s.Ls * s.Hkv * s.D * 4 > (32ll << 20);
  const int rows0 = pooled ? rows * s.B : rows;
  p.rows_per_tile = s.D == 64 && (rows0 <= kRowsKernelMax ? rows0 : rows) > 16 ? 32 : 16;
  auto fill = [&](int i, bool pool, bool sh, bool own, int part_rows) {
    CtxPart& part = p.part[i];
    const bool any = (sh && s.Ls > 0) || (own && s.Lkv > 0);  // without a key there is no tensor map to make
    const bool tiles = p.tiles[i] = part_rows > kRowsKernelMax && any;
    part.pooled = pool;
    part.use_shared = sh;
    part.use_own = own;
    part.row_tiles = ceil_div(part_rows, tiles ? 128 : p.rows_per_tile);
    const int64_t items = (int64_t)(pool ? 1 : s.B) * s.Hkv * part.row_tiles;
    const int keys = tiles ? kCtxTileKeys : 2048 / s.D, ctas = tiles ? ctx_tile_ctas(s.D) : kCtxRowCtas;
    const int chunks = (sh ? ceil_div(s.Ls, keys) : 0) + (own ? ceil_div(s.Lkv, keys) : 0);
    // Few items: the key list is cut so that one round of CTAs fills the GPU, down to 256 keys (or two chunks for each
    // of the four warps) per CTA. Below 24 chunks the few-rows kernel walks the list whole in the time that the merge
    // takes (17 tokens of 234 keys at D 128: 6.3 us whole, 7.5 cut; one token of 1,000 keys: 8.0 whole, 5.8 cut).
    part.splits = std::max(1, std::min({static_cast<int>(ctas / items), chunks / (tiles ? 256 / keys : 8), kMaxSplits}));
    if (!tiles && chunks < 24) part.splits = 1;
    if (tiles && s.masked) part.splits = std::max(part.splits, ceil_div(chunks, kCtxMaskTiles));
    if (items * part.splits >= (1ll << 30)) p.too_large = true;
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
  const Plan plan = make_plan(s);
  if (plan.too_large) return HB_ERR_SHAPE;
  *bytes = plan.bytes;
  return HB_OK;
}

extern "C" int hb_context_attn(const HbContextArgs* args, cudaStream_t stream) {
  if (!args) return HB_ERR_NULL;
  const HbContextArgs& a = *args;
  if (!a.q || !a.out || (a.kv_len > 0 && !a.kv) || (a.shared_len > 0 && !a.shared_kv)) return HB_ERR_NULL;
  const Shape s{a.batch,     a.q_len,    a.kv_len,   a.shared_len,
                a.num_heads, a.kv_heads, a.head_dim, a.mask || a.shared_mask ? 1 : 0};
  if (!shape_ok(s) || (a.dtype != HB_BF16 && a.dtype != HB_FP16)) return HB_ERR_SHAPE;
  if (!(a.scale > 0.f) || !std::isfinite(a.scale) || (a.q_weight && !(a.eps >= 0.f))) return HB_ERR_SHAPE;
  const int64_t qw = (int64_t)a.num_heads * a.head_dim, kw = 2ll * a.kv_heads * a.head_dim;
  if (a.q_row_stride < qw || a.out_row_stride < qw || (a.kv_len > 1 && a.kv_row_stride < kw) ||
      (a.shared_len > 1 && a.shared_row_stride < kw) || a.q_batch_stride < 0 || a.kv_batch_stride < 0 ||
      (a.mask && a.mask_batch_stride < 0))
    return HB_ERR_SHAPE;
  constexpr int64_t kMaxStride = (1ll << 39) - 1;  // a tensor map's: below 2^40 bytes
  if (a.kv_batch_stride > kMaxStride || a.kv_row_stride > kMaxStride || a.shared_row_stride > kMaxStride)
    return HB_ERR_SHAPE;
  // no two rows of the output share memory: batch elements one after the other, or interleaved row by row
  if (a.batch > 1 && a.out_batch_stride < (a.q_len - 1) * a.out_row_stride + qw &&
      (a.out_batch_stride < qw || a.out_row_stride < (a.batch - 1) * a.out_batch_stride + qw))
    return HB_ERR_SHAPE;
  const void* ptrs[] = {a.q, a.kv_len > 0 ? a.kv : nullptr, a.shared_len > 0 ? a.shared_kv : nullptr, a.out,
                        a.workspace};
  for (const void* pp : ptrs)
    if (pp && !aligned16(pp)) return HB_ERR_ALIGN;
  if (reinterpret_cast<uintptr_t>(a.workspace) % 32) return HB_ERR_ALIGN;
  if (a.q_batch_stride % 8 || a.q_row_stride % 8 || a.kv_batch_stride % 8 || a.kv_row_stride % 8 ||
      a.shared_row_stride % 8 || a.out_batch_stride % 8 || a.out_row_stride % 8)
    return HB_ERR_ALIGN;
  if ((reinterpret_cast<uintptr_t>(a.lens) & 3u) || (reinterpret_cast<uintptr_t>(a.q_weight) & 15u)) return HB_ERR_ALIGN;
  // What a tensor map describes: rows of at least their width; batch elements one after the other or interleaved
  // row by row, the larger stride a multiple of the smaller (or all of them the same rows: stride 0).
  const bool inter = a.batch > 1 && a.kv_len > 1 && a.kv_batch_stride > 0 && a.kv_batch_stride < a.kv_row_stride;
  if (a.batch > 1 && a.kv_len > 0 && a.kv_batch_stride > 0) {
    if (a.kv_batch_stride < kw) return HB_ERR_SHAPE;
    if (a.kv_len > 1 && (inter ? a.kv_row_stride % a.kv_batch_stride : a.kv_batch_stride % a.kv_row_stride))
      return HB_ERR_ALIGN;
  }
  const Plan plan = make_plan(s);
  if (plan.too_large) return HB_ERR_SHAPE;
  if (plan.bytes && (!a.workspace || a.workspace_bytes < 0 || static_cast<size_t>(a.workspace_bytes) < plan.bytes))
    return HB_ERR_WORKSPACE;
  const int st = check_device();
  if (st != HB_OK) return st;

  CtxParams p{};
  p.q = static_cast<const uint16_t*>(a.q);
  p.q_bs = a.q_batch_stride;
  p.q_rs = a.q_row_stride;
  p.kv = static_cast<const uint16_t*>(a.kv);
  p.kv_bs = a.kv_batch_stride;
  p.kv_rs = a.kv_len > 1 ? a.kv_row_stride : std::max(a.kv_row_stride, kw);
  if (a.kv_len == 1 && a.batch > 1 && a.kv_batch_stride > 0) p.kv_rs = a.kv_batch_stride;
  p.kv_inter = inter;
  p.skv = static_cast<const uint16_t*>(a.shared_kv);
  p.skv_rs = a.shared_len > 1 ? a.shared_row_stride : std::max(a.shared_row_stride, kw);
  p.lens = a.lens;
  p.mask = a.mask;
  p.mask_bs = a.mask_batch_stride;
  p.smask = a.shared_mask;
  p.q_w = a.q_weight;
  p.eps = a.eps;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.out = static_cast<uint16_t*>(a.out);
  p.o_bs = a.out_batch_stride;
  p.o_rs = a.out_row_stride;
  p.out_wide =
      reinterpret_cast<uintptr_t>(a.out) % 32 == 0 && a.out_row_stride % 16 == 0 && a.out_batch_stride % 16 == 0;
  p.B = a.batch;
  p.Lq = a.q_len;
  p.H = a.num_heads;
  p.Hkv = a.kv_heads;
  p.G = a.num_heads / a.kv_heads;
  p.Lkv = a.kv_len;
  p.Ls = a.shared_len;
  p.by_lq = fast_div(a.q_len);
  p.by_g = fast_div(p.G);
  p.by_h = fast_div(a.num_heads);
  p.by_hkv = fast_div(a.kv_heads);
  p.slots = plan.slots;
  p.prows = plan.prows;
  p.tail_rows = plan.tail_rows;
  p.o_part = static_cast<float*>(a.workspace);
  if (plan.bytes) p.ml_part = reinterpret_cast<float2*>(p.o_part + (size_t)plan.slots * plan.prows * a.head_dim);
  const bool fp16 = a.dtype == HB_FP16;
  bool launched = false;
  for (int kernel = 0; kernel < 2; ++kernel) {  // the parts of the few-rows kernel, then those of the tcgen05 one
    for (int i = 0; i < 2; ++i) {
      p.part[i] = plan.part[i];
      if (plan.tiles[i] != (kernel == 1)) p.part[i].count = 0;
    }
    if (p.part[0].count + p.part[1].count == 0) continue;
    const int rc = kernel ? launch_ctx_tiles(p, a.head_dim, fp16, plan.mask_tiles, launched, stream)
                          : launch_ctx_rows(p, a.head_dim, fp16, plan.rows_per_tile, stream);
    launched = true;
    if (rc != HB_OK) return rc;
  }
  p.part[1] = plan.part[1];
  return plan.slots > 1 ? launch_ctx_combine(p, a.head_dim, fp16, stream) : HB_OK;
}
