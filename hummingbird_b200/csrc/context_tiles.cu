// Context attention for many query rows: tcgen05 MMAs on tiles of 128 rows.
//
// One CTA takes 128 rows of one kv head (a row: a query token and one query head of the group) and walks its keys:
// S = Q K^T (fp32, TMEM), P = exp2(c S - m) (16-bit, over S in TMEM), O += P V (fp32, TMEM), with the running maximum
// m and sum of each row in the registers of one thread. The softmax's arithmetic bounds it: maxima, FMAs,
// exponentials and conversions of 128 scores a row take 980 cycles of an SM with four warps on each of its
// sub-partitions (1,170 a warp with two, 1,520 with one; measured without any memory or MMA), the MMAs of as many
// scores 660 to 800 at D 64; and within a tile S, softmax and P V wait for one another, about as long again. So at D 64
// four CTAs share an SM, as many as TMEM holds their S and O for (64 + 64 columns), and fill each other's waits. At
// D 128 there is room for two, each with two buffers of S (2 x 64 + 128 columns): the next tile's S runs while this
// one's softmax does. A lazy maximum (O is rescaled only when a row's maximum grows by more than 2^8, in fp16 2^4)
// keeps O in TMEM, and a share of the exponentials goes to the FMA pipe (exp2_poly2).
//
// The grid is one round of CTAs; each walks its share of the units (tiles of rows), so barriers, TMEM and tensor maps
// are set up once, K and V of the next unit are on their way early and its queries during the epilogue.
//
// Roles (8 warps): warps 0-3 load and norm the queries, then the softmax (one row per thread) and the epilogue;
// warp 4 TMA of K and V tiles (128-byte swizzle, rows past the end read as zero); warp 5 TMEM allocation and
// the MMAs; warp 6 reads the mask, one unit ahead. setmaxnreg moves registers from warps 4-7 to the softmax.
// Keys that are not valid: their scores are set to -inf, and in a tile that has some inside the tensor their V rows
// are zeroed in shared memory (0 * NaN would reach O); tiles without any valid key are skipped by every role.
//
// Batch 2, 2,648 queries, 16 heads, 8,184 keys, D 64: 235 us (754 TFLOP/s, 46 % of cuBLAS's bf16 burst) in runs of a
// few milliseconds, 262 us (677 TFLOP/s, 49 % of its sustained rate) in runs of a second, under the power cap. Issue
// slots 62 % used, MUFU 55 %, tensor pipe 37 %: no pipe is full. D 128: 320 to 338 us (1,109 to 1,050 TFLOP/s). The
// query norm stands before a unit's first S: 20.4 us with it, 17.8 without, at 2 x 2,648 queries over a padded 257.
//
// Compiled as whole-program device code, as setmaxnreg needs; its status word is read by hb_device_status.
#define HB_WHOLE_PROGRAM 1
#include <algorithm>
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include "context_attn.h"
#include "launch_after.h"
#include "hb_sm100.cuh"
#include "short_wait.cuh"

namespace hb {
namespace {

constexpr int kThreads = 256;
constexpr int kQAtom = 128 * 128;                // 128 rows of 128 bytes: 64 columns of a query tile
// By how much (log2 units) a row's maximum may grow before O is rescaled, and what all weights are multiplied by
// (2^kLift) so that small ones stay in P's normal range; P is at most 2^(kRescaleThreshold + kLift). bf16 has fp32's
// range. fp16's normal range ends at 2^-14, its subnormal at 2^-24: lifted, weights down to 2^-25 of the largest keep
// 11 bits and smaller ones are off by at most 2^-36 of it, 2^-11 in all over 2^25 keys (unlifted, 20,000 keys of weight
// 2^-25.2 beside one of 1 were lost whole).
template <bool kFp16>
constexpr float kRescaleThreshold = kFp16 ? 4.f : 8.f;
template <bool kFp16>
constexpr float kLift = kFp16 ? 11.f : 0.f;
constexpr int kCtxPolyMask = 3;                  // key pairs j with (j & 3) == 3 take exp2_poly2

template <int D>
struct Layout {
  static constexpr int kKeys = kCtxTileKeys;                // of a tile
  static constexpr int kWords = kKeys / 32;                 // of a tile's mask bits
  static constexpr int kCtasPerSm = ctx_tile_ctas(D) / kCtxSms;
  static constexpr int kLaunchRegs = 256 / kCtasPerSm;      // x 256 threads x kCtasPerSm = the SM's 65,536
  static constexpr int kSoftmaxRegs = D == 64 ? 88 : 184, kOtherRegs = 2 * kLaunchRegs - kSoftmaxRegs;
  static constexpr int kTmemCols = 512 / kCtasPerSm;
  static constexpr int kScores = D == 64 ? 1 : 2;           // buffers of S (and P) at 0, then O
  static constexpr int kTmemO = kScores * kKeys;
  static_assert(kTmemO + D <= kTmemCols, "TMEM columns");
  static constexpr int kHalves = D / 64;
  static constexpr int kAtom = kKeys * 128;                 // 64 columns of a K or V tile
  static constexpr int kTile = kHalves * kAtom;
  static constexpr int kStages = 2;
  static constexpr int kOffK = kHalves * kQAtom;            // queries at 0
  static constexpr int kOffV = kOffK + kStages * kTile;
  static constexpr int kOffBars = kOffV + kStages * kTile;
  static constexpr int kBars = 4 * kStages + 10;
  static constexpr int kOffMisc = kOffBars + kBars * 8;     // TMEM address, abort flag
  static constexpr int kOffBits = (kOffMisc + 8 + 15) & ~15;
  static constexpr int bytes(int mask_tiles) { return kOffBits + 2 * mask_tiles * kWords * 4 + 1024; }
  static_assert(kCtasPerSm * (bytes(kCtxMaskTiles) + 1024) <= 228 * 1024, "shared memory of an SM");
};

template <bool kFp16>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
  if constexpr (kFp16) {
    __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  } else {
    return pack_bf16x2(a, b);
  }
}
template <bool kFp16>
__device__ __forceinline__ float2 unpack16(uint32_t w) {
  if constexpr (kFp16) return __half22float2(*reinterpret_cast<__half2*>(&w));
  return make_float2(bf16_lo(w), bf16_hi(w));
}

// Instruction descriptor of kind::f16 with fp32 accumulators, N left out.
template <bool kFp16>
constexpr uint32_t idesc_base(bool b_mn_major) {
  const uint32_t fmt = kFp16 ? 0u : 1u;
  return (1u << 4) | (fmt << 7) | (fmt << 10) | ((b_mn_major ? 1u : 0u) << 16) | (static_cast<uint32_t>(128 >> 4) << 24);
}
// The MMA warp runs converged, so that descriptors stay in uniform registers (inside a one-lane branch each operand of
// each MMA is moved there one by one, which took longer than the MMAs); the elected lane's predicate picks the issuer.
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t e;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(e));
  return e;
}
__device__ __forceinline__ void mma_ss(uint32_t lead, uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %5, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(lead) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t lead, uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %5, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(lead) : "memory");
}
__device__ __forceinline__ void commit(uint32_t lead, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %1, 0;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
      ::"r"(smem_u32(bar)), "r"(lead) : "memory");
}

// The producer runs ahead: between tries it leaves the issue slots to the softmax.
__device__ __forceinline__ bool producer_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  return mbar_try_wait(bar, parity) || slow_wait<200>(bar, parity, abort_flag);
}
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, mbar_try_wait(bar, parity) || slow_wait<0>(bar, parity, abort_flag));
}

// A unit's key list: tiles [j0, j1) of the shared states' n0 tiles, then the batch element's own.
struct Keys {
  int n0, own_len, j0, j1;
};
template <int kKeys>
__device__ __forceinline__ Keys keys_of(const CtxParams& p, const CtxPart& part, const CtxUnit& u) {
  Keys k;
  k.own_len = part.use_own ? ctx_own_len(p, u.b) : 0;
  k.n0 = part.use_shared ? (p.Ls + kKeys - 1) / kKeys : 0;
  const int n = k.n0 + (k.own_len + kKeys - 1) / kKeys;
  k.j0 = part.by_splits.div(u.split * n);
  k.j1 = part.by_splits.div((u.split + 1) * n);
  return k;
}

// Keys [k0, k0 + kKeys) of either. `hi` counts them up to the last one that may be valid (0: skip the tile); with a
// mask, bits says which are.
template <int kKeys>
struct Tile {
  int k0, hi;
  bool shared, full, clean;  // full: all valid; clean: some of the tensor's rows in [0, hi) must not be read
  uint32_t bits[kKeys / 32];
};
template <int kKeys, bool kMask>
__device__ __forceinline__ Tile<kKeys> tile_of(const CtxParams& p, const Keys& ks, int j, const uint32_t* bits) {
  Tile<kKeys> t;
  t.shared = j < ks.n0;
  t.k0 = (t.shared ? j : j - ks.n0) * kKeys;
  if constexpr (kMask) {
    t.hi = 0;
    uint32_t all = 0xffffffffu;
#pragma unroll
    for (int i = 0; i < kKeys / 32; ++i) {
      const uint32_t b = t.bits[i] = bits[(j - ks.j0) * (kKeys / 32) + i];
      if (b) t.hi = 32 * i + 32 - __clz(b);
      all &= b;
    }
    t.full = all == 0xffffffffu;
    t.clean = !t.full;
  } else {
    t.hi = min(kKeys, (t.shared ? p.Ls : ks.own_len) - t.k0);
    t.full = t.hi == kKeys;
    // rows between hi and the next multiple of 16 enter P V: zeros past the tensor, anything before its end
    t.clean = !t.shared && (t.hi & 15) && ks.own_len < p.Lkv;
  }
  return t;
}

// Maximum of three, NaN where one is.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// One aligned 32-byte sector.
__device__ __forceinline__ void st_32b(void* dst, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
               ::"l"(dst), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

template <int D, bool kFp16, bool kMask>
__global__ void __launch_bounds__(kThreads, Layout<D>::kCtasPerSm)
    ctx_tiles_kernel(const __grid_constant__ CUtensorMap tm_own, const __grid_constant__ CUtensorMap tm_shared,
                     const __grid_constant__ CtxParams p, const int mask_tiles, const int beside) {
  using L = Layout<D>;
  constexpr int kStages = L::kStages, kKeys = L::kKeys, kWords = L::kWords;
  constexpr int PPR = D / 8;  // 16-byte pieces per row
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw + 1023u) & ~1023u) - raw);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kOffBars);
  uint64_t* k_full = bars;                  // [kStages] TMA bytes
  uint64_t* k_empty = k_full + kStages;     // [kStages] commit of the S MMAs
  uint64_t* v_full = k_empty + kStages;     // [kStages] TMA bytes
  uint64_t* v_empty = v_full + kStages;     // [kStages] commit of the P V MMAs
  uint64_t* q_full = v_empty + kStages;     // 4 softmax warps wrote the queries (units that have keys)
  uint64_t* s_full = q_full + 1;            // [kScores] commit: S written
  uint64_t* p_ready = s_full + 2;           // 4 softmax warps wrote P
  uint64_t* o_done = p_ready + 1;           // commit: P V added (one S buffer: the unit's last)
  uint64_t* drain = o_done + 1;
  uint64_t* m_full = drain + 1;             // [2] warp 6 wrote the unit's mask bits
  uint64_t* m_free = m_full + 2;            // [2] producer, MMA warp and softmax warps are through
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kOffMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kOffMisc + 4);
  uint32_t* bits0 = reinterpret_cast<uint32_t*>(smem + L::kOffBits);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int count0 = p.part[0].count, total = count0 + p.part[1].count;

  if (warp == 4 && lane == 0) {
    prefetch_tmap(&tm_own);
    prefetch_tmap(&tm_shared);
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    mbar_init(q_full, 4);
    mbar_init(&s_full[0], 1);
    mbar_init(&s_full[1], 1);
    mbar_init(p_ready, 4);
    mbar_init(o_done, 1);
    mbar_init(drain, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&m_full[i], 1);
      mbar_init(&m_free[i], 6);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  // Work unit w's queries, asynchronously into the shared-memory image (rows past the end as zeros): warp i its 32
  // rows, a row's PPR pieces by PPR consecutive lanes.
  constexpr int kRowsPerStep = 32 / PPR, kSteps = 32 / kRowsPerStep;
  const int qch = lane % PPR, qrow = warp * 32 + lane / PPR;
  auto load_q = [&](int w) {
    const CtxPart& part = p.part[w >= count0 ? 1 : 0];
    const CtxUnit u = ctx_unit(p, part, w - (w >= count0 ? count0 : 0));
    const bool plain = p.G == 1 && !part.pooled;  // rows one stride apart
    const uint16_t* src = p.q + (plain ? u.b * p.q_bs + (int64_t)(u.rt * 128 + qrow) * p.q_rs + u.g * D : 0) + qch * 8;
    const uint32_t dst = smem_u32(smem) + (qch >> 3) * kQAtom;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const int lr = qrow + i * kRowsPerStep, r = u.rt * 128 + lr;
      const bool live = r < u.rows;
      const uint16_t* from = src + i * kRowsPerStep * p.q_rs;
      if (!plain) {
        const CtxRow x = ctx_row(p, live ? r : 0, u.g, u.b, part.pooled);
        from = src + x.bq * p.q_bs + x.i * p.q_rs + x.hq * D;
      }
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + sw128_offset(lr, qch & 7)),
                   "l"(live ? from : p.q), "r"(live ? 16u : 0u) : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // Up to here nothing but parameters was read, so this may run while the kernel before still does (a call among others
  // 20.5 -> 19.1 us at the 120 s clip's cross-attention). The launch beside the few-rows kernel does not wait for that
  // one here: it was let in by a kernel that had waited itself, so all that it reads is in memory, and the fence keeps
  // ordinary loads (lengths, masks, the norm's weights) from older lines of this SM's L1.
  if (beside) __threadfence();
  else asm volatile("griddepcontrol.wait;" ::: "memory");
  // TMEM is asked for only now: the kernel before may be anyone's (a library's product) and may let this one in before
  // its own CTAs have theirs, so nothing is held while this one waits for it (that call takes 18.1 us instead of 19.0).
  if (warp == 5) {
    tmem_alloc(tmem_slot, L::kTmemCols);
    tmem_relinquish();
  }
  if (warp < 4) load_q(blockIdx.x);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // The merge, or the next early launch: they wait. Not before every CTA of this launch has its TMEM, whatever the next
  // one does with its own.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  if (warp >= 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::kOtherRegs));
    if (warp == 4 && lane == 0) {
      // -------------------------------------------------------------- TMA producer
      int it = 0;
      bool ok = true;
      for (int n = 0, w = blockIdx.x; ok && w < total; ++n, w += gridDim.x) {
        const CtxPart& part = p.part[w >= count0 ? 1 : 0];
        const CtxUnit u = ctx_unit(p, part, w - (w >= count0 ? count0 : 0));
        const Keys ks = keys_of<kKeys>(p, part, u);
        const uint32_t* bits = bits0 + (n & 1) * mask_tiles * kWords;
        const int kcol = u.g * D, vcol = p.Hkv * D + u.g * D;
        if (kMask && !(ok = producer_wait(&m_full[n & 1], (n >> 1) & 1, abort_flag))) break;
        for (int j = ks.j0; j < ks.j1; ++j) {
          const Tile<kKeys> t = tile_of<kKeys, kMask>(p, ks, j, bits);
          if (t.hi <= 0) continue;
          const int st = it % kStages;
          const uint32_t ph = ((it / kStages) & 1) ^ 1;
          const CUtensorMap* tm = t.shared ? &tm_shared : &tm_own;
          const bool inter = !t.shared && p.kv_inter;  // the map's second dimension is the batch
          const int bc = t.shared || p.kv_bs == 0 ? 0 : u.b;
          const int c1 = inter ? bc : t.k0, c2 = inter ? t.k0 : bc;
          if (it >= kStages && !(ok = producer_wait(&k_empty[st], ph, abort_flag))) break;
          mbar_arrive_expect_tx(&k_full[st], L::kTile);
#pragma unroll
          for (int h = 0; h < L::kHalves; ++h)
            tma_load_3d(smem + L::kOffK + st * L::kTile + h * L::kAtom, tm, kcol + 64 * h, c1, c2, &k_full[st]);
          if (it >= kStages && !(ok = producer_wait(&v_empty[st], ph, abort_flag))) {
            mbar_wait(&k_full[st], (it / kStages) & 1);  // K was issued already
            break;
          }
          mbar_arrive_expect_tx(&v_full[st], L::kTile);
#pragma unroll
          for (int h = 0; h < L::kHalves; ++h)
            tma_load_3d(smem + L::kOffV + st * L::kTile + h * L::kAtom, tm, vcol + 64 * h, c1, c2, &v_full[st]);
          ++it;
        }
        if (kMask) mbar_arrive(&m_free[n & 1]);
      }
      // every copy issued into this CTA's shared memory lands before it exits
      for (int i = max(0, it - kStages); i < it; ++i) {
        mbar_wait(&k_full[i % kStages], (i / kStages) & 1);
        mbar_wait(&v_full[i % kStages], (i / kStages) & 1);
      }
    } else if (warp == 5) {
      const uint32_t lead = elect_one();
      // -------------------------------------------------------------- MMA issuer
      constexpr uint32_t idS = idesc_base<kFp16>(false), idO = idesc_base<kFp16>(true) | ((D >> 3) << 17);
      const uint64_t dq = smem_desc_sw128(smem_u32(smem));
      const uint64_t dk = smem_desc_sw128(smem_u32(smem + L::kOffK));
      // V tiles are MN-major: 16 keys are 2,048 bytes on, the second 64 columns one atom on
      const uint64_t dv = smem_desc_sw128(smem_u32(smem + L::kOffV), D == 64 ? 16 : L::kAtom);
      const uint32_t tO = tmem + L::kTmemO;
      int it = 0, units = 0;
      auto issue_s = [&](int i, int n16) {
        const int st = i % kStages;
        if (!warp_wait(&k_full[st], (i / kStages) & 1, abort_flag)) return false;
        tc_fence_after();
        const uint32_t id = idS | (static_cast<uint32_t>(n16 >> 3) << 17);
        const uint64_t kd = dk + st * (L::kTile >> 4);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const int half = k / 4, at = (k % 4) * 32;
          mma_ss(lead, tmem + i % L::kScores * kKeys, dq + ((half * kQAtom + at) >> 4), kd + ((half * L::kAtom + at) >> 4), id, k > 0);
        }
        commit(lead, &s_full[i % L::kScores]);
        commit(lead, &k_empty[st]);
        return true;
      };
      bool ok = true;
      for (int n = 0, w = blockIdx.x; ok && w < total; ++n, w += gridDim.x) {
        const CtxPart& part = p.part[w >= count0 ? 1 : 0];
        const Keys ks = keys_of<kKeys>(p, part, ctx_unit(p, part, w - (w >= count0 ? count0 : 0)));
        const uint32_t* bits = bits0 + (n & 1) * mask_tiles * kWords;
        if (kMask && !(ok = warp_wait(&m_full[n & 1], (n >> 1) & 1, abort_flag))) break;
        auto next_tile = [&](int j, int& n16) {  // the first tile at or after j that has valid keys
          for (; j < ks.j1; ++j) {
            const Tile<kKeys> t = tile_of<kKeys, kMask>(p, ks, j, bits);
            n16 = (t.hi + 15) & ~15;
            if (t.hi > 0) break;
          }
          return j;
        };
        int n16 = 0, n16_next = 0;
        int j = next_tile(ks.j0, n16);
        if (j < ks.j1) ok = warp_wait(q_full, units++ & 1, abort_flag) && issue_s(it, n16);
        for (bool first = true; ok && j < ks.j1; first = false) {
          const int jn = next_tile(j + 1, n16_next), st = it % kStages;
          // two buffers: the next S while the softmax computes this tile's P
          if (L::kScores == 2 && jn < ks.j1 && !(ok = issue_s(it + 1, n16_next))) break;
          if (!(ok = warp_wait(&v_full[st], (it / kStages) & 1, abort_flag) && warp_wait(p_ready, it & 1, abort_flag)))
            break;
          tc_fence_after();
          const uint64_t vd = dv + st * (L::kTile >> 4);
#pragma unroll
          for (int k = 0; k < kKeys / 16; ++k)
            if (16 * k < n16) mma_ts(lead, tO, tmem + it % L::kScores * kKeys + 8 * k, vd + k * (2048 >> 4), idO, !first || k > 0);
          if (L::kScores == 2 || jn >= ks.j1) commit(lead, o_done);
          commit(lead, &v_empty[st]);
          // one: in the tensor pipe's order, P V reads P before the next S overwrites it
          if (L::kScores == 1 && jn < ks.j1 && !(ok = issue_s(it + 1, n16_next))) break;
          ++it;
          j = jn;
          n16 = n16_next;
        }
        if constexpr (kMask) {
          __syncwarp();  // every lane has read the unit's mask bits
          if (lead) mbar_arrive(&m_free[n & 1]);
        }
      }
      commit(lead, drain);  // every MMA this thread issued has finished before TMEM is freed
      mbar_wait(drain, 0);
    } else if (kMask && warp == 6) {
      // -------------------------------------------------------------- mask bits, one unit ahead of their readers
      for (int n = 0, w = blockIdx.x; w < total; ++n, w += gridDim.x) {
        const CtxPart& part = p.part[w >= count0 ? 1 : 0];
        const CtxUnit u = ctx_unit(p, part, w - (w >= count0 ? count0 : 0));
        const Keys ks = keys_of<kKeys>(p, part, u);
        uint32_t* bits = bits0 + (n & 1) * mask_tiles * kWords;
        if (n >= 2 && !warp_wait(&m_free[n & 1], ((n >> 1) & 1) ^ 1, abort_flag)) break;
        for (int j = ks.j0; j < ks.j1; ++j) {
          const bool sh = j < ks.n0;
          const int k0 = (sh ? j : j - ks.n0) * kKeys, len = sh ? p.Ls : ks.own_len;
          const uint8_t* mk = sh ? p.smask : (p.mask ? p.mask + u.b * p.mask_bs : nullptr);
          uint32_t v[kWords];
#pragma unroll
          for (int i = 0; i < kWords; ++i) {
            const int k = k0 + 32 * i + lane;
            v[i] = k < len ? (mk ? mk[k] : 1u) : 0u;
          }
#pragma unroll
          for (int i = 0; i < kWords; ++i) {
            v[i] = __ballot_sync(0xffffffffu, v[i] != 0u);
            if (lane == 0) bits[(j - ks.j0) * kWords + i] = v[i];
          }
        }
        if (lane == 0) mbar_arrive(&m_full[n & 1]);  // lane 0 wrote them all
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(L::kSoftmaxRegs));
    const uint32_t lane_base = static_cast<uint32_t>(warp * 32) << 16;
    const uint32_t tO = tmem + lane_base + L::kTmemO;
    const int row = warp * 32 + lane;
    int it = 0, done = 0;
    bool ok = true;
    for (int n = 0, w = blockIdx.x; ok && w < total; ++n, w += gridDim.x) {
      const CtxPart& part = p.part[w >= count0 ? 1 : 0];
      const CtxUnit u = ctx_unit(p, part, w - (w >= count0 ? count0 : 0));
      const Keys ks = keys_of<kKeys>(p, part, u);
      const uint32_t* bits = bits0 + (n & 1) * mask_tiles * kWords;
      if (kMask && !(ok = warp_wait(&m_full[n & 1], (n >> 1) & 1, abort_flag))) break;
      // -------------------------------------------------------------- queries: each lane's own pieces have landed
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      if (p.q_w) {  // rounded to the input's type, as the norm pass that this replaces stores it
        float wv[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) wv[e] = p.q_w[qch * 8 + e];
#pragma unroll 2
        for (int i = 0; i < kSteps; ++i) {
          uint4* at = reinterpret_cast<uint4*>(smem + (qch >> 3) * kQAtom + sw128_offset(qrow + i * kRowsPerStep, qch & 7));
          const uint4 v = *at;
          uint32_t x[4] = {v.x, v.y, v.z, v.w};
          float2 f[4];
          float ss = 0.f;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            f[e] = unpack16<kFp16>(x[e]);
            ss = fmaf(f[e].x, f[e].x, fmaf(f[e].y, f[e].y, ss));
          }
#pragma unroll
          for (int o = 1; o < PPR; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
          const float inv = rsqrtf(ss * (1.f / D) + p.eps);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = pack16<kFp16>(f[e].x * inv * wv[2 * e], f[e].y * inv * wv[2 * e + 1]);
          *at = make_uint4(x[0], x[1], x[2], x[3]);
        }
      }
      fence_proxy_async_smem();
      __syncwarp();

      // -------------------------------------------------------------- softmax
      float m = -INFINITY, l = 0.f;
      bool first = true;
      for (int j = ks.j0; j < ks.j1; ++j) {
        const Tile<kKeys> t = tile_of<kKeys, kMask>(p, ks, j, bits);
        if (t.hi <= 0) continue;
        if (first && lane == 0) mbar_arrive(q_full);
        if (!(ok = warp_wait(&s_full[it % L::kScores], (it / L::kScores) & 1, abort_flag))) break;
        tc_fence_after();
        const uint32_t tS = tmem + lane_base + it % L::kScores * kKeys;
        uint32_t r[kWords][32];
#pragma unroll
        for (int c = 0; c < kWords; ++c) tmem_ld32(tS + 32 * c, r[c]);
        tmem_wait_ld();
        if (!t.full) {  // columns past hi hold an earlier tile's bits
#pragma unroll
          for (int c = 0; c < kWords; ++c) {
            uint32_t word;
            if constexpr (kMask) {
              word = t.bits[c];
            } else {
              const int left = t.hi - 32 * c;
              word = left >= 32 ? 0xffffffffu : left <= 0 ? 0u : (1u << left) - 1u;
            }
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!((word >> e) & 1u)) r[c][e] = 0xff800000u;  // -inf
          }
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < kWords; ++c)
#pragma unroll
          for (int e = 0; e < 32; e += 2)
            mx[e / 2 & 3] = max3_nan(mx[e / 2 & 3], __uint_as_float(r[c][e]), __uint_as_float(r[c][e + 1]));
        const float rmax = max3_nan(max3_nan(mx[0], mx[1], mx[2]), mx[3], mx[3]) * p.scale_log2;
        const float m_new = fmaxf(m, rmax);
        const bool upd = m_new > m + kRescaleThreshold<kFp16>;
        float alpha = 1.f;
        if (upd) {
          alpha = m == -INFINITY ? 0.f : ex2_approx(m - m_new);
          m = m_new;
        }
        // A score of NaN or +inf makes the whole row NaN, l with it. (exp2_poly2 does not pass NaN on: its clamp drops
        // it.)
        const float nm = !(rmax < INFINITY) ? NAN : m == -INFINITY ? 0.f : kLift<kFp16> - m;
        float rs[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < kWords; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float x0, x1, p0, p1;
            ffma2(x0, x1, __uint_as_float(r[c][2 * e]), __uint_as_float(r[c][2 * e + 1]), p.scale_log2, p.scale_log2,
                  nm, nm);
            if ((e & kCtxPolyMask) == kCtxPolyMask) {  // a share of the exponentials on the FMA pipe
              exp2_poly2(x0, x1, p0, p1);
            } else {
              p0 = ex2_approx(x0);
              p1 = ex2_approx(x1);
            }
            const int a2 = (e & 1) * 2;
            fadd2(rs[a2], rs[a2 + 1], rs[a2], rs[a2 + 1], p0, p1);
            // P in the input's type for the MMA (relative error up to 2^-8 or 2^-11); l keeps fp32
            pk[e] = pack16<kFp16>(p0, p1);
          }
          tmem_st16(tS + 16 * c, pk);
        }
        l = l * alpha + ((rs[0] + rs[1]) + (rs[2] + rs[3]));
        // O has the tile before: with one buffer this tile's S came after it
        if (L::kScores == 2 && !first) {
          if (!(ok = warp_wait(o_done, done++ & 1, abort_flag))) break;
          tc_fence_after();
        }
        if (!first && __any_sync(0xffffffffu, upd)) {
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            tmem_ld32(tO + 32 * c, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tmem_st32(tO + 32 * c, o);
          }
        }
        if (t.clean) {  // V rows of keys that are not valid: 128 / kKeys threads to a row
          const int st = it % kStages;
          if (!(ok = warp_wait(&v_full[st], (it / kStages) & 1, abort_flag))) break;
          const int key = row % kKeys;
          bool valid = key < t.hi;
          if constexpr (kMask) {
            valid = false;
#pragma unroll
            for (int i = 0; i < kWords; ++i)
              if (key / 32 == i) valid = (t.bits[i] >> lane) & 1u;
          }
          if (!valid) {
            constexpr int kPieces = PPR * kKeys / 128;
            uint8_t* v = smem + L::kOffV + st * L::kTile;
#pragma unroll
            for (int c = 0; c < kPieces; ++c) {
              const int ch = row / kKeys * kPieces + c;
              *reinterpret_cast<uint4*>(v + (ch >> 3) * L::kAtom + sw128_offset(key, ch & 7)) = make_uint4(0u, 0u, 0u, 0u);
            }
          }
          fence_proxy_async_smem();
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_ready);
        ++it;
        first = false;
      }
      if constexpr (kMask) {
        __syncwarp();  // every lane has read the unit's mask bits
        if (lane == 0) mbar_arrive(&m_free[n & 1]);
      }
      // -------------------------------------------------------------- epilogue: one row per thread
      if (!ok) break;
      if (w + gridDim.x < total) load_q(w + gridDim.x);  // (the S MMAs of this unit are done)
      if (!first && !(ok = warp_wait(o_done, done++ & 1, abort_flag))) break;
      tc_fence_after();
      // Nothing but scores of -inf: no weight. (exp2_poly2 gives them 2^-125 instead of 0, which shows only here.)
      if (m == -INFINITY && l > 0.f) l = 0.f;
      const int gr = u.rt * 128 + row;
      const bool live = gr < u.rows;
      const CtxRow x = ctx_row(p, live ? gr : 0, u.g, u.b, part.pooled);
      if (part.direct) {
        const float inv = l > 0.f ? 1.f / l : l;  // l 0: no key; NaN stays
        uint16_t* dst = p.out + x.bq * p.o_bs + x.i * p.o_rs + x.hq * D;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32], v[16];
          tmem_ld32(tO + 32 * c, o);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 16; ++e)
            v[e] = l == 0.f ? 0u
                            : pack16<kFp16>(__uint_as_float(o[2 * e]) * inv, __uint_as_float(o[2 * e + 1]) * inv);
          if (live) {
            if (p.out_wide) {  // whole 32-byte sectors
              st_32b(dst + c * 32, v);
              st_32b(dst + c * 32 + 16, v + 8);
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                *reinterpret_cast<uint4*>(dst + c * 32 + e * 8) =
                    make_uint4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
            }
          }
        }
      } else {
        const int64_t pr = ctx_prow(p, part, u, x, row);
        if (live) p.ml_part[pr] = make_float2(l == 0.f ? -INFINITY : m - kLift<kFp16>, l);
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(tO + 32 * c, o);
          tmem_wait_ld();
          if (live) {
#pragma unroll
            for (int e = 0; e < 4; ++e) st_32b(p.o_part + pr * D + c * 32 + e * 8, o + 8 * e);
          }
        }
      }
      tc_fence_before();  // O has been read; the next unit's first P V follows this warp's p_ready
    }
    if (!ok) *abort_flag = 1;
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem, L::kTmemCols);
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the few-rows kernel, where this one runs beside it
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
                   q == cudaDriverEntryPointSuccess
               ? reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr)
               : nullptr;
  }();
  return fn;
}

// `outer` x `mid` rows of `width` states; box 64 columns x `keys` keys (the middle dimension, or the outer one where
// `keys_outer`), 128-byte swizzle; keys past the end read as zero.
bool encode_states(CUtensorMap* map, const void* base, bool fp16, unsigned keys, int64_t width, int64_t mid,
                   int64_t outer, int64_t mid_stride, int64_t outer_stride, bool keys_outer) {
  auto encode = encode_fn();
  if (!encode) return false;
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(width), static_cast<cuuint64_t>(mid), static_cast<cuuint64_t>(outer)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(mid_stride) * 2, static_cast<cuuint64_t>(outer_stride) * 2};
  cuuint32_t box[3] = {64, keys_outer ? 1u : keys, keys_outer ? keys : 1u};
  cuuint32_t estr[3] = {1, 1, 1};
  return encode(map, fp16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, bool kFp16, bool kMask>
int launch_tiles(const CUtensorMap& own, const CUtensorMap& shared, const CtxParams& p, int mask_tiles,
                 bool beside, cudaStream_t s) {
  auto kernel = ctx_tiles_kernel<D, kFp16, kMask>;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return HB_ERR_LAUNCH;
  static bool configured[64] = {};
  if (dev >= 64 || !configured[dev]) {
    // setmaxnreg's split counts on exactly kLaunchRegs registers per thread at launch: an increase that the CTA's
    // registers do not cover would never be granted
    cudaFuncAttributes attr{};
    if (cudaFuncGetAttributes(&attr, kernel) != cudaSuccess || attr.numRegs != Layout<D>::kLaunchRegs ||
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<D>::bytes(kCtxMaskTiles)) !=
            cudaSuccess)
      return HB_ERR_LAUNCH;
    if (dev < 64) configured[dev] = true;
  }
  const int grid = std::min(p.part[0].count + p.part[1].count, ctx_tile_ctas(D));
  return launch_after(kernel, grid, kThreads, Layout<D>::bytes(mask_tiles), s, own, shared, p, mask_tiles,
                      static_cast<int>(beside));
}

template <int D, bool kFp16>
int launch_tiles(const CUtensorMap& own, const CUtensorMap& shared, const CtxParams& p, bool mask, int mask_tiles,
                 bool beside, cudaStream_t s) {
  return mask ? launch_tiles<D, kFp16, true>(own, shared, p, mask_tiles, beside, s)
              : launch_tiles<D, kFp16, false>(own, shared, p, 0, beside, s);
}

}  // namespace

int ctx_tiles_take_status(unsigned int* status) {
  unsigned int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_device_status_local, sizeof(v)) != cudaSuccess) return HB_ERR_LAUNCH;
  if (v && cudaMemcpyToSymbol(g_device_status_local, &zero, sizeof(zero)) != cudaSuccess) return HB_ERR_LAUNCH;
  *status = v;
  return HB_OK;
}

int launch_ctx_tiles(const CtxParams& p, int D, bool fp16, int mask_tiles, bool beside, cudaStream_t s) {
  const int64_t width = 2ll * p.Hkv * D;
  const unsigned keys = kCtxTileKeys;
  CUtensorMap own{}, shared{};
  const bool use_own = p.Lkv > 0 && (p.part[0].use_own || p.part[1].use_own);
  const bool use_shared = p.part[0].use_shared != 0;
  const int64_t batch = p.kv_bs == 0 ? 1 : p.B;  // one copy of the states is a batch of one to the map
  if (use_own &&
      !(p.kv_inter ? encode_states(&own, p.kv, fp16, keys, width, batch, p.Lkv, p.kv_bs, p.kv_rs, true)
                   : encode_states(&own, p.kv, fp16, keys, width, p.Lkv, batch, p.kv_rs,
                                   batch > 1 ? p.kv_bs : p.kv_rs, false)))
    return HB_ERR_LAUNCH;
  if (use_shared && !encode_states(&shared, p.skv, fp16, keys, width, p.Ls, 1, p.skv_rs, p.skv_rs, false))
    return HB_ERR_LAUNCH;
  if (!use_own) own = shared;
  if (!use_shared) shared = own;
  const bool mask = p.mask || p.smask;
  if (D == 128)
    return fp16 ? launch_tiles<128, true>(own, shared, p, mask, mask_tiles, beside, s)
                : launch_tiles<128, false>(own, shared, p, mask, mask_tiles, beside, s);
  return fp16 ? launch_tiles<64, true>(own, shared, p, mask, mask_tiles, beside, s)
              : launch_tiles<64, false>(own, shared, p, mask, mask_tiles, beside, s);
}

}  // namespace hb
