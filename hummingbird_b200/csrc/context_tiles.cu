// Context attention for many query rows: tcgen05 MMAs on 128-row x 128-key tiles.
//
// One CTA takes 128 rows of one kv head (a row: a query token and one query head of the group) and walks its keys:
// S = Q K^T (fp32, TMEM), P = exp2(c S - m) (16-bit, back into TMEM over S), O += P V (fp32, TMEM), with the running
// maximum m and sum of each row in the registers of one thread. The exponentials bound it (one per score against
// 4 D flops: at D 64 the MUFU unit needs 1,024 cycles per tile and SM, the tensor pipe about 660), and within a
// tile the three steps wait for one another. So two CTAs share an SM, each with 256 TMEM columns: one's softmax runs
// while the other's MMAs do. A lazy maximum (O is rescaled only when a row's maximum grows by more than 2^8) keeps
// O in TMEM, and a quarter of the exponentials goes to the FMA pipe (exp2_poly2).
//
// Roles (8 warps): warps 0-3 load and norm the queries, then the softmax (one row per thread) and the epilogue;
// warp 4 TMA of K and V tiles (128-byte swizzle, rows past the end read as zero); warp 5 TMEM allocation and the one
// MMA-issuing thread; warps 4-7 read the mask first. setmaxnreg moves registers from warps 4-7 to the softmax.
// Keys that are not valid: their scores are set to -inf, and in a tile that has some inside the tensor their V rows
// are zeroed in shared memory (0 * NaN would reach O); tiles without any valid key are skipped by every role.
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
#include "hb_sm100.cuh"

namespace hb {
namespace {

constexpr int kThreads = 256;
constexpr int kLaunchRegs = 128;                 // 2 CTAs x 256 threads x 128 = the SM's 65,536
constexpr int kSoftmaxRegs = 200, kOtherRegs = 56;
static_assert(kSoftmaxRegs + kOtherRegs == 2 * kLaunchRegs, "the warpgroups share what the CTA was launched with");
constexpr int kAtom = 128 * 128;                 // 128 rows of 128 bytes: 64 columns of a tile
constexpr float kRescaleThreshold = 8.0f;        // log2 units
constexpr int kTmemCols = 256;                   // S (P over it) at 0, O at 128

template <int D>
struct Layout {
  static constexpr int kHalves = D / 64;
  static constexpr int kTile = kHalves * kAtom;
  static constexpr int kStages = D == 64 ? 2 : 1;
  static constexpr int kOffK = kTile;                       // queries (the output is staged there too) at 0
  static constexpr int kOffV = kOffK + kStages * kTile;
  static constexpr int kOffBars = kOffV + kStages * kTile;
  static constexpr int kBars = 4 * kStages + 4;
  static constexpr int kOffMisc = kOffBars + kBars * 8;     // TMEM address, abort flag
  static constexpr int kOffBits = (kOffMisc + 8 + 15) & ~15;
  static constexpr int bytes(int mask_tiles) { return kOffBits + mask_tiles * 16 + 1024; }
};
static_assert(Layout<64>::bytes(kCtxMaskTiles) <= 113 * 1024 && Layout<128>::bytes(kCtxMaskTiles) <= 113 * 1024,
              "two CTAs per SM");

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
__device__ __forceinline__ uint32_t idesc_n(uint32_t base, int n) { return base | (static_cast<uint32_t>(n >> 3) << 17); }

__device__ __forceinline__ bool role_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  if (mbar_wait(bar, parity) && !*abort_flag) return true;
  *abort_flag = 1;
  return false;
}
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity) && !*abort_flag);
}

// A tile of the key list: keys [k0, k0 + 128) of the shared states or of the batch element's own. `hi` counts the
// keys up to the last one that may be valid (0: skip the tile); with a mask, bits says which are.
struct Tile {
  int k0, hi;
  bool shared, full, clean;  // full: all 128 valid; clean: some of the tensor's rows in [0, hi) must not be read
  uint4 bits;
};

template <bool kMask>
__device__ __forceinline__ Tile tile_of(const CtxParams& p, int j, int n0, int own_len, const uint4* bits, int j0) {
  Tile t;
  t.shared = j < n0;
  t.k0 = (t.shared ? j : j - n0) * 128;
  t.hi = min(128, (t.shared ? p.Ls : own_len) - t.k0);
  t.full = t.hi == 128;
  // rows between hi and the next multiple of 16 enter P V: zeros past the tensor, anything before its end
  t.clean = !t.shared && (t.hi & 15) && own_len < p.Lkv;
  if constexpr (kMask) {
    t.bits = bits[j - j0];
    const uint32_t b[4] = {t.bits.x, t.bits.y, t.bits.z, t.bits.w};
    int hi = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (b[i]) hi = 32 * i + 32 - __clz(b[i]);
    t.hi = hi;
    t.full = (b[0] & b[1] & b[2] & b[3]) == 0xffffffffu;
    t.clean = !t.full;
  }
  return t;
}

__device__ __forceinline__ uint32_t word_of(const uint4& b, int i) {
  return i == 0 ? b.x : i == 1 ? b.y : i == 2 ? b.z : b.w;
}

template <int D, bool kFp16, bool kMask>
__global__ void __launch_bounds__(kThreads, 2)
    ctx_tiles_kernel(const __grid_constant__ CUtensorMap tm_own, const __grid_constant__ CUtensorMap tm_shared,
                     const CtxParams p) {
  using L = Layout<D>;
  constexpr int kStages = L::kStages;
  constexpr int PPR = D / 8;  // 16-byte pieces per row
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw + 1023u) & ~1023u) - raw);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kOffBars);
  uint64_t* k_full = bars;                  // [kStages] TMA bytes
  uint64_t* k_empty = k_full + kStages;     // [kStages] commit of the S MMAs
  uint64_t* v_full = k_empty + kStages;     // [kStages] TMA bytes
  uint64_t* v_empty = v_full + kStages;     // [kStages] commit of the P V MMAs
  uint64_t* q_full = v_empty + kStages;     // 4 softmax warps wrote the queries
  uint64_t* s_full = q_full + 1;            // commit: S written (and the tile before's P V done)
  uint64_t* p_ready = s_full + 1;           // 4 softmax warps wrote P
  uint64_t* o_full = p_ready + 1;           // commit: everything done
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kOffMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kOffMisc + 4);
  uint4* bits = reinterpret_cast<uint4*>(smem + L::kOffBits);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // ---- which item
  int idx = blockIdx.x;
  const bool second = idx >= p.part[0].ctas;
  const CtxPart& part = second ? p.part[1] : p.part[0];
  if (second) idx -= p.part[0].ctas;
  const int split = idx % part.splits;
  idx /= part.splits;
  const int rt = idx % part.row_tiles;
  idx /= part.row_tiles;
  const int g = idx % p.Hkv;
  const int b = idx / p.Hkv;  // 0 for pooled items
  const int rows = (part.pooled ? p.B : 1) * p.Lq * p.G;
  const int tok0 = part.pooled ? 0 : b * p.Lq;
  const int own_len = part.use_own ? ctx_own_len(p, b) : 0;
  const int n0 = part.use_shared ? (p.Ls + 127) / 128 : 0;
  const int n = n0 + (own_len + 127) / 128;
  const int j0 = static_cast<int>((int64_t)split * n / part.splits);
  const int j1 = static_cast<int>((int64_t)(split + 1) * n / part.splits);

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    mbar_init(q_full, 4);
    mbar_init(s_full, 1);
    mbar_init(p_ready, 4);
    mbar_init(o_full, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 5) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  if (kMask && warp >= 4) {
    for (int j = j0 + warp - 4; j < j1; j += 4) {
      const bool sh = j < n0;
      const int k0 = (sh ? j : j - n0) * 128, len = sh ? p.Ls : own_len;
      const uint8_t* mk = sh ? p.smask : (p.mask ? p.mask + b * p.mask_bs : nullptr);
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k = k0 + 32 * i + lane;
        bool v = k < len;
        if (v && mk) v = mk[k] != 0;
        w[i] = __ballot_sync(0xffffffffu, v);
      }
      if (lane == 0) bits[j - j0] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  // The queries are on their way while the CTA sets up: a row's PPR pieces in PPR consecutive lanes.
  constexpr int kRowsPerStep = 32 / PPR, kSteps = 32 / kRowsPerStep;
  uint4 qv[kSteps];
  const int qch = lane % PPR;
  if (warp < 4) {
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const int r = rt * 128 + warp * 32 + i * kRowsPerStep + lane / PPR;
      qv[i] = make_uint4(0u, 0u, 0u, 0u);
      if (r < rows) {
        const int tk = r / p.G, hq = g * p.G + (r - tk * p.G), t = tok0 + tk, bq = t / p.Lq;
        qv[i] = __ldg(reinterpret_cast<const uint4*>(p.q + bq * p.q_bs + (t - bq * p.Lq) * p.q_rs + (int64_t)hq * D +
                                                     qch * 8));
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp >= 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == 4 && lane == 0) {
      // -------------------------------------------------------------- TMA producer
      int it = 0;
      const int kcol = g * D, vcol = p.Hkv * D + g * D;
      for (int j = j0; j < j1; ++j) {
        const Tile t = tile_of<kMask>(p, j, n0, own_len, bits, j0);
        if (t.hi <= 0) continue;
        const int st = it % kStages;
        const uint32_t ph = ((it / kStages) & 1) ^ 1;
        const CUtensorMap* tm = t.shared ? &tm_shared : &tm_own;
        const bool inter = !t.shared && p.kv_inter;  // the map's second dimension is the batch
        const int bc = t.shared || p.kv_bs == 0 ? 0 : b;
        const int c1 = inter ? bc : t.k0, c2 = inter ? t.k0 : bc;
        if (it >= kStages && !role_wait(&k_empty[st], ph, abort_flag)) break;
        mbar_arrive_expect_tx(&k_full[st], L::kTile);
#pragma unroll
        for (int h = 0; h < L::kHalves; ++h)
          tma_load_3d(smem + L::kOffK + st * L::kTile + h * kAtom, tm, kcol + 64 * h, c1, c2, &k_full[st]);
        if (it >= kStages && !role_wait(&v_empty[st], ph, abort_flag)) {
          mbar_wait(&k_full[st], (it / kStages) & 1);
          break;
        }
        mbar_arrive_expect_tx(&v_full[st], L::kTile);
#pragma unroll
        for (int h = 0; h < L::kHalves; ++h)
          tma_load_3d(smem + L::kOffV + st * L::kTile + h * kAtom, tm, vcol + 64 * h, c1, c2, &v_full[st]);
        ++it;
      }
      // every copy issued into this CTA's shared memory lands before it exits
      for (int i = max(0, it - kStages); i < it; ++i) {
        mbar_wait(&k_full[i % kStages], (i / kStages) & 1);
        mbar_wait(&v_full[i % kStages], (i / kStages) & 1);
      }
    } else if (warp == 5 && lane == 0) {
      // -------------------------------------------------------------- MMA issuer
      constexpr uint32_t idS = idesc_base<kFp16>(false), idO = idesc_base<kFp16>(true);
      const uint32_t qa = smem_u32(smem), kb0 = smem_u32(smem + L::kOffK), vb0 = smem_u32(smem + L::kOffV);
      const uint32_t tS = tmem, tO = tmem + 128;
      int it = 0;
      for (int j = j0; j < j1; ++j) {
        const Tile t = tile_of<kMask>(p, j, n0, own_len, bits, j0);
        if (t.hi <= 0) continue;
        const int st = it % kStages, n16 = (t.hi + 15) & ~15;
        if (it == 0 && !role_wait(q_full, 0, abort_flag)) break;
        if (!role_wait(&k_full[st], (it / kStages) & 1, abort_flag)) break;
        tc_fence_after();
        const uint32_t kb = kb0 + st * L::kTile, vb = vb0 + st * L::kTile;
        const uint32_t id = idesc_n(idS, n16);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t off = (k / 4) * kAtom + (k % 4) * 32;
          mma_bf16_ss(tS, smem_desc_sw128(qa + off), smem_desc_sw128(kb + off), id, k > 0);
        }
        tc_commit(s_full);
        tc_commit(&k_empty[st]);
        if (!role_wait(p_ready, it & 1, abort_flag)) break;
        if (!role_wait(&v_full[st], (it / kStages) & 1, abort_flag)) break;
        tc_fence_after();
        // V tiles are MN-major: 16 keys are 2,048 bytes on, the second 64 columns one atom on
        for (int k = 0; k < n16 / 16; ++k)
          mma_bf16_ts(tO, tS + 8 * k, smem_desc_sw128(vb + 2048 * k, D == 64 ? 16 : kAtom), idesc_n(idO, D),
                      it > 0 || k > 0);
        tc_commit(&v_empty[st]);
        ++it;
      }
      tc_commit(o_full);
      mbar_wait(o_full, 0);  // every MMA this thread issued has finished before TMEM is freed
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    // ---------------------------------------------------------------- queries into shared memory
    if (p.q_w) {  // rounded to the input's type, as the norm pass that this replaces stores it
      float w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = __ldg(p.q_w + qch * 8 + e);
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        uint32_t u[4] = {qv[i].x, qv[i].y, qv[i].z, qv[i].w};
        float2 f[4];
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          f[e] = unpack16<kFp16>(u[e]);
          ss = fmaf(f[e].x, f[e].x, fmaf(f[e].y, f[e].y, ss));
        }
#pragma unroll
        for (int o = 1; o < PPR; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float inv = rsqrtf(ss * (1.f / D) + p.eps);
#pragma unroll
        for (int e = 0; e < 4; ++e) u[e] = pack16<kFp16>(f[e].x * inv * w[2 * e], f[e].y * inv * w[2 * e + 1]);
        qv[i] = make_uint4(u[0], u[1], u[2], u[3]);
      }
    }
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const int r = warp * 32 + i * kRowsPerStep + lane / PPR;
      *reinterpret_cast<uint4*>(smem + (qch >> 3) * kAtom + sw128_offset(r, qch & 7)) = qv[i];
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(q_full);

    // ---------------------------------------------------------------- softmax
    const uint32_t lane_base = static_cast<uint32_t>(warp * 32) << 16;
    const uint32_t tS = tmem + lane_base, tO = tmem + lane_base + 128;
    const int row = warp * 32 + lane;
    float m = -INFINITY, l = 0.f;
    int it = 0;
    bool ok = true;
    for (int j = j0; j < j1; ++j) {
      const Tile t = tile_of<kMask>(p, j, n0, own_len, bits, j0);
      if (t.hi <= 0) continue;
      if (!(ok = warp_wait(s_full, it & 1, abort_flag))) break;
      tc_fence_after();
      uint32_t r[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32(tS + 32 * c, r[c]);
      tmem_wait_ld();
      if (!t.full) {  // columns past n16 hold an earlier tile's bits
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t word;
          if constexpr (kMask) {
            word = word_of(t.bits, c);
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
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int e = 0; e < 32; e += 2)
          mx[c] = fmax3(mx[c], __uint_as_float(r[c][e]), __uint_as_float(r[c][e + 1]));
      const float rmax = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.scale_log2;
      const float m_new = fmaxf(m, rmax);
      const bool upd = m_new > m + kRescaleThreshold;
      float alpha = 1.f;
      if (upd) {
        alpha = m == -INFINITY ? 0.f : ex2_approx(m - m_new);
        m = m_new;
      }
      const float nm = m == -INFINITY ? 0.f : -m;
      float rs[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t pk[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float x0, x1, p0, p1;
          ffma2(x0, x1, __uint_as_float(r[c][2 * e]), __uint_as_float(r[c][2 * e + 1]), p.scale_log2, p.scale_log2,
                nm, nm);
          if ((e & kPolyMask) == kPolyMask) {  // a share of the exponentials on the FMA pipe
            exp2_poly2(x0, x1, p0, p1);
          } else {
            p0 = ex2_approx(x0);
            p1 = ex2_approx(x1);
          }
          const int a2 = (e & 1) * 2;
          fadd2(rs[a2], rs[a2 + 1], rs[a2], rs[a2 + 1], p0, p1);
          // P in the input's type for the MMA (at most 2^8 above 1, relative error up to 2^-8 or 2^-11)
          pk[e] = pack16<kFp16>(p0, p1);
        }
        tmem_st16(tS + 16 * c, pk);
      }
      l = l * alpha + ((rs[0] + rs[1]) + (rs[2] + rs[3]));
      if (it > 0 && __any_sync(0xffffffffu, upd)) {
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
      if (t.clean) {  // this thread's V row, where its key is not valid
        const int st = it % kStages;
        if (!(ok = warp_wait(&v_full[st], (it / kStages) & 1, abort_flag))) break;
        bool valid = row < t.hi;
        if constexpr (kMask) valid = (word_of(t.bits, warp) >> lane) & 1u;
        if (!valid) {
          uint8_t* v = smem + L::kOffV + st * L::kTile;
#pragma unroll
          for (int c = 0; c < PPR; ++c)
            *reinterpret_cast<uint4*>(v + (c >> 3) * kAtom + sw128_offset(row, c & 7)) = make_uint4(0u, 0u, 0u, 0u);
        }
        fence_proxy_async_smem();
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_ready);
      ++it;
    }
    if (!ok) *abort_flag = 1;

    // ---------------------------------------------------------------- epilogue
    ok = warp_wait(o_full, 0, abort_flag) && ok;
    tc_fence_after();
    const int r = rt * 128 + row;
    if (p.slots == 1) {
      const float inv = l > 0.f ? 1.f / l : l;  // l 0: no key; NaN stays
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        tmem_ld32(tO + 32 * c, o);
        tmem_wait_ld();
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float a = __uint_as_float(o[q * 8 + 2 * e]) * inv, z = __uint_as_float(o[q * 8 + 2 * e + 1]) * inv;
            w[e] = l == 0.f ? 0u : pack16<kFp16>(a, z);
          }
          const int ch = c * 4 + q;
          *reinterpret_cast<uint4*>(smem + (ch >> 3) * kAtom + sw128_offset(row, ch & 7)) =
              make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
      __syncwarp();
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {  // whole rows, coalesced
        const int lr = warp * 32 + i * kRowsPerStep + lane / PPR, gr = rt * 128 + lr;
        if (ok && gr < rows) {
          const int tk = gr / p.G, hq = g * p.G + (gr - tk * p.G), tt = tok0 + tk, bq = tt / p.Lq;
          *reinterpret_cast<uint4*>(p.out + bq * p.o_bs + (tt - bq * p.Lq) * p.o_rs + (int64_t)hq * D + qch * 8) =
              *reinterpret_cast<const uint4*>(smem + (qch >> 3) * kAtom + sw128_offset(lr, qch & 7));
        }
      }
    } else {
      const int64_t rall = (int64_t)p.B * p.Lq * p.H;
      const int tk = r / p.G;
      const int64_t pr = (part.slot0 + split) * rall + (int64_t)(tok0 + tk) * p.H + g * p.G + (r - tk * p.G);
      if (r < rows) p.ml_part[pr] = make_float2(l == 0.f ? -INFINITY : m, l);
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        tmem_ld32(tO + 32 * c, o);
        tmem_wait_ld();
        if (r < rows) {
          float4* dst = reinterpret_cast<float4*>(p.o_part + pr * D + c * 32);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            dst[e] = make_float4(__uint_as_float(o[4 * e]), __uint_as_float(o[4 * e + 1]),
                                 __uint_as_float(o[4 * e + 2]), __uint_as_float(o[4 * e + 3]));
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
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

// `outer` x `mid` rows of `width` states; box 64 columns x 128 keys (the middle dimension, or the outer one where
// `keys_outer`), 128-byte swizzle; keys past the end read as zero.
bool encode_states(CUtensorMap* map, const void* base, bool fp16, int64_t width, int64_t mid, int64_t outer,
                   int64_t mid_stride, int64_t outer_stride, bool keys_outer) {
  auto encode = encode_fn();
  if (!encode) return false;
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(width), static_cast<cuuint64_t>(mid), static_cast<cuuint64_t>(outer)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(mid_stride) * 2, static_cast<cuuint64_t>(outer_stride) * 2};
  cuuint32_t box[3] = {64, keys_outer ? 1u : 128u, keys_outer ? 128u : 1u};
  cuuint32_t estr[3] = {1, 1, 1};
  return encode(map, fp16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, bool kFp16, bool kMask>
int launch_tiles(const CUtensorMap& own, const CUtensorMap& shared, const CtxParams& p, int mask_tiles,
                 cudaStream_t s) {
  auto kernel = ctx_tiles_kernel<D, kFp16, kMask>;
  // setmaxnreg's split counts on exactly kLaunchRegs registers per thread at launch (an increase that the CTA's
  // registers do not cover would never be granted), and two CTAs per SM on their TMEM
  cudaFuncAttributes attr{};
  if (cudaFuncGetAttributes(&attr, kernel) != cudaSuccess || attr.numRegs != kLaunchRegs) return HB_ERR_LAUNCH;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<D>::bytes(kCtxMaskTiles)) !=
      cudaSuccess)
    return HB_ERR_LAUNCH;
  kernel<<<p.part[0].ctas + p.part[1].ctas, kThreads, Layout<D>::bytes(mask_tiles), s>>>(own, shared, p);
  return cudaGetLastError() == cudaSuccess ? HB_OK : HB_ERR_LAUNCH;
}

template <int D, bool kFp16>
int launch_tiles(const CUtensorMap& own, const CUtensorMap& shared, const CtxParams& p, bool mask, int mask_tiles,
                 cudaStream_t s) {
  return mask ? launch_tiles<D, kFp16, true>(own, shared, p, mask_tiles, s)
              : launch_tiles<D, kFp16, false>(own, shared, p, 0, s);
}

}  // namespace

int ctx_tiles_take_status(unsigned int* status) {
  unsigned int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_device_status_local, sizeof(v)) != cudaSuccess) return HB_ERR_LAUNCH;
  if (v && cudaMemcpyToSymbol(g_device_status_local, &zero, sizeof(zero)) != cudaSuccess) return HB_ERR_LAUNCH;
  *status = v;
  return HB_OK;
}

int launch_ctx_tiles(const CtxParams& p, int D, bool fp16, int mask_tiles, cudaStream_t s) {
  const int64_t width = 2ll * p.Hkv * D;
  CUtensorMap own{}, shared{};
  const bool use_own = p.Lkv > 0 && (p.part[0].use_own || p.part[1].use_own);
  const bool use_shared = p.part[0].use_shared != 0;
  const int64_t batch = p.kv_bs == 0 ? 1 : p.B;  // one copy of the states is a batch of one to the map
  if (use_own &&
      !(p.kv_inter ? encode_states(&own, p.kv, fp16, width, batch, p.Lkv, p.kv_bs, p.kv_rs, true)
                   : encode_states(&own, p.kv, fp16, width, p.Lkv, batch, p.kv_rs,
                                   batch > 1 ? p.kv_bs : p.kv_rs * p.Lkv, false)))
    return HB_ERR_LAUNCH;
  if (use_shared && !encode_states(&shared, p.skv, fp16, width, p.Ls, 1, p.skv_rs, p.skv_rs * p.Ls, false))
    return HB_ERR_LAUNCH;
  if (!use_own) own = shared;
  if (!use_shared) shared = own;
  const bool mask = p.mask || p.smask;
  if (D == 128)
    return fp16 ? launch_tiles<128, true>(own, shared, p, mask, mask_tiles, s)
                : launch_tiles<128, false>(own, shared, p, mask, mask_tiles, s);
  return fp16 ? launch_tiles<64, true>(own, shared, p, mask, mask_tiles, s)
              : launch_tiles<64, false>(own, shared, p, mask, mask_tiles, s);
}

}  // namespace hb
