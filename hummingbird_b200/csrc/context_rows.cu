// Context attention for few query rows (single tokens, short runs), and the merge of partial results.
//
// For every row r (a query token and a query head) of a kv head,
//   o_r = sum_j p_rj v_j / sum_j p_rj,   p_rj = exp2(c q_r . k_j - m_r),  m_r = max_j c q_r . k_j,
// over the valid keys j, in one pass over k and v: the maximum and the sum run along (fp32), o is rescaled when the
// maximum moves. With 16 or 32 rows per kv head the work is the bytes of k and v (4 D bytes per key and kv head
// against 64 D flops), so the kernel is a stream through shared memory: each warp walks its own 8 KiB chunks of the
// key list (32 keys at D 64, 16 at D 128) through a private three-stage ring of 16-byte asynchronous copies, with no
// barrier between warps; m16n8k16 MMAs take the scores and P V, whose unused rows cost nothing that the bytes do
// not cost already. The four warps of a CTA merge through shared memory, CTAs of a split key list through
// (m, l, o) partials that ctx_combine_kernel joins in slot order, so results do not depend on timing.
// Batch 8, one token, 32,768 keys, 16 heads over 4, D 64: 49 us with the merge, 5.5 TB/s, 84 % of the measured copy
// rate. Two CTAs per SM hold 128 KB of copies in flight, where about 35 KB cover the memory's latency.
// Keys that the mask or the length leaves out are copied as zeros (their memory is not read) and their scores set
// to -inf, so what lies there cannot reach the result; a row without keys gets zeros.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "context_attn.h"
#include "hb_sm100.cuh"
#include "launch_after.h"

namespace hb {
namespace {

constexpr int kWarps = 4;
constexpr int kStages = 3;
constexpr int kChunkBytes = 8192;  // K and V of one chunk
constexpr int kWarpBytes = kStages * kChunkBytes;
constexpr int kRowsSmem = kWarps * kWarpBytes + kWarps * kStages * 4 + kWarps * 32 * 8;

// kLift: all weights p <= 1 are multiplied by 2^kLift, so that small ones stay in the type's normal range for P V.
// fp16's ends at 2^-14 (its subnormals at 2^-24): lifted, weights down to 2^-29 of the largest keep 11 bits, smaller
// ones are off by at most 2^-40 of it.
struct Bf16 {
  static constexpr float kLift = 0.f;
  static __device__ __forceinline__ float2 unpack(uint32_t w) { return {bf16_lo(w), bf16_hi(w)}; }
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_bf16x2(a, b); }
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
struct Fp16 {
  static constexpr float kLift = 15.f;
  static __device__ __forceinline__ float2 unpack(uint32_t w) { return __half22float2(*reinterpret_cast<__half2*>(&w)); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// 16 bytes global -> shared; `bytes` 0 writes zeros and reads nothing.
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Byte offset of 16-byte piece `ch` of row `row` in a chunk of D-element rows, pieces exchanged by the row so that
// the eight rows of an 8x8 matrix lie in different banks.
template <int D>
__device__ __forceinline__ uint32_t piece(int row, int ch) {
  return static_cast<uint32_t>(row * (D * 2) + ((ch ^ (row & 7)) << 4));
}

template <int D, class T, int MT>
__global__ void __launch_bounds__(32 * kWarps, 2) ctx_rows_kernel(const CtxParams p) {
  constexpr int KC = kChunkBytes / (4 * D);  // keys per chunk
  constexpr int PPR = D / 8;                 // 16-byte pieces per row
  constexpr int KK = D / 16;
  extern __shared__ __align__(128) uint8_t smem[];
  uint32_t* bits_s = reinterpret_cast<uint32_t*>(smem + kWarps * kWarpBytes);
  float2* ml_s = reinterpret_cast<float2*>(smem + kWarps * kWarpBytes + kWarps * kStages * 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, tid = lane & 3;
  wait_for_kernel_before();

  // ---- which item
  const bool second = static_cast<int>(blockIdx.x) >= p.part[0].count;
  const CtxPart& part = p.part[second ? 1 : 0];
  const CtxUnit u = ctx_unit(p, part, blockIdx.x - (second ? p.part[0].count : 0));
  const int g = u.g, b = u.b, r0 = u.rt * 16 * MT;

  // ---- query fragments (a row's RMSNorm when asked for, rounded to the input's type like the norm it replaces)
  uint32_t qf[MT][KK][4];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const int r = r0 + mt * 16 + hf * 8 + gid;
      const bool live = r < u.rows;
      const CtxRow x = ctx_row(p, live ? r : 0, g, b, part.pooled);
      const uint16_t* src = p.q + x.bq * p.q_bs + x.i * p.q_rs + (int64_t)x.hq * D;
      float ss = 0.f;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint32_t w = live ? *reinterpret_cast<const uint32_t*>(src + kk * 16 + half * 8 + tid * 2) : 0u;
          qf[mt][kk][half * 2 + hf] = w;
          const float2 f = T::unpack(w);
          ss = fmaf(f.x, f.x, fmaf(f.y, f.y, ss));
        }
      if (p.q_w) {
        ss += __shfl_xor_sync(0xffffffffu, ss, 1);
        ss += __shfl_xor_sync(0xffffffffu, ss, 2);
        const float inv = rsqrtf(ss * (1.f / D) + p.eps);
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const float2 w = *reinterpret_cast<const float2*>(p.q_w + kk * 16 + half * 8 + tid * 2);
            const float2 f = T::unpack(qf[mt][kk][half * 2 + hf]);
            qf[mt][kk][half * 2 + hf] = T::pack(f.x * inv * w.x, f.y * inv * w.y);
          }
      }
    }
  }

  // ---- this CTA's chunks of the key list (shared keys, then the batch element's own)
  const int own_len = part.use_own ? ctx_own_len(p, b) : 0;
  const int n0 = part.use_shared ? (p.Ls + KC - 1) / KC : 0;
  const int n = n0 + (own_len + KC - 1) / KC;
  const int c_begin = part.by_splits.div(u.split * n);
  const int c_end = part.by_splits.div((u.split + 1) * n);
  const uint32_t ring = smem_u32(smem) + warp * kWarpBytes;
  uint32_t* bits_w = bits_s + warp * kStages;

  auto load = [&](int c, int st) {  // one commit group, also where nothing is copied
    if (c < c_end) {
      const bool sh = c < n0;
      const int k0 = (sh ? c : c - n0) * KC;
      const int len = sh ? p.Ls : own_len;
      const uint8_t* mk = sh ? p.smask : p.mask;
      if (mk && !sh) mk += b * p.mask_bs;
      bool v = lane < KC && k0 + lane < len;
      if (v && mk) v = mk[k0 + lane] != 0;
      const uint32_t bits = __ballot_sync(0xffffffffu, v);
      if (lane == 0) bits_w[st] = bits;
      if (bits) {
        const uint16_t* base = sh ? p.skv : p.kv + b * p.kv_bs;
        const int64_t rs = sh ? p.skv_rs : p.kv_rs;
        base += (int64_t)g * D;
        const uint32_t dst = ring + st * kChunkBytes;
        const int ch = lane % PPR;
#pragma unroll
        for (int i = 0; i < KC * PPR / 32; ++i) {
          const int key = i * (32 / PPR) + lane / PPR;
          const bool kv_ok = (bits >> key) & 1u;
          const uint16_t* src = base + (kv_ok ? (int64_t)(k0 + key) * rs + ch * 8 : 0);
          const uint32_t o = dst + piece<D>(key, ch);
          cp16(o, src, kv_ok ? 16u : 0u);
          cp16(o + kChunkBytes / 2, src + (kv_ok ? (int64_t)p.Hkv * D : 0), kv_ok ? 16u : 0u);
        }
      }
    }
    cp_commit();
  };

  float o[MT][D / 8][4];
  float m[MT][2], l[MT][2];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    m[mt][0] = m[mt][1] = -INFINITY;
    l[mt][0] = l[mt][1] = 0.f;
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[mt][i][e] = 0.f;
  }

  const int c0 = c_begin + warp;
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) load(c0 + s * kWarps, s);
  int st = 0;
  for (int c = c0; c < c_end; c += kWarps) {
    {
      int nst = st + kStages - 1;
      if (nst >= kStages) nst -= kStages;
      load(c + (kStages - 1) * kWarps, nst);  // the stage that the last iteration released
    }
    cp_wait<kStages - 1>();
    __syncwarp();
    const uint32_t bits = bits_w[st];
    if (bits) {
      const uint32_t kb = ring + st * kChunkBytes, vb = kb + kChunkBytes / 2;
      float s[MT][KC / 8][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < KC / 8; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[mt][i][e] = 0.f;
#pragma unroll
      for (int kt = 0; kt < KC / 16; ++kt) {
        const int key = kt * 16 + ((lane >> 4) << 3) + (lane & 7);
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
          uint32_t bfr[4];
          ldsm4(bfr, kb + piece<D>(key, kk * 2 + ((lane >> 3) & 1)));
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            T::mma(s[mt][kt * 2], qf[mt][kk], bfr[0], bfr[1]);
            T::mma(s[mt][kt * 2 + 1], qf[mt][kk], bfr[2], bfr[3]);
          }
        }
      }
      constexpr uint32_t kFull = KC == 32 ? 0xffffffffu : (1u << KC) - 1u;
      uint32_t pf[MT][KC / 16][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        if (bits != kFull) {
#pragma unroll
          for (int i = 0; i < KC / 8; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (!((bits >> (i * 8 + tid * 2 + (e & 1))) & 1u)) s[mt][i][e] = -INFINITY;
        }
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < KC / 8; ++i) {
          mx[0] = fmax3(mx[0], s[mt][i][0], s[mt][i][1]);
          mx[1] = fmax3(mx[1], s[mt][i][2], s[mt][i][3]);
        }
        float nm[2];
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          mx[hf] = fmaxf(mx[hf], __shfl_xor_sync(0xffffffffu, mx[hf], 1));
          mx[hf] = fmaxf(mx[hf], __shfl_xor_sync(0xffffffffu, mx[hf], 2));
          const float mn = fmaxf(m[mt][hf], mx[hf] * p.scale_log2);
          const float alpha = mn == -INFINITY ? 1.f : ex2_approx(m[mt][hf] - mn);
          m[mt][hf] = mn;
          nm[hf] = mn == -INFINITY ? 0.f : T::kLift - mn;
          l[mt][hf] *= alpha;
#pragma unroll
          for (int i = 0; i < D / 8; ++i) {
            o[mt][i][hf * 2] *= alpha;
            o[mt][i][hf * 2 + 1] *= alpha;
          }
        }
#pragma unroll
        for (int i = 0; i < KC / 8; ++i) {
          float e[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            e[j] = ex2_approx(fmaf(s[mt][i][j], p.scale_log2, nm[j >> 1]));
            l[mt][j >> 1] += e[j];
          }
          // P in the input's type for the MMA (relative error up to 2^-8 or 2^-11); l keeps fp32
          pf[mt][i >> 1][(i & 1) * 2] = T::pack(e[0], e[1]);
          pf[mt][i >> 1][(i & 1) * 2 + 1] = T::pack(e[2], e[3]);
        }
      }
#pragma unroll
      for (int kt = 0; kt < KC / 16; ++kt) {
        const int key = kt * 16 + (((lane >> 3) & 1) << 3) + (lane & 7);
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) {
          uint32_t bfr[4];
          ldsm4_t(bfr, vb + piece<D>(key, dt * 2 + (lane >> 4)));
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            T::mma(o[mt][dt * 2], pf[mt][kt], bfr[0], bfr[1]);
            T::mma(o[mt][dt * 2 + 1], pf[mt][kt], bfr[2], bfr[3]);
          }
        }
      }
    }
    __syncwarp();  // every lane has read this stage before it is filled again
    if (++st == kStages) st = 0;
  }
  cp_wait<0>();

  // ---- merge the warps
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      l[mt][hf] += __shfl_xor_sync(0xffffffffu, l[mt][hf], 1);
      l[mt][hf] += __shfl_xor_sync(0xffffffffu, l[mt][hf], 2);
    }
  __syncthreads();  // the rings are free
  constexpr int kRows = 16 * MT;
  constexpr int kPitch = D + 4;  // fp32 elements
  float* o_s = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const int row = mt * 16 + hf * 8 + gid;
      if (tid == 0) ml_s[warp * 32 + row] = make_float2(m[mt][hf], l[mt][hf]);
      float* dst = o_s + (warp * kRows + row) * kPitch + tid * 2;
#pragma unroll
      for (int i = 0; i < D / 8; ++i)
        *reinterpret_cast<float2*>(dst + i * 8) = make_float2(o[mt][i][hf * 2], o[mt][i][hf * 2 + 1]);
    }
  __syncthreads();
  for (int i = threadIdx.x; i < kRows * PPR; i += 32 * kWarps) {
    const int row = i / PPR, ch = i % PPR, r = r0 + row;
    if (r >= u.rows) continue;
    float mw[kWarps], mx = -INFINITY, sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, mw[w] = ml_s[w * 32 + row].x);
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = mw[w] == -INFINITY ? 0.f : ex2_approx(mw[w] - mx);
      sum = fmaf(f, ml_s[w * 32 + row].y, sum);
      const float* src = o_s + (w * kRows + row) * kPitch + ch * 8;
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = fmaf(f, src[e], acc[e]);
    }
    const CtxRow x = ctx_row(p, r, g, b, part.pooled);
    if (part.direct) {
      const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
      uint4 w;
      w.x = T::pack(acc[0] * inv, acc[1] * inv);
      w.y = T::pack(acc[2] * inv, acc[3] * inv);
      w.z = T::pack(acc[4] * inv, acc[5] * inv);
      w.w = T::pack(acc[6] * inv, acc[7] * inv);
      *reinterpret_cast<uint4*>(p.out + x.bq * p.o_bs + x.i * p.o_rs + (int64_t)x.hq * D + ch * 8) = w;
    } else {
      const int64_t pr = ctx_prow(p, part, u, x, row);
      if (ch == 0) p.ml_part[pr] = make_float2(mx - T::kLift, sum);
      float4* dst = reinterpret_cast<float4*>(p.o_part + pr * D + ch * 8);
      dst[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
      dst[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
    }
  }
}

// out = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s; four elements of a row per thread, kTeams teams of D / 4 threads
// to a row, which take every kTeams-th slot and join in order: a long list of slots would otherwise be one thread's.
template <int D, class T, int kTeams>
__global__ void __launch_bounds__(256) ctx_combine_kernel(const CtxParams p) {
  constexpr int TPR = D / 4;
  wait_for_kernel_before();  // the partial results of every kernel of this call
  __shared__ float4 acc_s[256];
  __shared__ float2 ml_s[256];
  const int idx = static_cast<int>(((int64_t)blockIdx.x * 256 + threadIdx.x) / TPR);
  const int row = idx / kTeams, team = idx % kTeams, ch = threadIdx.x % TPR;
  bool live = row < p.prows;
  CtxRow x{};
  if (p.tail_rows) {
    const CtxPart& part = p.part[1];
    const int i = row / p.tail_rows;
    const CtxUnit u = ctx_unit(p, part, live ? i * part.splits : 0);
    const int r = u.rt * p.tail_rows + (row - i * p.tail_rows);
    live = live && r < u.rows;
    if (live) x = ctx_row(p, r, u.g, u.b, part.pooled);
  } else if (live) {
    const int t = p.by_h.div(row);
    x.hq = row - t * p.H;
    x.bq = p.by_lq.div(t);
    x.i = t - x.bq * p.Lq;
  }
  float mx = -INFINITY, sum = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (live) {
    for (int s = team; s < p.slots; s += kTeams) mx = fmaxf(mx, p.ml_part[(int64_t)s * p.prows + row].x);
#pragma unroll 4
    for (int s = team; s < p.slots; s += kTeams) {
      const float2 ml = p.ml_part[(int64_t)s * p.prows + row];
      if (ml.y == 0.f) continue;  // a part without keys (m = -inf, but a NaN row may have that too) left no sums
      const float f = ex2_approx(ml.x - mx);
      const float4 v = *reinterpret_cast<const float4*>(p.o_part + ((int64_t)s * p.prows + row) * D + ch * 4);
      sum = fmaf(f, ml.y, sum);
      acc.x = fmaf(f, v.x, acc.x);
      acc.y = fmaf(f, v.y, acc.y);
      acc.z = fmaf(f, v.z, acc.z);
      acc.w = fmaf(f, v.w, acc.w);
    }
  }
  if constexpr (kTeams > 1) {
    acc_s[threadIdx.x] = acc;
    ml_s[threadIdx.x] = make_float2(mx, sum);
    __syncthreads();
    if (!live || team) return;
#pragma unroll
    for (int k = 1; k < kTeams; ++k) mx = fmaxf(mx, ml_s[threadIdx.x + k * TPR].x);
    sum = 0.f;
    acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < kTeams; ++k) {
      const float2 ml = ml_s[threadIdx.x + k * TPR];
      if (ml.y == 0.f) continue;
      const float f = ex2_approx(ml.x - mx);
      const float4 v = acc_s[threadIdx.x + k * TPR];
      sum = fmaf(f, ml.y, sum);
      acc.x = fmaf(f, v.x, acc.x);
      acc.y = fmaf(f, v.y, acc.y);
      acc.z = fmaf(f, v.z, acc.z);
      acc.w = fmaf(f, v.w, acc.w);
    }
  }
  if (!live) return;
  const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
  uint2 w;
  w.x = T::pack(acc.x * inv, acc.y * inv);
  w.y = T::pack(acc.z * inv, acc.w * inv);
  *reinterpret_cast<uint2*>(p.out + x.bq * p.o_bs + x.i * p.o_rs + (int64_t)x.hq * D + ch * 4) = w;
}

template <int D, class T, int MT>
int launch_rows(const CtxParams& p, cudaStream_t s) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return HB_ERR_LAUNCH;
  static bool configured[64] = {};
  if (dev >= 64 || !configured[dev]) {
    if (cudaFuncSetAttribute(ctx_rows_kernel<D, T, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRowsSmem) !=
        cudaSuccess)
      return HB_ERR_LAUNCH;
    if (dev < 64) configured[dev] = true;
  }
  return launch_after(ctx_rows_kernel<D, T, MT>, p.part[0].count + p.part[1].count, 32 * kWarps, kRowsSmem, s, p);
}

template <int D, class T, int kTeams>
int launch_teams(const CtxParams& p, cudaStream_t s) {
  const int64_t threads = (int64_t)p.prows * (D / 4) * kTeams;
  return launch_after(ctx_combine_kernel<D, T, kTeams>, static_cast<unsigned>((threads + 255) / 256), 256, 0, s, p);
}
// As many teams as it takes to have about a thousand threads on every SM, and no more than have slots to read.
template <int D, class T>
int launch_combine(const CtxParams& p, cudaStream_t s) {
  const int64_t threads = (int64_t)p.prows * (D / 4), want = kCtxSms * 1024;
  if (p.slots <= 4 || threads >= want) return launch_teams<D, T, 1>(p, s);
  if (p.slots <= 16 || 4 * threads >= want) return launch_teams<D, T, 4>(p, s);
  return launch_teams<D, T, 1024 / D>(p, s);
}

}  // namespace

int launch_ctx_rows(const CtxParams& p, int D, bool fp16, int rows_per_tile, cudaStream_t s) {
  if (D == 128) return fp16 ? launch_rows<128, Fp16, 1>(p, s) : launch_rows<128, Bf16, 1>(p, s);
  if (rows_per_tile == 32) return fp16 ? launch_rows<64, Fp16, 2>(p, s) : launch_rows<64, Bf16, 2>(p, s);
  return fp16 ? launch_rows<64, Fp16, 1>(p, s) : launch_rows<64, Bf16, 1>(p, s);
}

int launch_ctx_combine(const CtxParams& p, int D, bool fp16, cudaStream_t s) {
  if (D == 128) return fp16 ? launch_combine<128, Fp16>(p, s) : launch_combine<128, Bf16>(p, s);
  return fp16 ? launch_combine<64, Fp16>(p, s) : launch_combine<64, Bf16>(p, s);
}

}  // namespace hb
