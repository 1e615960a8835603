// Linear layers with 4-bit weights and group scales for a few rows (the conditioning vectors of a DiT step: one
// row per clip), and the quantiser that lays their weights out.
//
//   y[m, n] = act(sum_k x[m, k] q[n, k] s[n, k / group] + bias[n]),  q in [-8, 7]
//
// With few rows the work is the bytes of the weights (1/2 + 2 / group per weight), so the layout makes them one
// coalesced stream: blocks of 16 outputs x 128 inputs (1 KiB), in which a lane's two 16-byte loads are exactly its
// share of the A operand of m16n8k16 MMAs (A: 16 outputs x 16 inputs, B: 16 inputs x 8 rows of x). Lane (row r, t)
// holds inputs 32 w + 8 t .. + 8 of output rows r and r + 8 in its w-th words, so that 32 consecutive inputs are
// one word step of the warp and every group of 32, 64 or 128 inputs ends at a step. The nibbles of a word are
// ordered 0 2 4 6 1 3 5 7: shifting it by 4 i leaves inputs 2 i, 2 i + 1 in its two halves. A nibble u = q + 8 is
// or-ed into the mantissa of 128 (bf16) or 1024 (fp16) and 136 or 1032 subtracted: q exactly, without a conversion.
// Each group's sum is accumulated by the MMAs in fp32 and multiplied by its scale once, in fp32.
//
// One CTA takes 16 outputs (or 32); its four warps take every fourth block of 128 inputs, each through a ring of
// asynchronous copies of its own, and merge through shared memory in warp order, so the result does not depend on
// timing. x is read through L1 (it is the same few rows for every CTA).
// One row, 16,384 x 8,192, group 128: 17.4 us, 4.0 TB/s, 61 % of the measured copy rate. Nothing is full: issue 58 %,
// integer pipe 50 % (22 us with two logic operations to a nibble pair); the longest stall is the wait for x, and 1,024 CTAs
// on 888 places leave a short second round. 32 rows: 45.7 us, as long as a bf16 product takes (44.7): every CTA reads all
// of x through L1, eight warps an SM wait for it (issue 31 %, tensor pipe 40 %).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "../../include/hb_b200.h"
#include "abi_common.h"
#include "hb_sm100.cuh"
#include "launch_after.h"
#include "prep_common.cuh"

namespace hb {
namespace {

constexpr int kWarps = 4;
constexpr int kStages = 4;  // blocks of a warp on their way

struct W4Params {
  const uint16_t* x;
  int64_t ldx;
  const uint4* packed;
  const uint16_t* scales;  // bf16 [tiles][blocks][128 / group][16]
  const uint16_t* bias;
  uint16_t* y;
  int64_t ldy;
  int M, N, K, kblocks, silu;
};

// (a & b) | c as one operation (from the expression the compiler makes two, each with its constant in place).
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}

template <bool kFp16>
struct Half;
template <>
struct Half<false> {
  // The pairs 0 1, 2 3, 4 5, 6 7 of a word's weights.
  static __device__ __forceinline__ void weights(uint32_t w, uint32_t& p0, uint32_t& p1, uint32_t& p2, uint32_t& p3) {
    p0 = pair(w);
    p1 = pair(w >> 4);
    p2 = pair(w >> 8);
    p3 = pair(w >> 12);
  }
  static __device__ __forceinline__ uint32_t pair(uint32_t w) {  // nibbles 0 and 4
    const uint32_t u = and_or(w, 0x000f000fu, 0x43004300u);
    const __nv_bfloat162 off = __floats2bfloat162_rn(136.f, 136.f);
    const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&u), off);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ float load(const uint16_t* p) { return __uint_as_float((uint32_t)*p << 16); }
  static __device__ __forceinline__ uint16_t round(float v) { return __bfloat16_as_ushort(__float2bfloat16_rn(v)); }
};
template <>
struct Half<true> {
  // fp16's mantissa has room for a nibble at bit 4 too: 1024 + 16 u, exactly u - 8 after one FMA.
  static __device__ __forceinline__ void weights(uint32_t w, uint32_t& p0, uint32_t& p1, uint32_t& p2, uint32_t& p3) {
    const uint32_t v = w >> 8;
    p0 = low(w);
    p1 = high(w);
    p2 = low(v);
    p3 = high(v);
  }
  static __device__ __forceinline__ uint32_t low(uint32_t w) {
    const uint32_t u = and_or(w, 0x000f000fu, 0x64006400u);
    const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&u), __floats2half2_rn(1032.f, 1032.f));
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ uint32_t high(uint32_t w) {
    const uint32_t u = and_or(w, 0x00f000f0u, 0x64006400u);
    const __half2 v = __hfma2(*reinterpret_cast<const __half2*>(&u), __floats2half2_rn(0.0625f, 0.0625f),
                              __floats2half2_rn(-72.f, -72.f));
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ float load(const uint16_t* p) { return __half2float(__ushort_as_half(*p)); }
  static __device__ __forceinline__ uint16_t round(float v) { return __half_as_ushort(__float2half_rn(v)); }
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// NT: groups of eight rows of x. RT: tiles of 16 outputs that share what a warp reads of x.
template <bool kFp16, int NT, int RT, int kGroup>
__global__ void __launch_bounds__(32 * kWarps, NT == 1 ? 6 : NT == 2 ? 4 : 3 - RT / 2) w4_linear_kernel(const W4Params p) {
  using T = Half<kFp16>;
  constexpr int kSteps = kGroup / 32;        // word steps per group
  constexpr int kGroups = 128 / kGroup;      // groups per block
  constexpr int kTileBytes = 1024 + 32 * kGroups, kStageBytes = RT * kTileBytes;
  constexpr int kRing = kStages * kStageBytes;
  constexpr int kRow = 8 * NT + 1, kPart = RT * 16 * kRow * 4;
  __shared__ __align__(16) uint8_t smem[kWarps * (kRing > kPart ? kRing : kPart)];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, tid = lane & 3;
  wait_for_kernel_before();
  const int tile = blockIdx.x * RT, m0 = blockIdx.y * 8 * NT;

  float acc[RT][NT][4];
#pragma unroll
  for (int q = 0; q < RT; ++q)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[q][t][e] = 0.f;

  // Each warp's blocks through a ring of its own: a lane copies what it reads of the weights itself, the scales are
  // read by all. Integer operations are most of this loop (seven to a word of eight weights), so all else is kept off
  // that pipe: pointers that step, stages by unrolling, rows past M read as row M - 1 (their columns are dropped).
  const uint8_t* wp =
      reinterpret_cast<const uint8_t*>(p.packed) + ((int64_t)tile * p.kblocks + warp) * 1024 + lane * 16;
  const uint8_t* sp = reinterpret_cast<const uint8_t*>(p.scales) +
                      ((int64_t)tile * p.kblocks + warp) * (32 * kGroups) + (lane < 2 * kGroups ? lane * 16 : 0);
  const uint8_t* ring = smem + warp * kRing;
  const uint32_t ring_at = smem_u32(ring) + lane * 16;
  // (an odd number of tiles: the last one twice, and its second result dropped)
  const int64_t more_tiles = RT > 1 && (tile + 1) * 16 < p.N ? p.kblocks : 0;
  const int mine = (p.kblocks - warp + kWarps - 1) / kWarps;  // this warp's blocks
  auto load = [&](bool more, int st) {  // the next block; one commit group, also where there is none
    if (more) {
#pragma unroll
      for (int q = 0; q < RT; ++q) {
        const uint32_t dst = ring_at + st * kStageBytes + q * kTileBytes;
        const uint8_t *w = wp + q * more_tiles * 1024, *s = sp + q * more_tiles * (32 * kGroups);
        cp16(dst, w);
        cp16(dst + 512, w + 512);
        if (lane < 2 * kGroups) cp16(dst + 1024, s);
      }
      wp += kWarps * 1024;
      sp += kWarps * (32 * kGroups);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) load(s < mine, s);

  const uint16_t* xp[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) xp[t] = p.x + min(m0 + t * 8 + gid, p.M - 1) * p.ldx + warp * 128 + tid * 8;
  for (int i0 = 0; i0 < mine; i0 += kStages) {
#pragma unroll
    for (int st = 0; st < kStages; ++st) {
      const int i = i0 + st;
      if (i >= mine) break;
      load(i + kStages - 1 < mine, (st + kStages - 1) % kStages);
      uint4 xv[NT][4];
      if ((i * kWarps + warp) * 128 + 128 <= p.K) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int w = 0; w < 4; ++w) xv[t][w] = *reinterpret_cast<const uint4*>(xp[t] + 32 * w);
      } else {  // the row's last block, where K is no multiple of 128
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int w = 0; w < 4; ++w)
            xv[t][w] = (i * kWarps + warp) * 128 + 32 * w < p.K ? *reinterpret_cast<const uint4*>(xp[t] + 32 * w)
                                                                : make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) xp[t] += kWarps * 128;
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
      __syncwarp();
#pragma unroll
      for (int q = 0; q < RT; ++q) {
        const uint8_t* stage = ring + st * kStageBytes + q * kTileBytes;
        const uint4 wa = *reinterpret_cast<const uint4*>(stage + lane * 16);
        const uint4 wb = *reinterpret_cast<const uint4*>(stage + 512 + lane * 16);
        const uint32_t lo[4] = {wa.x, wa.y, wa.z, wa.w}, hi[4] = {wb.x, wb.y, wb.z, wb.w};
        const uint16_t* sc = reinterpret_cast<const uint16_t*>(stage + 1024) + gid;
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
          float c[NT][4];
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) c[t][e] = 0.f;
#pragma unroll
          for (int s = 0; s < kSteps; ++s) {
            const int w = g * kSteps + s;
            uint32_t a0[4], a1[4];
            T::weights(lo[w], a0[0], a0[2], a1[0], a1[2]);
            T::weights(hi[w], a0[1], a0[3], a1[1], a1[3]);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              T::mma(c[t], a0, xv[t][w].x, xv[t][w].y);
              T::mma(c[t], a1, xv[t][w].z, xv[t][w].w);
            }
          }
          const float s0 = __uint_as_float((uint32_t)sc[g * 16] << 16);
          const float s1 = __uint_as_float((uint32_t)sc[g * 16 + 8] << 16);
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[q][t][e] = fmaf(e < 2 ? s0 : s1, c[t][e], acc[q][t][e]);
        }
      }
      __syncwarp();  // every lane has read the stage's scales before it is filled again
    }
  }
  __syncthreads();  // (the copies still in flight are empty groups) the rings become the partial sums
  float* part = reinterpret_cast<float*>(smem);
  constexpr int kWarp = RT * 16 * kRow;
#pragma unroll
  for (int q = 0; q < RT; ++q)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        part[warp * kWarp + (q * 16 + gid + 8 * (e >> 1)) * kRow + t * 8 + tid * 2 + (e & 1)] = acc[q][t][e];
  __syncthreads();
  const int warps = min(kWarps, p.kblocks);
  for (int i = threadIdx.x; i < RT * 128 * NT; i += 32 * kWarps) {
    const int r = i % (16 * RT), c = i / (16 * RT), n = tile * 16 + r, m = m0 + c;
    if (n >= p.N || m >= p.M) continue;
    float v = part[r * kRow + c];
    for (int w = 1; w < warps; ++w) v += part[w * kWarp + r * kRow + c];
    if (p.bias) v += T::load(p.bias + n);
    if (p.silu) v = v / (1.f + expf(-v));
    p.y[m * p.ldy + n] = T::round(v);
  }
}

// Half a warp per (output row, 128-input block): lane i holds inputs 8 i .. 8 i + 8. Rows past N and inputs past K
// become zeros with scale 0, so the linear layer reads whole blocks.
template <int kGroup>
__global__ void __launch_bounds__(256) w4_quant_kernel(const uint16_t* __restrict__ w, int64_t ldw, int N, int K,
                                                       int tiles, int kblocks, uint32_t* __restrict__ packed,
                                                       uint16_t* __restrict__ scales) {
  const int64_t unit = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 4;
  const int i = threadIdx.x & 15;
  if (unit >= (int64_t)tiles * 16 * kblocks) return;  // whole half-warps; the shuffles below stay inside one
  const int64_t row = unit / kblocks;
  const int kb = static_cast<int>(unit - row * kblocks);
  const int k = kb * 128 + i * 8;
  const bool live = row < N && k < K;
  float v[8];
  if (live) {
    unpack8(__ldg(reinterpret_cast<const uint4*>(w + row * ldw + k)), v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.f;
  }
  float amax = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(v[e]));
  const unsigned half = 0xffffu << (threadIdx.x & 16);
#pragma unroll
  for (int o = 1; o < kGroup / 8; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(half, amax, o));
  float s = bf16_lo(__bfloat16_as_ushort(__float2bfloat16_rn(__fdiv_rn(amax, 7.f))));
  if (s == 0.f) s = 1.f;
  uint32_t word = 0u;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int q = static_cast<int>(fminf(fmaxf(rintf(__fdiv_rn(v[e], s)), -7.f), 7.f)) + 8;
    word |= static_cast<uint32_t>(q) << (4 * ((e >> 1) + 4 * (e & 1)));
  }
  const int64_t tile = row >> 4;
  const int r = static_cast<int>(row & 15), t = i & 3, ws = i >> 2;
  packed[(tile * kblocks + kb) * 256 + (r >> 3) * 128 + (r & 7) * 16 + t * 4 + ws] = word;
  if (i % (kGroup / 8) == 0)
    scales[((tile * kblocks + kb) * (128 / kGroup) + i / (kGroup / 8)) * 16 + r] =
        live ? __bfloat16_as_ushort(__float2bfloat16_rn(s)) : 0;
}

template <bool kFp16, int NT, int RT>
int launch_linear(const W4Params& p, int group, cudaStream_t s) {
  const dim3 grid((p.N + 16 * RT - 1) / (16 * RT), (p.M + 8 * NT - 1) / (8 * NT));
  if (group == 32) return launch_after(w4_linear_kernel<kFp16, NT, RT, 32>, grid, 32 * kWarps, 0, s, p);
  if (group == 64) return launch_after(w4_linear_kernel<kFp16, NT, RT, 64>, grid, 32 * kWarps, 0, s, p);
  return launch_after(w4_linear_kernel<kFp16, NT, RT, 128>, grid, 32 * kWarps, 0, s, p);
}
template <bool kFp16>
int launch_linear(const W4Params& p, int group, cudaStream_t s) {
  // Two tiles to a CTA halve the reads of x, at half the CTAs: worth it where x is more than L1 keeps beside the rings
  // and the CTAs still fill the GPU (16,384 x 8,192: 16 rows 36.8 -> 25.2 us, 32 rows 59.9 -> 46.0; below that
  // slower: 8,201 x 4,096, 13 rows 9.1 -> 9.9 us, 2,000 x 4,096 5.9 -> 7.8).
  const bool wide = (int64_t)p.M * p.K * 2 > 160 * 1024 && p.N > 2 * 148 * 16;
  if (p.M <= 8) return launch_linear<kFp16, 1, 1>(p, group, s);
  if (p.M <= 16) return wide ? launch_linear<kFp16, 2, 2>(p, group, s) : launch_linear<kFp16, 2, 1>(p, group, s);
  return wide ? launch_linear<kFp16, 4, 2>(p, group, s) : launch_linear<kFp16, 4, 1>(p, group, s);
}

bool w4_shape_ok(int N, int K, int group) {
  return N >= 1 && K >= 1 && (group == 32 || group == 64 || group == 128) && K % group == 0 && N < (1 << 30) &&
         K < (1 << 30);
}

}  // namespace
}  // namespace hb

using namespace hb;

extern "C" int hb_quant_w4(const void* w, int64_t ldw, int N, int K, int group, void* packed, void* scales,
                           cudaStream_t stream) {
  if (!w || !packed || !scales) return HB_ERR_NULL;
  if (!w4_shape_ok(N, K, group) || ldw < K) return HB_ERR_SHAPE;
  if (!aligned16(w) || !aligned16(packed) || !aligned16(scales) || ldw % 8) return HB_ERR_ALIGN;
  const int st = check_device();
  if (st != HB_OK) return st;
  const int tiles = (N + 15) / 16, kblocks = (K + 127) / 128;
  const int64_t grid = ((int64_t)tiles * 16 * kblocks * 16 + 255) / 256;
  if (grid >= (1ll << 31)) return HB_ERR_SHAPE;
  const uint16_t* wp = static_cast<const uint16_t*>(w);
  uint32_t* pp = static_cast<uint32_t*>(packed);
  uint16_t* sp = static_cast<uint16_t*>(scales);
  const unsigned g = static_cast<unsigned>(grid);
  if (group == 32) w4_quant_kernel<32><<<g, 256, 0, stream>>>(wp, ldw, N, K, tiles, kblocks, pp, sp);
  if (group == 64) w4_quant_kernel<64><<<g, 256, 0, stream>>>(wp, ldw, N, K, tiles, kblocks, pp, sp);
  if (group == 128) w4_quant_kernel<128><<<g, 256, 0, stream>>>(wp, ldw, N, K, tiles, kblocks, pp, sp);
  return cudaGetLastError() == cudaSuccess ? HB_OK : HB_ERR_LAUNCH;
}

extern "C" int hb_w4_linear(const HbW4Args* args, cudaStream_t stream) {
  if (!args) return HB_ERR_NULL;
  const HbW4Args& a = *args;
  if (!a.x || !a.packed || !a.scales || !a.y) return HB_ERR_NULL;
  if (!w4_shape_ok(a.N, a.K, a.group) || a.M < 1 || a.M > 32 * 65535 || a.ldx < a.K || a.ldy < a.N ||
      (a.dtype != HB_BF16 && a.dtype != HB_FP16) || (a.silu != 0 && a.silu != 1))
    return HB_ERR_SHAPE;
  if (!aligned16(a.x) || !aligned16(a.packed) || !aligned16(a.scales) || a.ldx % 8 ||
      (reinterpret_cast<uintptr_t>(a.y) & 1u) || (reinterpret_cast<uintptr_t>(a.bias) & 1u))
    return HB_ERR_ALIGN;
  const int st = check_device();
  if (st != HB_OK) return st;
  const W4Params p{static_cast<const uint16_t*>(a.x),
                   a.ldx,
                   static_cast<const uint4*>(a.packed),
                   static_cast<const uint16_t*>(a.scales),
                   static_cast<const uint16_t*>(a.bias),
                   static_cast<uint16_t*>(a.y),
                   a.ldy,
                   a.M,
                   a.N,
                   a.K,
                   (a.K + 127) / 128,
                   a.silu};
  return a.dtype == HB_FP16 ? launch_linear<true>(p, a.group, stream) : launch_linear<false>(p, a.group, stream);
}
