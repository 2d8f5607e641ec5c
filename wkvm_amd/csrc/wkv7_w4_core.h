// Device code of the products with 4-bit weights (wkv7_proj_w4).
//
// A code c is turned into the bf16 number 1 + c / 16 by putting its bits into the mantissa: a word
// of eight codes is laid out so that (w rotated by 4 p) & 0x00780078 | 0x3f803f80 is the p-th pair of
// them, an operand register of v_mfma_f32_16x16x32_bf16 (7 instructions for 8 codes, exact). With X the
// sum of x over a group, from the same instruction with ones for weights,
//   sum_k x_k s (c_k - z) = 16 s ( sum_k x_k (1 + c_k / 16) - (1 + z / 16) X )
// so scale and zero point come in once per group, on the fp32 sums.
#pragma once

#include "wkv7_common.h"

namespace wkv7 {
namespace {

typedef __bf16 w4_bf16x8 __attribute__((ext_vector_type(8)));
typedef float w4_f32x4 __attribute__((ext_vector_type(4)));

constexpr int kW4N = 16, kW4K = 128;  // a block of codes: 1 KiB

__device__ __forceinline__ w4_f32x4 w4_mma(const uint4& a, const uint4& b, w4_f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(w4_bf16x8, a),
                                                 __builtin_bit_cast(w4_bf16x8, b), c, 0, 0, 0);
}

// bit at which code e (0 .. 7) of a word starts
__host__ __device__ __forceinline__ int w4_bit(int e) { return (3 + 4 * (e >> 1) + 16 * (e & 1)) & 31; }
__device__ __forceinline__ uint32_t w4_rotr(uint32_t w, int by) {
  return by ? (w >> by) | (w << (32 - by)) : w;
}
__device__ __forceinline__ int w4_code(uint32_t w, int e) { return int(w4_rotr(w, w4_bit(e)) & 15u); }

// The constants of w4_expand in registers: as literals, of which an instruction holds one, each
// pair of codes would take an and and an or.
struct W4Bits {
  uint32_t mask, one;
  __device__ __forceinline__ W4Bits() {
    asm volatile("v_mov_b32 %0, 0x780078\n\tv_mov_b32 %1, 0x3f803f80" : "=&v"(mask), "=v"(one));
  }
};

// eight codes as the bf16 numbers 1 + c / 16
__device__ __forceinline__ uint4 w4_expand(uint32_t w, const W4Bits& k) {
  return make_uint4((w & k.mask) | k.one, ((w >> 4) & k.mask) | k.one, ((w >> 8) & k.mask) | k.one,
                    (__builtin_amdgcn_alignbit(w, w, 12) & k.mask) | k.one);
}

__device__ __forceinline__ float w4_scale(uint32_t word) { return __uint_as_float(word & ~15u); }
__device__ __forceinline__ int w4_zero(uint32_t word) { return int(word & 15u); }
// -(1 + z / 16)
__device__ __forceinline__ float w4_minus_zero(uint32_t word) {
  return __uint_as_float(0xbf800000u | (word << 19 & 0x00780000u));
}

__device__ __forceinline__ float w4_activate(float v, int act) {
  if (act == WKV7_ACT_TANH) return tanhf(v);
  if (act == WKV7_ACT_SIGMOID) return 1.f / (1.f + __expf(-v));
  return v;
}

// One output as the formula is written: for a result that is not finite. (With an infinite x the sums
// above are infinity less infinity, whatever the weights.)
__device__ __forceinline__ void w4_store_direct(const wkv7_w4_group& G, int64_t m, int n) {
  const int k = G.w.k, group = G.w.group;
  const int blocks = (k + kW4K - 1) / kW4K, groups = (k + group - 1) / group;
  const int64_t tile = n / kW4N;
  const uint16_t* x = G.x + m * G.ldx;
  float sum = 0.f;
#pragma unroll 1
  for (int i = 0; i < k; ++i) {
    const int lane = (n & 15) + 16 * (i >> 3 & 3);
    const uint32_t w = G.w.codes[((tile * blocks + i / kW4K) * 64 + lane) * 4 + (i >> 5 & 3)];
    const uint32_t sc = G.w.scales[(tile * groups + i / group) * kW4N + (n & 15)];
    sum = fmaf(bf16_to_f32(x[i]), w4_scale(sc) * float(w4_code(w, i & 7) - w4_zero(sc)), sum);
  }
  if (G.bias) sum += bf16_to_f32(G.bias[n]);
  G.y[m * G.ldy + n] = f32_to_bf16(w4_activate(sum, G.act));
}

struct W4Args {
  wkv7_w4_group g[WKV7_PROJ_MAX_GROUPS];
  int32_t tile_end[WKV7_PROJ_MAX_GROUPS];  // exclusive prefix sums of column tiles
  int64_t m;
  int32_t ngroups;
};

// 16 TM rows by 16 columns: the blocks of 128 inputs are dealt to the NW waves, their sums joined in
// LDS. Operands come from memory straight to registers.
template <int NW, int TM>
__global__ __launch_bounds__(64 * NW) void w4_thin_kernel(const W4Args args) {
  __shared__ w4_f32x4 red[NW][TM][64];
  const int lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int g = 0;
  while (g + 1 < args.ngroups && int(blockIdx.x) >= args.tile_end[g]) ++g;
  const wkv7_w4_group& G = args.g[g];
  const int64_t tile = int(blockIdx.x) - (g ? args.tile_end[g - 1] : 0);
  const int64_t m0 = int64_t(blockIdx.y) * (16 * TM);
  const int k = G.w.k, blocks = (k + kW4K - 1) / kW4K, groups = (k + G.w.group - 1) / G.w.group;
  const int steps = G.w.group / 32;  // of 32 inputs in a group: 1, 2 or 4
  const uint4* codes = reinterpret_cast<const uint4*>(G.w.codes) + tile * blocks * 64 + lane;
  const uint32_t* scales = G.w.scales + tile * groups * kW4N + li;
  const uint16_t* x[TM];
#pragma unroll
  for (int i = 0; i < TM; ++i) x[i] = G.x + min(m0 + 16 * i + li, args.m - 1) * G.ldx + 8 * lg;

  const W4Bits bits;
  const uint4 ones = make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u);
  w4_f32x4 total[TM], acc[TM], sum[TM];
#pragma unroll
  for (int i = 0; i < TM; ++i) total[i] = acc[i] = sum[i] = w4_f32x4{0.f, 0.f, 0.f, 0.f};
  for (int b = wave; b < blocks; b += NW) {
    const uint4 c = codes[int64_t(b) * 64];
    const uint32_t words[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int step = 4 * b + j;
      if (32 * step >= k) break;  // (uniform)
      const uint4 w = w4_expand(words[j], bits);
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const uint4 xf = *reinterpret_cast<const uint4*>(x[i] + 32 * step);
        acc[i] = w4_mma(xf, w, acc[i]);
        sum[i] = w4_mma(xf, ones, sum[i]);
      }
      if ((j + 1) % steps && 32 * (step + 1) < k) continue;  // (uniform) inside a group
      const uint32_t word = scales[step / steps * kW4N];
      const float s = w4_scale(word), z = w4_minus_zero(word);
#pragma unroll
      for (int i = 0; i < TM; ++i) {
#pragma unroll
        for (int e = 0; e < 4; ++e) total[i][e] = fmaf(s, fmaf(z, sum[i][e], acc[i][e]), total[i][e]);
        acc[i] = sum[i] = w4_f32x4{0.f, 0.f, 0.f, 0.f};
      }
    }
  }
#pragma unroll
  for (int i = 0; i < TM; ++i) red[wave][i][lane] = total[i];
  __syncthreads();
  const int n = int(tile) * kW4N + li;
  for (int i = wave; i < TM; i += NW) {
    w4_f32x4 v = red[0][i][lane];
#pragma unroll
    for (int w = 1; w < NW; ++w) v += red[w][i][lane];
    const float bias = G.bias && n < G.w.n ? bf16_to_f32(G.bias[n]) : 0.f;
    uint32_t again = 0;  // results that are not finite
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int64_t m = m0 + 16 * i + 4 * lg + e;
      if (m >= args.m || n >= G.w.n) continue;
      const float r = 16.f * v[e];
      G.y[m * G.ldy + n] = f32_to_bf16(w4_activate(r + bias, G.act));
      if (!(fabsf(r) < INFINITY)) again |= 1u << e;
    }
    for (; again; again &= again - 1)
      w4_store_direct(G, m0 + 16 * i + 4 * lg + __builtin_ctz(again), n);
  }
}

}  // namespace
}  // namespace wkv7
