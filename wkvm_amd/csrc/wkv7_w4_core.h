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
  for (int i = 0; i < k && sum == sum; i += 8) {  // (NaN stays NaN)
    const int lane = (n & 15) + 16 * (i >> 3 & 3);
    const uint4 xv = *reinterpret_cast<const uint4*>(x + i);
    const uint32_t xw[4] = {xv.x, xv.y, xv.z, xv.w};
    const uint32_t w = G.w.codes[((tile * blocks + i / kW4K) * 64 + lane) * 4 + (i >> 5 & 3)];
    const uint32_t sc = G.w.scales[(tile * groups + i / group) * kW4N + (n & 15)];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      sum = fmaf(e % 2 ? bf16_hi(xw[e / 2]) : bf16_lo(xw[e / 2]),
                 w4_scale(sc) * float(w4_code(w, e) - w4_zero(sc)), sum);
  }
  if (G.bias) sum += bf16_to_f32(G.bias[n]);
  G.y[m * G.ldy + n] = f32_to_bf16(w4_activate(sum, G.act));
}

struct W4Args {
  wkv7_w4_group g[WKV7_PROJ_MAX_GROUPS];
  int32_t wg_end[WKV7_PROJ_MAX_GROUPS];  // exclusive prefix sums of workgroups
  int64_t m;
  int32_t ngroups;
};

// The product that workgroup `at` works on, its number there and how many others do.
__device__ __forceinline__ int w4_product(const W4Args& args, int at, int& first, int& count) {
  int g = 0;
  while (g + 1 < args.ngroups && at >= args.wg_end[g]) ++g;
  first = at - (g ? args.wg_end[g - 1] : 0);
  count = args.wg_end[g] - (g ? args.wg_end[g - 1] : 0);
  return g;
}

// Up to 16 rows: a workgroup walks column tiles of 16, the blocks of 128 inputs of each dealt to its NW
// waves, U of them to a wave at once, their sums joined in LDS. Everything comes from memory straight
// to registers: codes and scales of the next tile while this one is multiplied, x (and its sums over
// the groups of 32 KS inputs) once where a wave's blocks are the same for every tile. Bound by how many
// loads are under way: 65536 x 2048 at one row 15.3 us, 4.6 TB/s; below some 4 us it is latency.
template <int NW, int U, int KS>
__global__ __launch_bounds__(64 * NW, 4) void w4_thin_kernel(const W4Args args) {
  constexpr int NG = 4 / KS;  // groups of a block
  __shared__ w4_f32x4 red[2][NW][64];
  const int lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int first, count;
  const wkv7_w4_group& G = args.g[w4_product(args, blockIdx.x, first, count)];
  const int k = G.w.k, blocks = (k + kW4K - 1) / kW4K, groups = (k + 32 * KS - 1) / (32 * KS);
  const int tiles = (G.w.n + kW4N - 1) / kW4N;
  const int passes = (blocks + NW * U - 1) / (NW * U);
  const uint4* codes = reinterpret_cast<const uint4*>(G.w.codes) + lane;
  const uint32_t* scales = G.w.scales + li;
  const uint16_t* x = G.x + min(int64_t(li), args.m - 1) * G.ldx + 8 * lg;

  const W4Bits bits;
  const uint4 ones = make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u);
  uint4 xf[U][4];
  w4_f32x4 sums[U][NG];
  // What lies past k is read from inside it and multiplied by zeros. No load stands behind a branch, and
  // two passes' registers take turns: else the wait for one pass would be one for the next one's loads
  // too (65536 x 2048, one row: 17.2 us; 15.3 so, 4.6 TB/s, and 16.3 with three passes).
  struct Pass {
    uint4 c[U];
    uint32_t sc[U][NG];
  } even, odd;
  int next_tile = first, next_pass = 0;
  auto fetch = [&](Pass& p) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int b = min(wave + NW * (next_pass * U + u), blocks - 1);
      p.c[u] = codes[(int64_t(next_tile) * blocks + b) * 64];
#pragma unroll
      for (int q = 0; q < NG; ++q)
        p.sc[u][q] = scales[(int64_t(next_tile) * groups + min(b * NG + q, groups - 1)) * kW4N];
    }
    if (++next_pass == passes) {  // (behind the last tile it once more, unused)
      next_pass = 0;
      if (next_tile + count < tiles) next_tile += count;
    }
  };
  auto load_x = [&](int pass) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int at = kW4K * (wave + NW * (pass * U + u)) + 32 * j;
        xf[u][j] = *reinterpret_cast<const uint4*>(x + min(at, k - 32));
        if (at >= k || li >= args.m) xf[u][j] = make_uint4(0, 0, 0, 0);
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int q = 0; q < NG; ++q) {
        sums[u][q] = w4_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < KS; ++j) sums[u][q] = w4_mma(xf[u][q * KS + j], ones, sums[u][q]);
      }
  };
  auto join = [&](int tile, int turn) {
    w4_f32x4 v = red[turn & 1][0][lane];
#pragma unroll
    for (int w = 1; w < NW; ++w) v += red[turn & 1][w][lane];
    const int n = tile * kW4N + li;
    if (n >= G.w.n) return;
    const float bias = G.bias ? bf16_to_f32(G.bias[n]) : 0.f;
#pragma unroll 1
    for (int e = 0; e < 4; ++e) {
      const int m = 4 * lg + e;
      if (m >= args.m) break;
      const float r = fmaf(16.f, v[0], bias);
      v = w4_f32x4{v[1], v[2], v[3], 0.f};
      if (fabsf(r) < INFINITY) G.y[m * G.ldy + n] = f32_to_bf16(w4_activate(r, G.act));
      else w4_store_direct(G, m, n);
    }
  };
  int tile = first, pass = 0, turn = 0;
  w4_f32x4 total = {0.f, 0.f, 0.f, 0.f};
  // One pass over a tile; false behind the last.
  auto step = [&](const Pass& now, Pass& ahead) {
    if (passes > 1) load_x(pass);
    fetch(ahead);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t words[4] = {now.c[u].x, now.c[u].y, now.c[u].z, now.c[u].w};
#pragma unroll
      for (int q = 0; q < NG; ++q) {
        w4_f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < KS; ++j)
          acc = w4_mma(xf[u][q * KS + j], w4_expand(words[q * KS + j], bits), acc);
        const float s = w4_scale(now.sc[u][q]), z = w4_minus_zero(now.sc[u][q]);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          total[e] = fmaf(s, fmaf(z, sums[u][q][e], acc[e]), total[e]);
      }
    }
    if (++pass < passes) return true;
    red[turn & 1][wave][lane] = total;
    __syncthreads();
    if (wave == turn % NW) join(tile, turn);  // the waves take turns to join the sums
    total = w4_f32x4{0.f, 0.f, 0.f, 0.f};
    pass = 0;
    ++turn;
    tile += count;
    return tile < tiles;
  };
  fetch(even);
  if (passes == 1) load_x(0);
  while (step(even, odd) && step(odd, even)) {
  }
}

typedef float w4_f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ w4_f32x16 w4_mma32(const uint4& a, const uint4& b, w4_f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(w4_bf16x8, a),
                                                 __builtin_bit_cast(w4_bf16x8, b), c, 0, 0, 0);
}

constexpr int kW4Xcds = 8;  // workgroups are dealt round-robin over 8 XCDs

typedef __attribute__((address_space(3))) uint4 w4_lds_u4;

// Direct loads, lane l's 16 (4) bytes to lds + 16 l (4 l). The compiler does not see them: they are waited
// for by the waits and barriers written below alone.
__device__ __forceinline__ void w4_lds16(const void* src, uint32_t lds) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "{m0}"(lds), "v"(src) : "memory");
}
__device__ __forceinline__ void w4_lds4(const void* src, uint32_t lds) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dword %1, off" : : "{m0}"(lds), "v"(src) : "memory");
}

// Some tens of rows: a workgroup per tile of 32 rows by 32 TN columns, the blocks of 128 inputs dealt
// to its NW waves, on v_mfma_f32_32x32x16_bf16 (lane l, c = l % 32, h = l / 32: row or column c at 8 h ..
// of 16 inputs; result lane D[8 (i / 4) + 4 h + i % 4][c]). There is no barrier before the sums are
// joined: a wave's x goes through LDS of its own, whole rows by direct loads (rows read straight into
// operands, neighbouring lanes from different ones, pass the load unit at 16 bytes a cycle, not 64), its
// codes and scales to registers; those of its next block are under way while it multiplies one. Bound by
// the latency of a block's loads and by the vector work: 32 rows of 4096 in 11.8 us, three products of
// 4096 columns; of 2048 by 8192 11.5 (19.3 with x straight to registers).
template <int NW, int TN, int KS>
__global__ __launch_bounds__(64 * NW, 2) void w4_mid_kernel(const W4Args args, int row_tiles,
                                                            int span) {
  constexpr int NG = 4 / KS, XL = 8;  // direct loads of a block
  __shared__ uint4 xs[NW][2][32 * 16];  // rows of 16 chunks, chunk i of row r at i ^ (r % 16)
  const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int bid = int(blockIdx.x % kW4Xcds) * span + int(blockIdx.x / kW4Xcds);
  if (bid >= args.wg_end[args.ngroups - 1]) return;
  int at, count;
  const wkv7_w4_group& G = args.g[w4_product(args, bid, at, count)];
  const int64_t m0 = int64_t(at % row_tiles) * 32, M = args.m;
  const int n0 = at / row_tiles * (32 * TN);
  const int k = G.w.k, blocks = (k + kW4K - 1) / kW4K, groups = (k + 32 * KS - 1) / (32 * KS);
  const uint4* codes[TN];
  const uint32_t* scales[TN];
#pragma unroll
  for (int t = 0; t < TN; ++t) {
    const int64_t tile = min(n0 / kW4N + 2 * t + c / kW4N, (G.w.n + kW4N - 1) / kW4N - 1);
    codes[t] = reinterpret_cast<const uint4*>(G.w.codes) + tile * blocks * 64 + (c & 15) + 16 * h;
    scales[t] = G.w.scales + tile * groups * kW4N + (c & 15);
  }
  const uint16_t* xsrc[XL];
#pragma unroll
  for (int i = 0; i < XL; ++i)
    xsrc[i] = G.x + min(m0 + 4 * i + lane / 16, M - 1) * G.ldx + kW4K * wave;

  const W4Bits bits;
  const uint4 ones = make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u);
  w4_f32x16 total[TN] = {};
  struct Codes {
    uint4 w[TN][2];  // words j of inputs 32 j + 8 h .. and of 32 j + 16 + 8 h ..
    uint32_t sc[TN][NG];
  } even, odd;
  // (past k something inside it is read, and not used)
  auto fetch = [&](Codes& to, int b) {
#pragma unroll
    for (int t = 0; t < TN; ++t) {
      to.w[t][0] = codes[t][int64_t(b) * 64];
      to.w[t][1] = codes[t][int64_t(b) * 64 + 32];
#pragma unroll
      for (int q = 0; q < NG; ++q) to.sc[t][q] = scales[t][min(b * NG + q, groups - 1) * kW4N];
    }
  };
  auto issue = [&](int b, int slot) {
    const uint32_t to = uint32_t(reinterpret_cast<uintptr_t>((w4_lds_u4*)xs[wave][slot]));
#pragma unroll
    for (int i = 0; i < XL; ++i) {
      const int chunk = 8 * ((lane & 15) ^ ((4 * i + lane / 16) & 15));
      w4_lds16(xsrc[i] + min(chunk, k - 8 - kW4K * b), to + 1024 * i);
      xsrc[i] += NW * kW4K;
    }
  };
  // Block b; false behind the wave's last.
  auto step = [&](int& b, int slot, const Codes& now, Codes& next) {
    asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
    const bool more = b + NW < blocks;
    fetch(next, more ? b + NW : b);
    if (more) issue(b + NW, slot ^ 1);
    const uint4* st = xs[wave][slot] + c * 16;
#pragma unroll
    for (int q = 0; q < NG; ++q) {
      w4_f32x16 acc[TN] = {}, sum = {};
#pragma unroll
      for (int j = q * KS; j < (q + 1) * KS; ++j) {
        if (kW4K * b + 32 * j >= k) continue;  // (uniform)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint4 xf = st[(4 * j + 2 * u + h) ^ (c & 15)];
          sum = w4_mma32(xf, ones, sum);
#pragma unroll
          for (int t = 0; t < TN; ++t) {
            const uint4& w = now.w[t][u];
            acc[t] = w4_mma32(xf, w4_expand(j == 0 ? w.x : j == 1 ? w.y : j == 2 ? w.z : w.w, bits),
                              acc[t]);
          }
        }
      }
#pragma unroll
      for (int t = 0; t < TN; ++t) {
        const float s = w4_scale(now.sc[t][q]), z = w4_minus_zero(now.sc[t][q]);
#pragma unroll
        for (int e = 0; e < 16; ++e) total[t][e] = fmaf(s, fmaf(z, sum[e], acc[t][e]), total[t][e]);
      }
      if (NG > 1) __builtin_amdgcn_sched_barrier(0);  // (one group's sums at a time in registers)
    }
    b += NW;
    return more;
  };
  if (wave < blocks) {
    int b = wave;
    issue(b, 0);
    fetch(even, b);
    while (step(b, 0, even, odd) && step(b, 1, odd, even)) {
    }
  }
  float* red = reinterpret_cast<float*>(xs[wave]);
#pragma unroll
  for (int t = 0; t < TN; ++t)
#pragma unroll
    for (int e = 0; e < 16; ++e) red[(16 * t + e) * 64 + lane] = total[t][e];
  __syncthreads();
#pragma unroll 1
  for (int i = wave; i < 16 * TN; i += NW) {
    const int e = i & 15, n = n0 + 32 * (i >> 4) + c;
    const int64_t m = m0 + 8 * (e / 4) + 4 * h + e % 4;
    float v = reinterpret_cast<const float*>(xs[0])[i * 64 + lane];
#pragma unroll
    for (int w = 1; w < NW; ++w) v += reinterpret_cast<const float*>(xs[w])[i * 64 + lane];
    if (m >= M || n >= G.w.n) continue;
    const float r = fmaf(16.f, v, G.bias ? bf16_to_f32(G.bias[n]) : 0.f);
    if (fabsf(r) < INFINITY) G.y[m * G.ldy + n] = f32_to_bf16(w4_activate(r, G.act));
    else w4_store_direct(G, m, n);
  }
}

}  // namespace
}  // namespace wkv7
