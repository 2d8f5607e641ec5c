// Products with 4-bit weights for more rows than one tile (wkv7_proj_w4): output tiles on
// v_mfma_f32_32x32x16_bf16.
//
// Lane l, c = l % 32, h = l / 32, of that instruction holds row or column c at 8 h .. 8 h + 7 of 16
// inputs, its result lane D[8 (i / 4) + 4 h + i % 4][c]. A workgroup of GM x GN waves has a tile of
// 32 TM GM rows by 32 TN GN columns and walks k in blocks of 128, each of them a stage of an LDS ring
// that direct loads fill S - 1 stages ahead: x rows (256 bytes, 16-byte chunks swizzled by row), codes
// and scale words as they lie in memory. Codes become operands in registers (wkv7_w4_core.h), once per
// wave and column; a group's sum gets its scale by 16 fused multiply-adds per tile. The zero points'
// part, sum over groups of -s (1 + z / 16) X with X the sums of x, is a product of its own with one
// input per group, in front: X comes from w4_sums_kernel, both factors as three bf16 parts.
#pragma once

#include <type_traits>

#include "wkv7_w4_core.h"

namespace wkv7 {
namespace {

typedef __attribute__((address_space(3))) uint4 w4_lds_u4;

struct W4TileArgs {
  wkv7_w4_group g[WKV7_PROJ_MAX_GROUPS];
  int32_t tile_end[WKV7_PROJ_MAX_GROUPS];  // exclusive prefix sums of work items
  const uint16_t* sums[WKV7_PROJ_MAX_GROUPS];  // [m][3][groups, a multiple of 16] parts of X
  int64_t m;
  int32_t ngroups;
  int32_t span;  // work items per XCD
};

struct W4SumArgs {
  const uint16_t* x[WKV7_PROJ_MAX_GROUPS];
  uint16_t* sums[WKV7_PROJ_MAX_GROUPS];
  int64_t ldx[WKV7_PROJ_MAX_GROUPS];
  int32_t k[WKV7_PROJ_MAX_GROUPS];
  int64_t m;
};

__host__ __device__ constexpr int w4_padded_groups(int k, int group) {
  return ((k + group - 1) / group + 15) / 16 * 16;
}

__device__ __forceinline__ void w4_split3(float v, uint16_t (&p)[3]) {
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    p[i] = f32_to_bf16(v);
    v -= bf16_to_f32(p[i]);
  }
}

// Sums of x over its groups: a wave takes 512 inputs of a row, eight to a lane.
template <int KS>
__global__ __launch_bounds__(256) void w4_sums_kernel(const W4SumArgs a) {
  constexpr int kLanes = 4 * KS;  // lanes of a group
  const int g = blockIdx.y;
  const int lane = threadIdx.x & 63;
  const int k = a.k[g], padded = w4_padded_groups(k, 32 * KS);
  const int parts = (padded * 32 * KS + 511) / 512;  // waves of a row
  const int64_t item = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int64_t row = item / parts;
  if (row >= a.m) return;
  const int i0 = int(item % parts) * 512 + 8 * lane;
  float s = 0.f;
  if (i0 < k) {
    const uint4 v = *reinterpret_cast<const uint4*>(a.x[g] + row * a.ldx[g] + i0);
    s = ((bf16_lo(v.x) + bf16_hi(v.x)) + (bf16_lo(v.y) + bf16_hi(v.y))) +
        ((bf16_lo(v.z) + bf16_hi(v.z)) + (bf16_lo(v.w) + bf16_hi(v.w)));
  }
#pragma unroll
  for (int d = 1; d < kLanes; d *= 2) s += __shfl_xor(s, d);
  const int gi = i0 / (32 * KS);
  if (lane % kLanes || gi >= padded) return;
  uint16_t p[3];
  w4_split3(s, p);
#pragma unroll
  for (int i = 0; i < 3; ++i) a.sums[g][(row * 3 + i) * padded + gi] = p[i];
}

__device__ __forceinline__ void w4_activate_all(w4_f32x16& v, int act) {
  if (act == WKV7_ACT_TANH) {
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = w4_activate(v[e], WKV7_ACT_TANH);
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = w4_activate(v[e], WKV7_ACT_SIGMOID);
  }
}

// Direct loads, lane l's 16 (4) bytes to lds + 16 l (4 l); waited for by w4_barrier alone.
__device__ __forceinline__ void w4_lds16(const void* src, uint32_t lds) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "{m0}"(lds), "v"(src) : "memory");
}
__device__ __forceinline__ void w4_lds4(const void* src, uint32_t lds) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dword %1, off" : : "{m0}"(lds), "v"(src) : "memory");
}
template <int N>
__device__ __forceinline__ void w4_barrier() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(N) : "memory");
}

// KS: groups of 32 KS inputs.
template <int GM, int GN, int TM, int TN, int S, int KS>
__global__ __launch_bounds__(64 * GM * GN, 2) void w4_tile_kernel(const W4TileArgs args) {
  constexpr int NW = GM * GN, BM = 32 * TM * GM, BN = 32 * TN * GN;
  constexpr int NG = 4 / KS;                   // groups of a block
  constexpr int XL = BM * 256 / 1024 / NW;     // direct loads of a wave and stage: x rows,
  constexpr int CL = BN / 16 / NW;             // codes,
  constexpr int SL = (BN * NG + 64 * NW - 1) / (64 * NW);  // scale words
  constexpr int L = XL + CL + SL;
  static_assert(BM % (4 * NW) == 0 && BN % (16 * NW) == 0 && BN % 64 == 0, "tile shape");
  struct Stage {
    uint4 x[BM * 16];
    uint4 codes[BN * 4];
    uint32_t scales[NG * BN];
  };
  __shared__ Stage ring[S];

  const int bid = int(blockIdx.x % kW4Xcds) * args.span + int(blockIdx.x / kW4Xcds);
  int g = 0;
  while (g + 1 < args.ngroups && bid >= args.tile_end[g]) ++g;
  if (bid >= args.tile_end[g]) return;
  const wkv7_w4_group& G = args.g[g];
  const int item = bid - (g ? args.tile_end[g - 1] : 0);
  const int N = G.w.n, K = G.w.k;
  const int tiles_n = (N + BN - 1) / BN;
  const int64_t m0 = int64_t(item / tiles_n) * BM, M = args.m;
  const int n0 = item % tiles_n * BN;
  const int blocks = (K + kW4K - 1) / kW4K, groups = (K + 32 * KS - 1) / (32 * KS);
  const int ntiles = (N + 15) / 16;

  const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % GM, wn = wave / GM;

  // Sources of the direct loads. x: load i fills rows 4 (NW i + wave) .. + 3 of a stage, lane l chunk
  // l % 16 of row l / 16, which holds logical chunk (l % 16) ^ swizzle(row). Rows past m and columns past
  // n load valid ones and are not stored.
  const uint16_t* xsrc[XL];
  int xk[XL];
#pragma unroll
  for (int i = 0; i < XL; ++i) {
    const int r = 4 * (NW * i + wave) + lane / 16;
    xk[i] = 8 * ((lane & 15) ^ (r & 15));
    xsrc[i] = G.x + min(m0 + r, M - 1) * G.ldx;
  }
  auto issue = [&](int kb, int slot) {
    Stage& st = ring[slot];
    const uint32_t xl = uint32_t(reinterpret_cast<uintptr_t>((w4_lds_u4*)st.x));
    const uint32_t cl = uint32_t(reinterpret_cast<uintptr_t>((w4_lds_u4*)st.codes));
#pragma unroll
    for (int i = 0; i < XL; ++i)  // (chunks past k read the row's last one again)
      w4_lds16(xsrc[i] + min(kb * kW4K + xk[i], K - 8), xl + 1024 * (NW * i + wave));
#pragma unroll
    for (int i = 0; i < CL; ++i) {
      const int t = NW * i + wave;
      const int64_t tile = min(n0 / 16 + t, ntiles - 1);
      w4_lds16(reinterpret_cast<const uint4*>(G.w.codes) + (tile * blocks + kb) * 64 + lane,
               cl + 1024 * t);
    }
#pragma unroll
    for (int i = 0; i < SL; ++i) {  // (where there are fewer words than lanes, some twice)
      const int at = (NW * i + wave) * 64 % (NG * BN);
      const int gi = min(kb * NG + at / BN, groups - 1);
      const int64_t tile = min((n0 + at % BN) / 16 + lane / 16, ntiles - 1);
      w4_lds4(G.w.scales + (tile * groups + gi) * kW4N + (lane & 15),
              cl + BN * 64 + 4 * at);
    }
  };

#pragma unroll
  for (int s = 0; s < S - 1; ++s)
    if (s < blocks) issue(s, s);

  // The zero points' part.
  w4_f32x16 total[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) total[i][j] = w4_f32x16{};
  {
    const int padded = w4_padded_groups(K, 32 * KS);
    for (int g0 = 0; g0 < padded; g0 += 16) {
      uint4 xs[TM][3], zs[TN][3];
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const int64_t r = min(m0 + 32 * (TM * wm + i) + c, M - 1);
#pragma unroll
        for (int p = 0; p < 3; ++p)
          xs[i][p] = *reinterpret_cast<const uint4*>(args.sums[g] + (r * 3 + p) * padded + g0 + 8 * h);
      }
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int64_t tile = min((n0 + 32 * (TN * wn + j)) / 16 + c / 16, ntiles - 1);
        uint16_t parts[8][3];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int gi = g0 + 8 * h + e;
          const uint32_t word = gi < groups ? G.w.scales[(tile * groups + gi) * kW4N + (c & 15)] : 0u;
          w4_split3(w4_scale(word) * w4_minus_zero(word), parts[e]);
        }
#pragma unroll
        for (int p = 0; p < 3; ++p)
          zs[j][p] = make_uint4(parts[0][p] | uint32_t(parts[1][p]) << 16,
                                parts[2][p] | uint32_t(parts[3][p]) << 16,
                                parts[4][p] | uint32_t(parts[5][p]) << 16,
                                parts[6][p] | uint32_t(parts[7][p]) << 16);
      }
#pragma unroll
      for (int sum = 2; sum >= 0; --sum)  // the small products first
#pragma unroll
        for (int p = 0; p <= sum; ++p)
#pragma unroll
          for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j)
              total[i][j] = w4_mma32(xs[i][p], zs[j][sum - p], total[i][j]);
    }
  }

  const W4Bits bits;
  // One stage, `steps` (at most 4) times 32 inputs of it.
  auto stage = [&](int kb, auto whole, int steps) {
    constexpr bool kWhole = decltype(whole)::value;
    // stage kb has landed, and every wave is done with stage kb - 1, whose slot the next loads take
    if (kb + S - 2 < blocks) w4_barrier<(S - 2) * L>();
    else w4_barrier<0>();
    if (kb + S - 1 < blocks) issue(kb + S - 1, (kb + S - 1) % S);
    const Stage& st = ring[kb % S];
    uint4 cw[TN][2];  // words j of inputs 32 j + 8 h .. and 32 j + 16 + 8 h ..
    float sc[TN][NG];
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int col = 32 * (TN * wn + j) + c;
      cw[j][0] = st.codes[(col / 16) * 64 + (col & 15) + 16 * h];
      cw[j][1] = st.codes[(col / 16) * 64 + (col & 15) + 16 * (2 + h)];
#pragma unroll
      for (int q = 0; q < NG; ++q) sc[j][q] = w4_scale(st.scales[q * BN + col]);
    }
    uint4 wf[TN][8];  // the operands of 16 inputs each
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const uint4& w4 = cw[j][q & 1];
        wf[j][q] = w4_expand(q < 2 ? w4.x : q < 4 ? w4.y : q < 6 ? w4.z : w4.w, bits);
      }
    // Row tile by row tile and group by group; a group's sums get their scale behind the first
    // products of the next one.
    w4_f32x16 acc[2][TN];
    constexpr int kRuns = TM * NG;
    auto flush = [&](int run) {
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          total[run / NG][j][e] =
              fmaf(sc[j][run % NG], acc[run & 1][j][e], total[run / NG][j][e]);
    };
#pragma unroll
    for (int run = 0; run < kRuns; ++run) {
      const int i = run / NG, first = run % NG * 2 * KS;  // steps of 16 inputs
      const int r = 32 * (TM * wm + i) + c;
#pragma unroll
      for (int q = 0; q < 2 * KS; ++q) {
        if (!kWhole && first + q >= 2 * steps) continue;  // (uniform)
        const uint4 xf = st.x[r * 16 + ((2 * (first + q) + h) ^ (r & 15))];
#pragma unroll
        for (int j = 0; j < TN; ++j)
          acc[run & 1][j] = w4_mma32(xf, wf[j][first + q], q ? acc[run & 1][j] : w4_f32x16{});
        if (kWhole && q == 0 && run) flush(run - 1);
      }
      if (!kWhole && first < 2 * steps) flush(run);
    }
    if (kWhole) flush(kRuns - 1);
  };
  for (int kb = 0; kb < K / kW4K; ++kb) stage(kb, std::true_type{}, 4);
  if (K % kW4K) stage(K / kW4K, std::false_type{}, K % kW4K / 32);

  // Outputs. (The branches stay outside the loops over the tiles: an output is a handful of
  // instructions, and a workgroup has them all at its end.)
  float wrong = 0.f;  // NaN as soon as one is not finite
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    const int n = n0 + 32 * (TN * wn + j) + c;
    const float bias = G.bias && n < N ? bf16_to_f32(G.bias[n]) : 0.f;
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float v = fmaf(16.f, total[i][j][e], bias);
        wrong = fmaf(v, 0.f, wrong);
        total[i][j][e] = v;
      }
  }
  uint32_t again[TM][TN] = {};
  if (__ballot(wrong != wrong)) {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (!(fabsf(total[i][j][e]) < INFINITY)) again[i][j] |= 1u << e;
  }
  if (G.act != WKV7_ACT_NONE) {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) w4_activate_all(total[i][j], G.act);
  }
  auto row_of = [&](int i, int e) { return 32 * (TM * wm + i) + 8 * (e / 4) + 4 * h + e % 4; };
  const int64_t mine = m0 * G.ldy + n0 + c;
  if (m0 + BM <= M && n0 + BN <= N) {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        uint16_t* y = G.y + mine + row_of(i, e) * G.ldy;
#pragma unroll
        for (int j = 0; j < TN; ++j) y[32 * (TN * wn + j)] = f32_to_bf16(total[i][j][e]);
      }
  } else {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        if (m0 + row_of(i, e) >= M) continue;
        uint16_t* y = G.y + mine + row_of(i, e) * G.ldy;
#pragma unroll
        for (int j = 0; j < TN; ++j)
          if (n0 + 32 * (TN * wn + j) + c < N)
            y[32 * (TN * wn + j)] = f32_to_bf16(total[i][j][e]);
      }
  }
  // those that are not finite once more, as the formula is written
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
      for (; again[i][j]; again[i][j] &= again[i][j] - 1) {
        const int64_t m = m0 + row_of(i, __builtin_ctz(again[i][j]));
        const int n = n0 + 32 * (TN * wn + j) + c;
        if (m < M && n < N) w4_store_direct(G, m, n);
      }
}

}  // namespace
}  // namespace wkv7
