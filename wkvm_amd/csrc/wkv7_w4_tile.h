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
//
// What bounds it (three products of 4096 x 4096 with 4096 rows, 64 x 256 tiles, 1.0 PFLOP/s): the
// clock, 1.92 GHz, with matrix and vector units busy for 55 and 58 % of the cycles; the direct
// loads, 1 KiB in 16 cycles of the unit's one load path, are a sixth of the time (left out of a copy; a
// tile of 128 x 256 loads fewer bytes, but its eight waves wait for one another: 443 us for 409). Few rows
// (256 rows, 64 x 128 tiles): matrix units busy for 25 % of the cycles; in copies with parts left out, a
// stage has some 440 cycles until its first operands are there, beside 530 of products.
#pragma once

#include <type_traits>

#include "wkv7_w4_core.h"

namespace wkv7 {
namespace {

struct W4TileArgs {
  wkv7_w4_group g[WKV7_PROJ_MAX_GROUPS];
  int32_t tile_end[WKV7_PROJ_MAX_GROUPS];  // exclusive prefix sums of work items
  // parts of X, [ceil(m / 32)][groups / 16][3][64][8]: lane c + 32 h of a part has row c at groups 8 h .. + 7
  const uint16_t* sums[WKV7_PROJ_MAX_GROUPS];
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

// Sums of x over its groups: a wave takes 512 inputs of a row, eight to a lane. (3 x 3,001 rows of 2048
// in 9 us, 4.1 TB/s. A product with ones in the tile kernel would be half as many matrix instructions
// again, shared among four waves a quarter of that.)
template <int KS>
__global__ __launch_bounds__(256) void w4_sums_kernel(const W4SumArgs a) {
  constexpr int kLanes = 4 * KS;  // lanes of a group
  const int g = blockIdx.y;
  const int lane = threadIdx.x & 63;
  const int k = a.k[g], padded = w4_padded_groups(k, 32 * KS);
  const int parts = (padded * 32 * KS + 511) / 512;  // waves of a row
  const int64_t item = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int64_t row = item / parts;
  if (row >= (a.m + 31) / 32 * 32) return;
  const int i0 = int(item % parts) * 512 + 8 * lane;
  float s = 0.f;
  if (i0 < k && row < a.m) {
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
  for (int i = 0; i < 3; ++i)
    a.sums[g][(((row / 32 * (padded / 16) + gi / 16) * 3 + i) * 64 + row % 32 + 32 * (gi / 8 % 2)) * 8 +
              gi % 8] = p[i];
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

template <int N>
__device__ __forceinline__ void w4_barrier() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(N) : "memory");
}

// Waves on a SIMD: two workgroups of 4 waves on a unit, or one of more.
constexpr int w4_waves_per_simd(int waves) { return waves <= 4 ? 2 : waves / 4; }

// KS: groups of 32 KS inputs; KH: parts of the waves that take blocks in turn, each with a ring of its
// own, and add up their sums at the end.
template <int GM, int GN, int TM, int TN, int KH, int S, int KS>
__global__ __launch_bounds__(64 * GM * GN * KH, w4_waves_per_simd(GM * GN * KH))
void w4_tile_kernel(const W4TileArgs args) {
  static_assert(KH == 1 || (KH == 2 && TM == 2), "parts");
  constexpr int NW = GM * GN, BM = 32 * TM * GM, BN = 32 * TN * GN;
  constexpr int NG = 4 / KS;                   // groups of a block
  // direct loads of a wave and stage: x rows, codes, scale words (where there are fewer than waves,
  // some twice)
  constexpr int XL = (BM / 4 + NW - 1) / NW, CL = (BN / 16 + NW - 1) / NW;
  constexpr int SL = (BN * NG / 64 + NW - 1) / NW, L = XL + CL + SL;
  static_assert(BN % 64 == 0, "tile shape");
  struct Stage {
    uint4 x[BM * 16];
    uint4 codes[BN * 4];
    uint32_t scales[NG * BN];
  };
  __shared__ Stage rings[KH][S];

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
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wave = wid % NW, kh = KH > 1 ? wid / NW : 0;
  const int wm = wave % GM, wn = wave / GM;
  Stage(&ring)[S] = rings[kh];
  const int mine = (blocks - kh + KH - 1) / KH;  // blocks kh, kh + KH, ..

  // Sources of the direct loads, moved on by a block at each issue. x: load i fills rows 4 (NW i + wave)
  // .. + 3 of a stage, lane l chunk l % 16 of row l / 16, which holds logical chunk (l % 16) ^
  // swizzle(row). Rows past m and columns past n load valid ones and are not stored.
  const uint16_t* xsrc[XL];
  int xk[XL];
#pragma unroll
  for (int i = 0; i < XL; ++i) {
    const int r = 4 * ((NW * i + wave) % (BM / 4)) + lane / 16;
    xk[i] = 8 * ((lane & 15) ^ (r & 15));
    xsrc[i] = G.x + min(m0 + r, M - 1) * G.ldx + xk[i] + kh * kW4K;
  }
  const uint4* csrc[CL];
#pragma unroll
  for (int i = 0; i < CL; ++i)
    csrc[i] = reinterpret_cast<const uint4*>(G.w.codes) +
              (int64_t(min(n0 / 16 + (NW * i + wave) % (BN / 16), ntiles - 1)) * blocks + kh) * 64 +
              lane;
  const uint32_t* ssrc[SL];
  int sgroup[SL];
#pragma unroll
  for (int i = 0; i < SL; ++i) {
    const int at = (NW * i + wave) * 64 % (NG * BN);
    sgroup[i] = at / BN + kh * NG;
    ssrc[i] = G.w.scales + (lane & 15) +
              (int64_t(min((n0 + at % BN) / 16 + lane / 16, ntiles - 1)) * groups + sgroup[i]) * kW4N;
  }
  // Load `part` of L of this part's block t.
  auto issue = [&](int t, int part) {
    Stage& st = ring[t % S];
    const uint32_t xl = uint32_t(reinterpret_cast<uintptr_t>((w4_lds_u4*)st.x));
    const uint32_t cl = uint32_t(reinterpret_cast<uintptr_t>((w4_lds_u4*)st.codes));
    if (part == 0 && KH * t + kh == K / kW4K) {
      // chunks past k read the row's last one, groups past the last that one
#pragma unroll
      for (int i = 0; i < XL; ++i) xsrc[i] += min(K - 8 - K / kW4K * kW4K - xk[i], 0);
#pragma unroll
      for (int i = 0; i < SL; ++i) ssrc[i] += min(groups - 1 - KH * NG * t - sgroup[i], 0) * kW4N;
    }
    if (part < XL) {
      w4_lds16(xsrc[part], xl + 1024 * ((NW * part + wave) % (BM / 4)));
      xsrc[part] += KH * kW4K;
    } else if (part < XL + CL) {
      const int i = part - XL;
      w4_lds16(csrc[i], cl + 1024 * ((NW * i + wave) % (BN / 16)));
      csrc[i] += KH * 64;
    } else {
      const int i = part - XL - CL;
      w4_lds4(ssrc[i], cl + BN * 64 + 4 * ((NW * i + wave) * 64 % (NG * BN)));
      ssrc[i] += KH * NG * kW4N;
    }
  };

#pragma unroll
  for (int s = 0; s < S - 1; ++s)
    if (s < mine)
#pragma unroll
      for (int p = 0; p < L; ++p) issue(s, p);

  // The zero points' part.
  w4_f32x16 total[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) total[i][j] = w4_f32x16{};
  {
    const int padded = w4_padded_groups(K, 32 * KS);
    for (int g0 = 16 * kh; g0 < padded; g0 += 16 * KH) {
      uint4 xs[TM][3], zs[TN][3];
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const int64_t tile = min(m0 / 32 + TM * wm + i, (M - 1) / 32);
#pragma unroll
        for (int p = 0; p < 3; ++p)
          xs[i][p] = *reinterpret_cast<const uint4*>(
              args.sums[g] + (((tile * (padded / 16) + g0 / 16) * 3 + p) * 64 + lane) * 8);
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
  w4_f32x16 acc[TM][TN];  // sums of the group at hand, and its scale
  float scale[TN];
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    scale[j] = 0.f;
#pragma unroll
    for (int i = 0; i < TM; ++i) acc[i][j] = w4_f32x16{};
  }
  auto flush = [&](int i, int j) {
#pragma unroll
    for (int e = 0; e < 16; ++e) total[i][j][e] = fmaf(scale[j], acc[i][j][e], total[i][j][e]);
  };
  // One stage; of one that is not whole `steps` times 32 inputs.
  auto stage = [&](int t, auto whole, auto more, int steps) {
    constexpr bool kWhole = decltype(whole)::value, kMore = decltype(more)::value;
    // stage t has landed, and every wave is done with stage t - 1, whose slot the next loads take
    if (kMore) w4_barrier<(S - 2) * L>();
    else w4_barrier<0>();
    const Stage& st = ring[t % S];
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
    // Steps of 16 inputs: the next one's operands are made while this one is multiplied (x read
    // further ahead was no faster, and a load each is issued there so that the waves do not wait for
    // the load unit one after the other). A group's sums get their scale where the next group begins.
    uint4 wf[2][TN], xf[2][TM];
    auto prepare = [&](int q) {
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const int r = 32 * (TM * wm + i) + c;
        uint4& x = xf[q & 1][i];
        x = st.x[r * 16 + ((2 * q + h) ^ (r & 15))];
        if (!kWhole) {
          const uint32_t keep = q < 2 * steps ? ~0u : 0u;
          x = make_uint4(x.x & keep, x.y & keep, x.z & keep, x.w & keep);
        }
      }
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const uint4& w4 = cw[j][q & 1];
        wf[q & 1][j] = w4_expand(q < 2 ? w4.x : q < 4 ? w4.y : q < 6 ? w4.z : w4.w, bits);
      }
    };
    prepare(0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      if (q < 7) prepare(q + 1);
      if (kMore) {
#pragma unroll
        for (int p = q * L / 8; p < (q + 1) * L / 8; ++p) issue(t + S - 1, p);
      }
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          if (q % (2 * KS) == 0) flush(i, j);
          acc[i][j] = w4_mma32(xf[q & 1][i], wf[q & 1][j],
                               q % (2 * KS) ? acc[i][j] : w4_f32x16{});
        }
      if (q % (2 * KS) == 0) {
#pragma unroll
        for (int j = 0; j < TN; ++j) scale[j] = sc[j][q / (2 * KS)];
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  const int whole = (K / kW4K - kh + KH - 1) / KH;
  int t = 0;
  for (; t + S - 1 < mine; ++t) stage(t, std::true_type{}, std::true_type{}, 4);
  for (; t < whole; ++t) stage(t, std::true_type{}, std::false_type{}, 4);
  if (t < mine) stage(t, std::false_type{}, std::false_type{}, K % kW4K / 32);
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) flush(i, j);

  // Each part gives the other one row tile's sums and finishes the other tile.
  constexpr int TO = TM / KH;  // row tiles of a wave to finish
  w4_f32x16 out[TO][TN];
  if constexpr (KH == 1) {
#pragma unroll
    for (int i = 0; i < TO; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) out[i][j] = total[i][j];
  } else {
    static_assert(sizeof(rings) >= 2 * NW * TN * 64 * sizeof(w4_f32x16), "room for the sums");
    float* sums = reinterpret_cast<float*>(&rings);
    if (mine < (blocks + KH - 1) / KH) w4_barrier<0>();  // (the other part's last block)
    w4_barrier<0>();
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        sums[((wid * TN + j) * 16 + e) * 64 + lane] = kh ? total[0][j][e] : total[1][j][e];
    w4_barrier<0>();
    const int other = kh ? wid - NW : wid + NW;
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        out[0][j][e] = (kh ? total[1][j][e] : total[0][j][e]) +
                       sums[((other * TN + j) * 16 + e) * 64 + lane];
  }
  // Outputs. (The branches stay outside the loops over the tiles: an output is a handful of
  // instructions, and a workgroup has them all at its end.)
  float wrong = 0.f;  // NaN as soon as one is not finite
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    const int n = n0 + 32 * (TN * wn + j) + c;
    const float bias = G.bias && n < N ? bf16_to_f32(G.bias[n]) : 0.f;
#pragma unroll
    for (int i = 0; i < TO; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float v = fmaf(16.f, out[i][j][e], bias);
        wrong = fmaf(v, 0.f, wrong);
        out[i][j][e] = v;
      }
  }
  uint32_t again[TO][TN] = {};
  if (__ballot(wrong != wrong)) {
#pragma unroll
    for (int i = 0; i < TO; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (!(fabsf(out[i][j][e]) < INFINITY)) again[i][j] |= 1u << e;
  }
  if (G.act != WKV7_ACT_NONE) {
#pragma unroll
    for (int i = 0; i < TO; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) w4_activate_all(out[i][j], G.act);
  }
  auto row_of = [&](int i, int e) { return 32 * (TM * wm + kh + i) + 8 * (e / 4) + 4 * h + e % 4; };
  const int64_t corner = m0 * G.ldy + n0 + c;
  if (m0 + BM <= M && n0 + BN <= N) {
#pragma unroll
    for (int i = 0; i < TO; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        uint16_t* y = G.y + corner + row_of(i, e) * G.ldy;
#pragma unroll
        for (int j = 0; j < TN; ++j) y[32 * (TN * wn + j)] = f32_to_bf16(out[i][j][e]);
      }
  } else {
#pragma unroll
    for (int i = 0; i < TO; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        if (m0 + row_of(i, e) >= M) continue;
        uint16_t* y = G.y + corner + row_of(i, e) * G.ldy;
#pragma unroll
        for (int j = 0; j < TN; ++j)
          if (n0 + 32 * (TN * wn + j) + c < N)
            y[32 * (TN * wn + j)] = f32_to_bf16(out[i][j][e]);
      }
  }
  // those that are not finite once more, as the formula is written
#pragma unroll
  for (int i = 0; i < TO; ++i)
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
