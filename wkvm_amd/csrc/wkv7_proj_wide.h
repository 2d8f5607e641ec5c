// The projection kernel for many rows (prompts): 128 or 256 x 256 tiles, 4 waves.
//
// Wave tile 32 TM x 128 (2 x 2 waves) on v_mfma_f32_32x32x16_bf16 with w as the first operand.
// Operand layout (lane l): A holds A[l % 32][8 (l / 32) .. + 7], B the same of its columns, the
// accumulator D[8 (e / 4) + 4 (l / 32) + e % 4][l % 32] in element e: columns of y in runs of 4
// for one row of it. k advances in stages of 64 through two LDS slots filled by direct loads, and
// each stage in four steps of 16. While a step is multiplied, the operands of the next are read
// from LDS between its MFMAs; in the last step of a stage and the first of the next one, the loads
// of the stage after it are issued into the slot that was read last before the barrier between
// them. So the matrix cores always have operands in registers, a load has two to three steps'
// time to arrive, and each operand byte is read from LDS twice per tile.
//
// 32,768 rows of a 2048 x 2048 product 0.85 PFLOP/s (three with adapters of 32 ranks 0.90), k of 4096
// 0.99, 8192^3 1.17: 0.66 to 0.79 of what the vendor's library reaches at these sizes. The loop
// alone is at 1.69 PFLOP/s where nothing is loaded, 1.62 with every load a hit in the unit's
// cache, 1.35 in the XCD's; with the real rows about 1.10, so what bounds it is x's lines on their
// way to the unit, and about 15 us per round of tiles for first loads and results. No gain:
// prefetches into the XCD's cache, k started at another stage in every tile, waves set apart in
// time, 1 to 16 row tiles side by side, three to five slots, eight waves.
#pragma once

#include "wkv7_proj_core.h"

namespace wkv7 {
namespace {

constexpr int kWideN = 256, kWideWaves = 4;
constexpr int kRowGroup = 4;  // row tiles that an XCD works on side by side

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) u32x4 lds_u32x4;

__device__ __forceinline__ f32x16 mma16(const uint4& a, const uint4& b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                 __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// load_lds16 from a wave-uniform address and a lane's byte offset.
__device__ __forceinline__ void load_lds16_from(const char* base, uint32_t off, uint32_t lds_base) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               :
               : "{m0}"(lds_base), "v"(off), "s"(base)
               : "memory");
}

// 16 bytes at an LDS byte address.
__device__ __forceinline__ uint4 lds_read(uint32_t at, uint32_t offset) {
  return __builtin_bit_cast(uint4, *(const lds_u32x4*)(uintptr_t(at + offset)));
}

__device__ __forceinline__ void lds_write(uint32_t at, uint32_t offset, f32x4 v) {
  *(lds_u32x4*)(uintptr_t(at + offset)) = __builtin_bit_cast(u32x4, v);
}

// tanh to 2^-18 of its value, in few instructions (it is inlined for every output of a lane):
// (1 - t) / (1 + t) with t = exp(-2 |x|) to 1.5 ulp, and x - x^3 / 3 where 1 - t would be below
// 0.03 and its error of 1.5 x 2^-24 above that bound.
__device__ __forceinline__ float wide_tanh(float x) {
  const float t = __expf(-2.f * fabsf(x));
  const float big = copysignf((1.f - t) / (1.f + t), x);
  return fabsf(x) < 0.015625f ? x - x * x * x * 0.33333334f : big;
}

// Adds the low-rank terms of 32 TM positions from p0 and 32 TN columns from n0 to acc. In a plan of
// many rows the runs of an adapter start at multiples of 32 positions, so that a tile is one
// adapter's; a slab of 16 ranks is one MFMA per part of h.
template <int TM, int TN>
__device__ __forceinline__ void expand_wide(const Adapters& ad, int g, int64_t p0, int64_t M, int n0,
                                            int N, f32x16 (&acc)[TM][TN]) {
  if (!ad.b[g]) return;
  const int lane = threadIdx.x & 63, li = lane & 31, lh = lane >> 5;
  const int slabs = ad.slabs[g];
  int id[TM], ns[TM], most = 0;
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    id[i] = p0 + 32 * i < M ? ad.id[p0 + 32 * i] : -1;
    ns[i] = id[i] >= 0 && id[i] < ad.count[g] ? min((ad.rank[g][id[i]] + 15) >> 4, slabs) : 0;
    most = max(most, ns[i]);
  }
  const uint16_t* hp = ad.h[g] + ((p0 + li) * slabs) * 48 + 8 * lh;
  for (int s = 0; s < most; ++s) {
    uint4 hf[TM][3], bf[TN];
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      if (s >= ns[i]) continue;
      const uint16_t* p = hp + (int64_t(32 * i) * slabs + s) * 48;
#pragma unroll
      for (int q = 0; q < 3; ++q) hf[i][q] = *reinterpret_cast<const uint4*>(p + 16 * q);
    }
    int held = -1;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      if (s >= ns[i]) continue;
      if (id[i] != held) {
        held = id[i];
        const uint16_t* bp = ad.b[g] + ((int64_t(held) * slabs + s) * N) * 16 + 8 * lh;
#pragma unroll
        for (int j = 0; j < TN; ++j)
          bf[j] = *reinterpret_cast<const uint4*>(bp + int64_t(min(n0 + 32 * j + li, N - 1)) * 16);
      }
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int q = 2; q >= 0; --q) acc[i][j] = mma16(bf[j], hf[i][q], acc[i][j]);
    }
  }
}

template <int TM, class Extra>
__global__ __launch_bounds__(64 * kWideWaves) void proj_wide_kernel(const ProjArgs args,
                                                                    const Extra ex) {
  constexpr int BM = 64 * TM, BN = kWideN;
  constexpr int TN = 4, WM = 32 * TM, WN = 128;
  constexpr int kRows = BM + BN;                 // of a stage: x rows, then w rows
  constexpr int LR = kRows / (8 * kWideWaves);   // a wave's direct loads per stage
  constexpr int LX = BM / (8 * kWideWaves);      // of them of x
  constexpr int LE = LR / 2;                     // of them issued early
  constexpr uint32_t kSlot = kRows * 128;        // bytes of a stage
  constexpr uint32_t kOut = 64 * WN * 4;         // bytes of a wave's results on their way out
  __shared__ uint4 ring[(2 * kSlot > kWideWaves * kOut ? 2 * kSlot : kWideWaves * kOut) / 16];

  // Tiles go to the XCDs in contiguous runs, ordered by product, then by groups of kRowGroup row
  // tiles, then by columns: what an XCD works on at one time re-reads few rows of x and of w.
  const int bid = int(blockIdx.x % kXcds) * args.xcd_span + int(blockIdx.x / kXcds);
  int g = 0;
  while (g + 1 < args.ngroups && bid >= args.tile_end[g]) ++g;
  if (bid >= args.tile_end[g]) return;
  const wkv7_proj_group& G = args.g[g];
  const int item = bid - (g ? args.tile_end[g - 1] : 0);
  const int N = G.n, K = G.k;
  const int tiles_n = (N + BN - 1) / BN;
  const int group = item / (kRowGroup * tiles_n), inside = item - group * kRowGroup * tiles_n;
  const int high = min(kRowGroup, args.tiles_m - group * kRowGroup);
  const int tm = group * kRowGroup + inside % high, tn = inside / high;
  const int64_t M = args.m;
  const int64_t m0 = int64_t(tm) * BM;
  const int n0 = tn * BN;
  if (ex.empty(m0)) return;

  const int t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int wm = wave & 1, wn = wave >> 1;
  const int li = lane & 31, lh = lane >> 5;

  // A stage's rows are 128 bytes (whole cache lines of x and w), chunk c of row r at
  // c ^ (r / 2 % 8): 16 neighbouring rows of an operand read touch all 64 banks once. Load i of a wave fills rows
  // 8 (4 i + wave) .. + 7. Row addresses are 32-bit byte offsets from x and w (the launch sees to
  // it that they fit).
  const int chunk = (lane & 7) ^ ((4 * wave + (lane >> 4)) & 7);
  uint32_t off[LR];
#pragma unroll
  for (int i = 0; i < LR; ++i) {
    const int row = 8 * (kWideWaves * i + wave) + lane / 8;
    const int64_t r = i < LX ? ex.row(min(m0 + row, M - 1)) * G.ldx
                             : int64_t(min(n0 + row - BM, N - 1)) * G.ldw;
    off[i] = uint32_t((r + 8 * chunk) * 2);
  }
  const int nk = K / 64;
  const char* const xb = reinterpret_cast<const char*>(G.x);
  const char* const wb = reinterpret_cast<const char*>(G.w);
  const uint32_t ring_base = lds_addr(ring);
  // Load i of the stage at byte k of the rows, into the slot at `to` (this wave's part of it).
  auto load = [&](uint32_t k, uint32_t to, int i) {
    load_lds16_from((i < LX ? xb : wb) + k, off[i], to + 1024u * kWideWaves * i);
  };
  // (what is loaded ahead of the end, and not used, is the last stage again)
  auto stage_k = [&](int kt) { return uint32_t(min(kt, nk - 1)) * 128; };

  f32x16 acc[TM][TN] = {};
  // Operands of a step: two sets of w tiles; of the x tiles one set, which the next step's reads
  // refill as its tiles are done with, and a second of the last one, so that no read is the last
  // thing before a barrier.
  uint4 wf[2][TN], xf[TM - 1], xl[2];
  uint32_t x_at[4], w_at[4];  // of the four steps, in the slot that is read
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const uint32_t in_tile = 128 * li + 16 * ((2 * s + lh) ^ ((li >> 1) & 7));
    x_at[s] = ring_base + 128 * (wm * WM) + in_tile;
    w_at[s] = ring_base + 128 * (BM + wn * WN) + in_tile;
  }
  auto read_w = [&](auto s_c, int i) {
    constexpr int s = decltype(s_c)::value;
    wf[s & 1][i] = lds_read(w_at[s], 4096 * i);
  };
  auto read_x = [&](auto s_c, int i) {
    constexpr int s = decltype(s_c)::value;
    const uint4 v = lds_read(x_at[s], 4096 * i);
    if (i < TM - 1) xf[i] = v;
    else xl[s & 1] = v;
  };
  // Multiplies step s of a stage with the reads of step r and the loads [l0, l1) of the stage at
  // byte k, to the slot at `to`, placed between the MFMAs. Between two MFMAs a wave issues
  // only a handful of instructions, so addresses are kept ready: the operands' are advanced once
  // per stage (through an asm, lest the compiler add the slot to each of them at every read).
  auto multiply = [&](auto s_c, auto r_c, auto l0, auto l1, uint32_t k, uint32_t to) {
    constexpr int s = decltype(s_c)::value & 1;
    constexpr int kFrom = decltype(l0)::value, kLoads = decltype(l1)::value - kFrom;
    constexpr int kAll = TM * TN;
    int done = 0;
#pragma unroll
    for (int m = 0; m < kAll; ++m) {
      const int a = m / TN, b = m % TN;
      acc[a][b] = mma16(wf[s][b], a < TM - 1 ? xf[a] : xl[s], acc[a][b]);
      if (m < TN) read_w(r_c, m);
      else if (b == 0) read_x(r_c, a - 1);
      else if (m == TN + 1) read_x(r_c, TM - 1);
      if (done < kLoads && (m + 1) * kLoads >= (done + 1) * kAll) load(k, to, kFrom + done++);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  const std::integral_constant<int, 0> c0{};
  const std::integral_constant<int, 1> c1{};
  const std::integral_constant<int, 2> c2{};
  const std::integral_constant<int, 3> c3{};
  const std::integral_constant<int, LE> le{};
  const std::integral_constant<int, LR> lr{};

  uint32_t to = ring_base + 1024u * wave;  // the slot of the stage at hand
  uint32_t flip = kSlot;                   // from it to the other one
#pragma unroll
  for (int i = 0; i < LR; ++i) load(0, to, i);
#pragma unroll
  for (int i = 0; i < LE; ++i) load(stage_k(1), to + flip, i);
  stage_barrier<LE>();
#pragma unroll
  for (int i = 0; i < TN; ++i) read_w(c0, i);
#pragma unroll
  for (int i = 0; i < TM; ++i) read_x(c0, i);
  // The early loads of stage kt + 1 are under way. At the barrier before its last step, stage kt + 1
  // has arrived and every wave has read stage kt, whose slot then takes the early loads of
  // stage kt + 2.
  for (int kt = 0; kt < nk; ++kt) {
    multiply(c0, c1, le, lr, stage_k(kt + 1), to + flip);
    multiply(c1, c2, c0, c0, 0, 0);
    multiply(c2, c3, c0, c0, 0, 0);
    stage_barrier<0>();
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      x_at[s] += flip;
      w_at[s] += flip;
      asm volatile("" : "+v"(x_at[s]), "+v"(w_at[s]));
    }
    multiply(c3, c0, c0, le, stage_k(kt + 2), to);
    to += flip;
    flip = -flip;
  }
  // (the loads past the last stage: none may be under way when the workgroup ends)
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");

  if constexpr (Extra::kOn) expand_wide(ex, g, m0 + wm * WM, M, n0 + wn * WN, N, acc);

  // The results go through LDS, two row tiles at a time, so that bias, activation and the stores
  // are a short loop over whole rows: a lane has 8 neighbouring columns of every fourth row. A
  // wave has its own 32 KiB there; unit u of 16 bytes of row r is at u ^ (r % 16).
  __syncthreads();  // (no wave reads operands any more)
  const uint32_t out_at = ring_base + kOut * wave;
  const int col = n0 + wn * WN + 8 * (lane & 15);
  const bool whole = G.ldy % 8 == 0 && (reinterpret_cast<uintptr_t>(G.y) & 15u) == 0 && col + 8 <= N;
  const int act = G.act;
  float bias[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) bias[e] = G.bias ? bf16_to_f32(G.bias[min(col + e, N - 1)]) : 0.f;
#pragma unroll
  for (int a = 0; a < TM; a += 2) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f32x16& c = acc[a + i][j];
          const uint32_t unit = uint32_t(8 * j + 2 * q + lh) ^ (li & 15);
          lds_write(out_at + 512 * li + 16 * unit, 16384 * i,
                    f32x4{c[4 * q], c[4 * q + 1], c[4 * q + 2], c[4 * q + 3]});
        }
#pragma unroll 2
    for (int r = lane >> 4; r < 64; r += 4) {
      const uint32_t at = out_at + 512 * r;
      const uint32_t u = 2 * (lane & 15);
      const uint4 lo = lds_read(at + 16 * (u ^ (r & 15)), 0);
      const uint4 hi = lds_read(at + 16 * ((u + 1) ^ (r & 15)), 0);
      const uint32_t bits[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(bits[e]) + bias[e];
      if (act != WKV7_ACT_NONE) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          v[e] = act == WKV7_ACT_TANH ? wide_tanh(v[e]) : 1.f / (1.f + __expf(-v[e]));
      }
      const uint4 out = {pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]),
                         pack_bf16(v[6], v[7])};
      const int64_t p = m0 + wm * WM + 32 * a + r;
      const int64_t to = p < M ? ex.out_row(p) : -1;
      if (to < 0) continue;
      uint16_t* const y = G.y + to * G.ldy + col;
      if (whole) {
        *reinterpret_cast<uint4*>(y) = out;
      } else {
        const uint32_t w[4] = {out.x, out.y, out.z, out.w};
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (col + e < N) y[e] = uint16_t(w[e / 2] >> (16 * (e & 1)));
      }
    }
  }
}

template <int TM, class Extra>
int launch_wide(int64_t m, const wkv7_proj_group* gs, int ng, const Extra& ex, hipStream_t s) {
  ProjArgs args{};
  args.m = m;
  args.ngroups = ng;
  args.parts = 1;
  const int64_t tiles_m = (m + 64 * TM - 1) / (64 * TM);
  int64_t end = 0;
  for (int i = 0; i < ng; ++i) {
    args.g[i] = gs[i];
    end += tiles_m * ((gs[i].n + kWideN - 1) / kWideN);
    if (end > int64_t(0x7fffffff) - kXcds) return WKV7_ERR_ARG;
    args.tile_end[i] = int32_t(end);
  }
  args.tiles_m = int32_t(tiles_m);
  args.xcd_span = int32_t((end + kXcds - 1) / kXcds);
  proj_wide_kernel<TM>
      <<<unsigned(args.xcd_span) * kXcds, 64 * kWideWaves, 0, s>>>(args, ex);
  return launch_status();
}

}  // namespace
}  // namespace wkv7
