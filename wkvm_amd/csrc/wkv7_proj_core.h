// Kernels of thin products of many weights in one launch (wkv7_proj_grouped), and the same with a
// low-rank adapter of each row's own beside the shared weight (wkv7_proj_adapters): a second
// kernel argument says which.
#pragma once

#include <type_traits>

#include "wkv7_common.h"

namespace wkv7 {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));


constexpr int kXcds = 8;  // MI355X: workgroups are dealt round-robin over 8 XCDs

struct ProjArgs {
  wkv7_proj_group g[WKV7_PROJ_MAX_GROUPS];
  int32_t tile_end[WKV7_PROJ_MAX_GROUPS];  // exclusive prefix sums of work items per group
  int64_t ws_off[WKV7_PROJ_MAX_GROUPS];    // split k: group's partials, [parts][m][n] fp32
  int64_t elem_end[WKV7_PROJ_MAX_GROUPS];  // split k: prefix sums of m * n
  float* ws;
  int64_t m;
  int32_t tiles_m;
  int32_t ngroups;
  int32_t xcd_span;  // work items per XCD: ceil(items / kXcds)
  int32_t parts;     // k parts per output tile (1: the tile's workgroup covers all of k)
};

__device__ __forceinline__ f32x4 mma(const uint4& a, const uint4& b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                 __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

template <int KC>
__device__ __forceinline__ int swz(int row, int chunk) {
  return row * KC + (chunk ^ (row & (KC - 1)));
}

__device__ __forceinline__ float activate(float v, int act) {
  if (act == WKV7_ACT_TANH) return tanhf(v);
  if (act == WKV7_ACT_SIGMOID) return 1.f / (1.f + __expf(-v));
  return v;
}

// One stage of the LDS ring: the A rows (x) then the B rows (w) of a
// (8 KC)-wide k block, KC swizzled 16-byte chunks per row.
template <int BM, int BN, int KC>
struct Stage {
  uint4 c[(BM + BN) * KC];
};

typedef __attribute__((address_space(3))) uint4 lds_uint4;

// LDS byte address of a __shared__ location.
__device__ __forceinline__ uint32_t lds_addr(const uint4* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const lds_uint4*)p));
}

// Direct load: 16 bytes per lane from global memory into LDS, lane l's bytes
// at lds_base + 16 l (lds_base is wave-uniform and bound to M0 as an input
// operand, so the compiler writes M0 itself and knows its value; one wait
// state separates that write from its use). Issued as inline assembly so that the
// compiler's wait insertion neither sees these LDS writes (it would wait for
// every pending direct load before any LDS read) nor counts them: all waits
// for them are the explicit ones of stage_barrier below.
__device__ __forceinline__ void load_lds16(const void* src, uint32_t lds_base) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :
               : "{m0}"(lds_base), "v"(src)
               : "memory");
}

// Wait until at most N direct loads of this wave are pending and its LDS
// reads are done, then the workgroup barrier.
template <int N>
__device__ __forceinline__ void stage_barrier() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(N) : "memory");
}

// stage_barrier for a run-time count of pending stages (0 .. P) of L loads.
template <int L, int P>
__device__ __forceinline__ void wait_pending(int pending) {
  if constexpr (P == 0) {
    stage_barrier<0>();
  } else {
    if (pending >= P) stage_barrier<P * L>();
    else wait_pending<L, P - 1>(pending);
  }
}

// Every row's own low-rank term, or none of it.
struct NoAdapters {
  static constexpr bool kOn = false;
  __device__ __forceinline__ int64_t row(int64_t m) const { return m; }
  __device__ __forceinline__ int64_t out_row(int64_t m) const { return m; }
  __device__ __forceinline__ bool empty(int64_t) const { return false; }
};

// The rows are taken in the order of their adapters ("positions"), so that a tile holds few of
// them. h holds s_a x A_a^T of every position, per slab of 16 ranks as three bf16 parts of 16 (all
// 24 bits of the fp32 sum: with two parts the terms' 2^-18 shows where an output nearly cancels,
// up to 1.03 bf16 ulp of it), b the other factors as [adapter][slab][n][16]. Two MFMAs of 32 k
// values multiply a slab's parts with the same 16 columns of B: the first two parts, then half of
// the last one twice (not once beside zeros, which an infinite B would turn into NaN).
struct Adapters {
  static constexpr bool kOn = true;
  const int32_t* order;  // [positions] row of every position, or a negative number: none
  const int32_t* id;     // [positions] its adapter, or a negative number
  const int32_t* end;    // [positions] one past the last position of its adapter
  int64_t rows;
  const uint16_t* h[WKV7_PROJ_MAX_GROUPS];
  const uint16_t* b[WKV7_PROJ_MAX_GROUPS];  // NULL: a product without adapters
  const int32_t* rank[WKV7_PROJ_MAX_GROUPS];
  int32_t count[WKV7_PROJ_MAX_GROUPS];
  int32_t slabs[WKV7_PROJ_MAX_GROUPS];
  // the row that a position reads (one that has none reads some row)
  __device__ __forceinline__ int64_t row(int64_t p) const {
    return min(max(int64_t(order[p]), int64_t(0)), rows - 1);
  }
  // the row that it writes, or a negative number
  __device__ __forceinline__ int64_t out_row(int64_t p) const {
    const int64_t r = order[p];
    return r < rows ? r : -1;
  }
  // In a plan of many rows: no row at the first position of a tile, a multiple of 32, none in all of
  // it (every run starts at such a position, so an empty one lies behind the last run). A plan has
  // room for a gap behind every adapter that is loaded: 600 rows of 2080 beside 8 of them 26 us,
  // beside 1,000 39, without this 255.
  __device__ __forceinline__ bool empty(int64_t p) const { return order[p] < 0; }
};

// Walks the (run, slab) pairs of up to 64 positions from p0: runs of positions that share an
// adapter, and the slabs of 16 ranks that it has. Uniform over the wave; a lane looks at one
// position, so that the walk itself waits for nothing.
struct Pairs {
  int lo = 0, hi = 0, a = 0, s = 0;  // positions [lo, hi), adapter, slab
  int sn = 0;
  int id = -1, end = 0, ns = 0;      // of the lane's position
  uint64_t starts;
  __device__ __forceinline__ Pairs(const Adapters& ad, int g, int64_t p0, int rows) {
    const int lane = threadIdx.x & 63;
    if (lane < rows) {
      id = ad.id[p0 + lane];
      end = int(min(int64_t(ad.end[p0 + lane]) - p0, int64_t(rows)));
      if (id >= 0 && id < ad.count[g]) ns = min((ad.rank[g][id] + 15) >> 4, ad.slabs[g]);
    }
    const int before = __shfl_up(end, 1);
    starts = __ballot(ns > 0 && (lane == 0 || before != end));
  }
  __device__ __forceinline__ bool next() {
    if (++s < sn) return true;
    if (!starts) return false;
    lo = __builtin_ctzll(starts);
    starts &= starts - 1;
    hi = __builtin_amdgcn_readlane(end, lo);
    a = __builtin_amdgcn_readlane(id, lo);
    sn = __builtin_amdgcn_readlane(ns, lo);
    s = 0;
    return true;
  }
  __device__ __forceinline__ bool next(int n) {
    bool more = true;
    for (int i = 0; i < n && more; ++i) more = next();
    return more;
  }
};

// The low-rank terms of 16 TM positions from p0 (at most 64) and 16 TN columns from n0: for every
// run of positions that share an adapter and every slab of it, two MFMAs per tile, of which the
// run's own positions are taken (not the others times zero: an adapter with an inf or NaN in it
// must not reach other requests). The operands come straight to registers, U (run, slab) pairs
// in flight at once: a tile of a decode batch may meet an adapter per row, and each of them is
// one pass from memory. This comes after the shared product: with the first U fetched ahead of it
// they would be held in registers all through the loop, and the compiler waits for them before the
// first of the loop's own loads (three products of 256 rows of 2048, 32 adapters of 32 ranks: 34.6
// us so, 34.1 now; one of 203 rows of 4096, 24 adapters of 64 ranks: 45 and 42).
// kSwap: acc holds the transposed tile. Pairs are dealt to `step` waves, or workgroups that share
// a tile.
template <int TM, int TN, int U, bool kSwap>
struct Expand {
  static_assert(TM <= 4, "a lane per position");
  const uint16_t *hp, *bp;
  int n0, N, rows, slabs, step;
  Pairs pairs;
  bool more;
  uint4 hf[U][TM][2], bf[U][TN];
  int from[U], to[U];

  __device__ __forceinline__ Expand(const Adapters& ad, int g, int64_t p0, int64_t M, int n0_,
                                    int N_, int mine, int step_)
      : n0(n0_),
        N(N_),
        rows(ad.b[g] ? int(min(int64_t(16 * TM), M - p0)) : 0),
        slabs(ad.slabs[g]),
        step(step_),
        pairs(ad, g, p0, rows) {
    const int lg = (threadIdx.x & 63) >> 4;
    hp = ad.h[g] + (p0 * slabs) * 48 + 8 * lg;
    bp = ad.b[g] + 8 * (lg & 1);
    more = pairs.next(mine + 1);
  }

  __device__ __forceinline__ void fetch() {
    const int lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      from[u] = to[u] = 0;
      if (!more) continue;
      from[u] = pairs.lo;
      to[u] = pairs.hi;
      const uint16_t* b = bp + ((int64_t(pairs.a) * slabs + pairs.s) * N) * 16;
#pragma unroll
      for (int j = 0; j < TN; ++j)
        bf[u][j] = *reinterpret_cast<const uint4*>(b + int64_t(min(n0 + 16 * j + li, N - 1)) * 16);
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const int r = min(max(16 * i + li, pairs.lo), pairs.hi - 1);
        const uint16_t* p = hp + (int64_t(r) * slabs + pairs.s) * 48;
        hf[u][i][0] = *reinterpret_cast<const uint4*>(p);
        hf[u][i][1] = *reinterpret_cast<const uint4*>(p + 32 - 16 * (lg >> 1));
      }
      more = pairs.next(step);
    }
  }

  __device__ __forceinline__ void add(f32x4 (&acc)[TM][TN]) {
    const int lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
    while (more) {
      fetch();
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          if (to[u] <= 16 * i || from[u] >= 16 * i + 16) continue;
          const bool whole = from[u] <= 16 * i && to[u] >= min(rows, 16 * i + 16);
#pragma unroll
          for (int j = 0; j < TN; ++j) {
            auto term = [&](f32x4 c) {  // the small parts first
#pragma unroll
              for (int q = 1; q >= 0; --q)
                c = kSwap ? mma(bf[u][j], hf[u][i][q], c) : mma(hf[u][i][q], bf[u][j], c);
              return c;
            };
            if (whole) {
              acc[i][j] = term(acc[i][j]);
              continue;
            }
            const f32x4 d = term(f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int r = 16 * i + (kSwap ? li : 4 * lg + e);
              acc[i][j][e] += r >= from[u] && r < to[u] ? d[e] : 0.f;
            }
          }
        }
    }
  }
};

template <int BM, int BN, int S, int GM, int GN, int BK, bool kSplit, class Extra>
__global__ __launch_bounds__(64 * GM * GN) void proj_kernel(const ProjArgs args, const Extra ex) {
  constexpr int NW = GM * GN;                 // waves, a GM x GN grid
  constexpr int WM = BM / GM, WN = BN / GN;   // wave tile
  constexpr int TM = WM / 16, TN = WN / 16;   // accumulator tiles per wave
  // k per stage BK = 64 or 128: KC chunks of 16 bytes per row. Each
  // wave-wide direct load fills 1 KiB of a stage = 64 / KC rows; a thread
  // issues L of them per stage.
  constexpr int KC = BK / 8, kStepsFull = BK / 32;
  static_assert(BK == 64 || BK == 128, "stage depth");
  constexpr int kRowsPerLoad = 64 / KC;
  constexpr int L = (BM + BN) / (kRowsPerLoad * NW);
  static_assert(TM >= 1 && TN >= 1 && (BM + BN) % (kRowsPerLoad * NW) == 0 && BM % 8 == 0,
                "tile shape");
  __shared__ Stage<BM, BN, KC> ring[S];

  // Workgroup b runs on XCD b % 8; XCD x takes the x-th contiguous run of
  // tiles (ordered by group, then output columns, then rows), so each XCD's
  // L2 holds the x rows of one or two groups instead of all of them.
  const int bid = int(blockIdx.x % kXcds) * args.xcd_span + int(blockIdx.x / kXcds);
  int g = 0;
  while (g + 1 < args.ngroups && bid >= args.tile_end[g]) ++g;
  if (bid >= args.tile_end[g]) return;
  const wkv7_proj_group& G = args.g[g];
  const int item = bid - (g ? args.tile_end[g - 1] : 0);
  const int part = kSplit ? item % args.parts : 0;
  const int local = kSplit ? item / args.parts : item;
  const int tm = local % args.tiles_m, tn = local / args.tiles_m;
  const int64_t M = args.m;
  const int N = G.n, K = G.k;
  const int64_t m0 = int64_t(tm) * BM;
  const int n0 = tn * BN;
  static_assert(BM % 32 == 0, "a tile starts where a run may");
  if (M > WKV7_ADAPTER_PACKED_ROWS && ex.empty(m0)) return;

  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int wm = wave % GM, wn = wave / GM;
  const int li = lane & 15, lg = lane >> 4;
  // LDS destinations are wave-uniform: computed in scalar registers.
  const int wave_s = __builtin_amdgcn_readfirstlane(wave);
  const uint32_t ring_base = lds_addr(&ring[0].c[0]) + 1024u * wave_s;
  constexpr uint32_t kStageBytes = sizeof(Stage<BM, BN, KC>);

  // Load i of this wave fills stage rows R j .. R j + R - 1 (R = 64 / KC,
  // j = NW i + wave); lane l writes slot KC row + q (row = R j + l / KC,
  // q = l % KC), which holds logical chunk q ^ (row & (KC - 1)) of that row.
  const uint16_t* src[L];
  int chunk_k[L];
#pragma unroll
  for (int i = 0; i < L; ++i) {
    const int row = kRowsPerLoad * (NW * i + wave) + lane / KC;
    const int c = (lane % KC) ^ (row & (KC - 1));
    chunk_k[i] = 8 * c;
    if (row < BM) {
      const int64_t m = ex.row(min(m0 + row, M - 1));
      src[i] = G.x + m * G.ldx + 8 * c;
    } else {
      const int64_t n = min(int64_t(n0 + row - BM), int64_t(N - 1));
      src[i] = G.w + n * G.ldw + 8 * c;
    }
  }
  // Issue stage kt's loads into ring slot `slot`. In a partial tail stage
  // (k % BK != 0) chunks past k re-read a valid chunk; nothing multiplies
  // them.
  // This workgroup's k stages: [kb, kb + nk) of the product's nk_all, all
  // of them unless k is split over `parts` workgroups.
  const int nk_all = (K + BK - 1) / BK;
  const int spp = kSplit ? (nk_all + args.parts - 1) / args.parts : nk_all;
  const int kb = kSplit ? min(part * spp, nk_all) : 0;
  const int nk = kSplit ? min(nk_all, kb + spp) - kb : nk_all;
  const bool has_tail = (K % BK) && kb + nk == nk_all;  // the partial stage is ours
  auto issue = [&](int kt, int slot) {
    const int k0 = (kb + kt) * BK;
    const uint32_t base = ring_base + kStageBytes * slot;
    if (k0 + BK <= K) {
#pragma unroll
      for (int i = 0; i < L; ++i) load_lds16(src[i] + k0, base + 1024u * NW * i);
    } else {
#pragma unroll
      for (int i = 0; i < L; ++i)
        load_lds16(src[i] + (k0 + chunk_k[i] >= K ? K - 8 - chunk_k[i] : k0),
                   base + 1024u * NW * i);
    }
  };

  f32x4 acc[TM][TN];
#pragma unroll
  for (int a = 0; a < TM; ++a)
#pragma unroll
    for (int b = 0; b < TN; ++b) acc[a][b] = f32x4{0.f, 0.f, 0.f, 0.f};

  // A stage: all fragment reads first, then its MFMAs with the next stage's
  // loads (when kIssue) spread between them, so the matrix core works while
  // a load waits for the load pipe. Inline-assembly loads are scheduling
  // boundaries, which keeps that placement.
  auto stage = [&](int kt, auto steps_c, auto issue_c) {
    constexpr int kSteps = decltype(steps_c)::value;
    constexpr bool kIssue = decltype(issue_c)::value;
    constexpr int kMfma = kSteps * TM * TN;
    const Stage<BM, BN, KC>& st = ring[kt % S];
    // (kt counts this workgroup's stages; k offsets add kb)
    uint4 af[kSteps][TM], bf[kSteps][TN];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
#pragma unroll
      for (int a = 0; a < TM; ++a) af[s][a] = st.c[swz<KC>(wm * WM + a * 16 + li, 4 * s + lg)];
#pragma unroll
      for (int b = 0; b < TN; ++b)
        bf[s][b] = st.c[swz<KC>(BM + wn * WN + b * 16 + li, 4 * s + lg)];
    }
    const int k1 = (kb + kt + S - 1) * BK;
    const uint32_t base = ring_base + kStageBytes * ((kt + S - 1) % S);
    int issued = 0;
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int a = 0; a < TM; ++a)
#pragma unroll
        for (int b = 0; b < TN; ++b) {
          acc[a][b] = mma(af[s][a], bf[s][b], acc[a][b]);
          if constexpr (kIssue) {
            // load i goes after MFMA number ((i + 1) * kMfma) / (L + 1)
            const int m = (s * TM + a) * TN + b + 1;
#pragma unroll
            for (int i = 0; i < L; ++i)
              if (m == ((i + 1) * kMfma) / (L + 1) && issued == i) {
                load_lds16(src[i] + k1, base + 1024u * NW * i);
                ++issued;
              }
          }
        }
    if constexpr (kIssue) {
#pragma unroll
      for (int i = 0; i < L; ++i)
        if (issued == i) {
          load_lds16(src[i] + k1, base + 1024u * NW * i);
          ++issued;
        }
    }
  };

  // Stages 0 .. S-2 in flight before the loop. In iteration kt the wave waits
  // until only the loads of stages kt+1 .. min(kt+S-2, nk-1) are pending and
  // its LDS reads are done; one barrier publishes stage kt to every wave and
  // retires slot (kt-1) % S, which receives stage kt + S - 1 while stage kt
  // is multiplied. Only the last stage can be partial (32, 64 or 96 wide),
  // and nothing is issued after it.
  static_assert(S >= 2 && S <= 8, "wait ladder covers rings of 2..8 stages");
#pragma unroll
  for (int p = 0; p < S - 1; ++p)
    if (p < nk) issue(p, p);
  for (int kt = 0; kt < nk; ++kt) {
    wait_pending<L, S - 2>(min(S - 2, nk - 1 - kt));
    if (kt + S - 1 < nk) {
      if (kt + S - 1 == nk - 1 && has_tail) {
        issue(kt + S - 1, (kt + S - 1) % S);  // the tail stage's clamped loads
        stage(kt, std::integral_constant<int, kStepsFull>{}, std::false_type{});
      } else {
        stage(kt, std::integral_constant<int, kStepsFull>{}, std::true_type{});
      }
    } else if ((kb + kt) * BK + BK <= K) {
      stage(kt, std::integral_constant<int, kStepsFull>{}, std::false_type{});
    } else {
      const int steps = (K - (kb + kt) * BK) / 32;  // 1 .. kStepsFull - 1
      if (steps == 1) {
        stage(kt, std::integral_constant<int, 1>{}, std::false_type{});
      } else if constexpr (kStepsFull > 2) {
        if (steps == 2)
          stage(kt, std::integral_constant<int, 2>{}, std::false_type{});
        else
          stage(kt, std::integral_constant<int, 3>{}, std::false_type{});
      }
    }
  }

  if constexpr (Extra::kOn) {
    // (Pairs under way: 16 waves have 128 registers each, and 4 pairs fit them as well as 2, 16 in
    // the tiles of 8 waves as well as 8. They gain nothing: 256 rows over 32 adapters 34.0 us and
    // 33.7 so, 203 rows of 4096 42.2 and 41.5, 64 rows with one of their own each 23.7 either way.)
    constexpr int kPairs = NW >= 16 ? 2 : TM > 1 ? 4 : 8;
    Expand<TM, TN, kPairs, false>(ex, g, m0 + wm * WM, M, n0 + wn * WN, N, part,
                                  kSplit ? args.parts : 1)
        .add(acc);
  }

  if constexpr (kSplit) {  // fp32 partial tile; proj_reduce_kernel finishes the sum
    float* wsp = args.ws + args.ws_off[g] + int64_t(part) * M * N;
#pragma unroll
    for (int b = 0; b < TN; ++b) {
      const int col = n0 + wn * WN + b * 16 + li;
      if (col >= N) continue;
#pragma unroll
      for (int a = 0; a < TM; ++a)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int64_t row = m0 + wm * WM + a * 16 + 4 * lg + e;
          if (row < M) wsp[row * N + col] = acc[a][b][e];
        }
    }
    return;
  }
  const int act = G.act;
#pragma unroll
  for (int b = 0; b < TN; ++b) {
    const int col = n0 + wn * WN + b * 16 + li;
    if (col >= N) continue;
    const float bias = G.bias ? bf16_to_f32(G.bias[col]) : 0.f;
#pragma unroll
    for (int a = 0; a < TM; ++a) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t p = m0 + wm * WM + a * 16 + 4 * lg + e;
        const int64_t row = p < M ? ex.out_row(p) : -1;
        if (row >= 0) G.y[row * G.ldy + col] = f32_to_bf16(activate(acc[a][b][e] + bias, act));
      }
    }
  }
}

// Split k: y = act(sum of the k parts' partials, in part order, + bias), one
// thread per output element.
template <class Extra>
__global__ __launch_bounds__(256) void proj_reduce_kernel(const ProjArgs args, const Extra ex) {
  const int64_t e = int64_t(blockIdx.x) * 256 + threadIdx.x;
  int g = 0;
  while (g + 1 < args.ngroups && e >= args.elem_end[g]) ++g;
  if (e >= args.elem_end[g]) return;
  const wkv7_proj_group& G = args.g[g];
  const int64_t local = e - (g ? args.elem_end[g - 1] : 0);
  const int64_t row = local / G.n;
  const int col = int(local - row * G.n);
  const int64_t plane = args.m * G.n;
  const float* src = args.ws + args.ws_off[g] + local;
  float sum = 0.f;
  for (int p = 0; p < args.parts; ++p) sum += src[p * plane];
  const float bias = G.bias ? bf16_to_f32(G.bias[col]) : 0.f;
  const int64_t to = ex.out_row(row);
  if (to >= 0) G.y[to * G.ldy + col] = f32_to_bf16(activate(sum + bias, G.act));
}

// One row tile (m <= 16): a 16-column tile of a product by one workgroup, its
// k dealt to NW waves in 64-wide chunks (wave w: chunks w, w + NW, ..), so that
// the workgroup reads contiguous bytes of each weight row. Every operand goes
// from memory straight to registers and up to four chunks of a wave are in
// flight at once: with few rows there is nothing to share through LDS, and what
// bounds the launch is the latency of the weights' one pass from memory, which
// a ring with a barrier per stage pays several times. The waves' fp32 partial
// tiles are summed through LDS in wave order. 16 rows, us per launch in a HIP
// graph over distinct weights, before (32 x 32 tiles, k split) and now: LoRA
// up-projections 4.3 -> 3.6, o_proj 8.0 -> 6.7 (8.6 MB); hidden size 768: first
// stage 5.4 -> 4.6, o_proj 5.0 -> 4.0. Slower: 32 columns per workgroup (o_proj
// 8.7: half of the workgroups), non-temporal weight loads (7.2), 16 waves.
template <int NW, class Extra>
__global__ __launch_bounds__(64 * NW) void proj_thin_kernel(const ProjArgs args, const Extra ex) {
  __shared__ f32x4 red[NW][64];
  const int bid = int(blockIdx.x);
  int g = 0;
  while (g + 1 < args.ngroups && bid >= args.tile_end[g]) ++g;
  const wkv7_proj_group& G = args.g[g];
  const int n0 = (bid - (g ? args.tile_end[g - 1] : 0)) * 16;
  const int M = int(args.m), N = G.n, K = G.k;
  const int t = threadIdx.x, lane = t & 63, li = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  // A: 16 rows of w, B: 16 rows of x (rows past the end repeat the last one and
  // are not stored); the accumulator holds columns n0 + 4 lg .. + 3 of row li.
  const uint16_t* wp = G.w + int64_t(min(n0 + li, N - 1)) * G.ldw + 8 * lg;
  const uint16_t* xp = G.x + ex.row(min(li, M - 1)) * G.ldx + 8 * lg;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  // U chunks of this wave from chunk c on. Only the last chunk of all can be
  // half a chunk wide: its second half re-reads the first and is left out.
  auto chunks = [&](int c, auto u_c) {
    constexpr int U = decltype(u_c)::value;
    uint4 wf[U][2], xf[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k0 = 64 * (c + u * NW), k1 = k0 + 32 < K ? k0 + 32 : k0;
      wf[u][0] = *reinterpret_cast<const uint4*>(wp + k0);
      wf[u][1] = *reinterpret_cast<const uint4*>(wp + k1);
      xf[u][0] = *reinterpret_cast<const uint4*>(xp + k0);
      xf[u][1] = *reinterpret_cast<const uint4*>(xp + k1);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      acc = mma(wf[u][0], xf[u][0], acc);
      if (64 * (c + u * NW) + 32 < K) acc = mma(wf[u][1], xf[u][1], acc);
    }
  };
  const int nc = (K + 63) / 64;
  int c = wave;
  for (; c + 3 * NW < nc; c += 4 * NW) chunks(c, std::integral_constant<int, 4>{});
  if (c + 2 * NW < nc) chunks(c, std::integral_constant<int, 3>{});
  else if (c + NW < nc) chunks(c, std::integral_constant<int, 2>{});
  else if (c < nc) chunks(c, std::integral_constant<int, 1>{});
  if constexpr (Extra::kOn) {
    f32x4 sum[1][1] = {{acc}};
    Expand<1, 1, 4, true>(ex, g, 0, M, n0, N, wave, NW).add(sum);
    acc = sum[0][0];
  }
  red[wave][lane] = acc;
  __syncthreads();
  if (t >= 256) return;  // thread t: row t / 16, column t % 16 of the tile
  const int row = t >> 4, col = t & 15;
  if (row >= M || n0 + col >= N) return;
  const float* part = reinterpret_cast<const float*>(&red[0][(col >> 2) * 16 + row]) + (col & 3);
  float sum = 0.f;
#pragma unroll
  for (int w = 0; w < NW; ++w) sum += part[w * 64 * 4];
  const float bias = G.bias ? bf16_to_f32(G.bias[n0 + col]) : 0.f;
  const int64_t to = ex.out_row(row);
  if (to >= 0) G.y[to * G.ldy + n0 + col] = f32_to_bf16(activate(sum + bias, G.act));
}

}  // namespace
}  // namespace wkv7
