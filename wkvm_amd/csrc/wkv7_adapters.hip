// Projections shared by all rows with a low-rank adapter of each row's own beside them:
//   y[m] = act( x[m] W^T + bias + s_a (x[m] A_a^T) B_a^T ),   a = id[m]
//
// Two launches for any mix of adapters. The first computes h = s_a x A_a^T, tiles of at most 16
// rows of one adapter by 16 ranks; the rows are visited in the order of their adapters, so every
// A is read about once. The second is the shared product itself (wkv7_proj_core.h) over the rows
// in that order, which adds h B_a^T to its accumulators before bias, activation and the one
// rounding. h is summed in fp32 and kept whole as three bf16 parts, which the matrix cores
// multiply with B in two instructions per slab of 16 ranks. Two launches because every output
// column needs all of h, and a workgroup per tile of y would compute it once per column tile. (For
// a few rows over a few ranks that may cost less than a second launch: not measured.)
//
// Three products in a HIP graph (the shared products alone in brackets): 8 rows of 2048 x 2048 with
// two adapters of 16 ranks 14.9 us (8.5), 64 rows with one of their own each 23.7 (9.9), 256 rows over
// 32 of 32 ranks 33.4 (16.9), 3,001 rows of prompts 126, 32,768 rows 987 to 1,003.
#include <algorithm>
#include <numeric>

#include "wkv7_proj_plan.h"
#include "wkv7_proj_wide.h"

namespace wkv7 {
namespace {

constexpr int kSlab = WKV7_ADAPTER_SLAB;  // ranks of a slab, rows of a tile
constexpr int kParts = 3;                 // bf16 parts of a value of h
constexpr int kAlign = 32;                // positions that a run starts at a multiple of (many rows)

struct ShrinkGroup {
  const uint16_t* x;
  const uint16_t* a;    // [count][16 slabs][k]
  const float* scale;   // [count]
  const int32_t* rank;  // [count]
  uint16_t* h;          // [m][slabs][kParts][16]
  int64_t ldx;
  int32_t k, count, slabs;
};

constexpr int kTileInts = 20;  // first position, rows, adapter, 0, the 16 rows

struct ShrinkArgs {
  ShrinkGroup g[WKV7_PROJ_MAX_GROUPS];
  const int32_t* tiles;  // [ntiles][kTileInts]
  int32_t ntiles;
  int64_t m, positions;
  float last;  // factor of the last part of h: 1 / 2 where the products take it twice
};

// A tile of the plan, held to what the call has: rows is 0 where there is nothing to do. `row` is
// the row of the lane's position (of the last one, past the end).
struct Tile {
  int64_t first, row;
  int rows, id;
};
__device__ __forceinline__ Tile get_tile(const ShrinkArgs& args, const ShrinkGroup& G, int64_t t,
                                         int li) {
  const int32_t* e = args.tiles + kTileInts * t;
  const int4 head = *reinterpret_cast<const int4*>(e);
  Tile tile{head.x, e[4 + li], head.y, head.z};
  if (tile.rows < 1 || tile.rows > kSlab || tile.id < 0 || tile.id >= G.count || tile.first < 0 ||
      tile.first + tile.rows > args.positions)
    tile.rows = 0;
  tile.row = min(max(tile.row, int64_t(0)), args.m - 1);
  return tile;
}

// s times four of a row's sums, `left` of them ranks that the adapter has (a padding rank is 0
// also where x is not finite), as bf16 parts whose sum is the value, each of its sign and zero only
// where it is: a part takes the upper half of the next smaller number in 32 bits, the last one
// what is left (24 bits less twice 8). So an infinite B gives the infinity that the whole value
// gives; times a part of zero, or of the other sign, it would be NaN. All parts of a value that is
// not finite are the value. (Below 2^-94 parts underflow.) The last part is stored times `last`.
__device__ __forceinline__ void store_h(uint16_t* h, const f32x4& v, float s, int left,
                                        float last) {
  float x[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = e < left ? s * v[e] : 0.f;
#pragma unroll
  for (int p = 0; p + 1 < kParts; ++p) {
    uint32_t top[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t bits = __float_as_uint(x[e]);
      const bool finite = (bits & 0x7f800000u) != 0x7f800000u;
      top[e] = (finite && bits << 1 ? bits - 1 : bits) & 0xffff0000u;
      x[e] = finite ? x[e] - __uint_as_float(top[e]) : x[e];
    }
    *reinterpret_cast<uint2*>(h + p * kSlab) = {top[0] >> 16 | top[1], top[2] >> 16 | top[3]};
  }
  *reinterpret_cast<uint2*>(h + (kParts - 1) * kSlab) = {pack_bf16(last * x[0], last * x[1]),
                                                         pack_bf16(last * x[2], last * x[3])};
}

// Few tiles: a workgroup per tile and slab, k dealt to NW waves in 64-wide chunks whose sums
// are joined through LDS in wave order. Bound by latency (a launch, the tile, the operands of four
// chunks in flight, the join: 6 us for 8 rows of 2048 and 64 rows alike); 256 rows over 32 adapters of
// 32 ranks 9.9 us.
template <int NW>
__global__ __launch_bounds__(64 * NW) void shrink_thin_kernel(const ShrinkArgs args) {
  __shared__ f32x4 red[NW][64];
  const ShrinkGroup& G = args.g[blockIdx.z];
  const int slab = blockIdx.y;
  if (!G.a || slab >= G.slabs) return;
  const int t = threadIdx.x, lane = t & 63, li = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const Tile tile = get_tile(args, G, blockIdx.x, li);
  if (tile.rows == 0) return;
  const int K = G.k;
  // (the first slab is read before its adapter's rank is known: it nearly always has one)
  const int left = G.rank[tile.id] - slab * kSlab;
  if (slab > 0 && left <= 0) return;
  const float scale = G.scale[tile.id];
  const uint16_t* xp = G.x + tile.row * G.ldx + 8 * lg;
  const uint16_t* ap = G.a + ((int64_t(tile.id) * G.slabs + slab) * kSlab + li) * K + 8 * lg;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  auto chunks = [&](int c, auto u_c) {
    constexpr int U = decltype(u_c)::value;
    uint4 af[U][2], xf[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k0 = 64 * (c + u * NW), k1 = k0 + 32 < K ? k0 + 32 : k0;
      af[u][0] = *reinterpret_cast<const uint4*>(ap + k0);
      af[u][1] = *reinterpret_cast<const uint4*>(ap + k1);
      xf[u][0] = *reinterpret_cast<const uint4*>(xp + k0);
      xf[u][1] = *reinterpret_cast<const uint4*>(xp + k1);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      acc = mma(af[u][0], xf[u][0], acc);
      if (64 * (c + u * NW) + 32 < K) acc = mma(af[u][1], xf[u][1], acc);
    }
  };
  const int nc = (K + 63) / 64;
  int c = wave;
  for (; c + 3 * NW < nc; c += 4 * NW) chunks(c, std::integral_constant<int, 4>{});
  if (c + 2 * NW < nc) chunks(c, std::integral_constant<int, 3>{});
  else if (c + NW < nc) chunks(c, std::integral_constant<int, 2>{});
  else if (c < nc) chunks(c, std::integral_constant<int, 1>{});
  red[wave][lane] = acc;
  __syncthreads();
  if (wave != 0) return;
#pragma unroll
  for (int w = 1; w < NW; ++w) acc += red[w][lane];
  // lane: ranks 4 lg .. 4 lg + 3 of row li
  if (li < tile.rows)
    store_h(G.h + ((tile.first + li) * G.slabs + slab) * kParts * kSlab + 4 * lg, acc, scale,
            left - 4 * lg, args.last);
}

// Many tiles: a workgroup for two of them, k dealt to its waves as above and up to four slabs at
// once. Two tiles of one adapter, as nearly all of a prompt's are, share the reads of A, which
// are otherwise twice x's. (32,768 rows of 2048 in three products of rank 32, x alone 400 MB: with
// a wave per tile, which walks 16 rows in steps of 64 bytes, 165 us; a workgroup per tile 148;
// two tiles 109 or 3.7 TB/s of x, which is what bounds it, and 116 with four chunks of k in flight in
// place of two.)
constexpr int kWideShrink = 4;

__global__ __launch_bounds__(64 * kWideShrink) void shrink_wide_kernel(const ShrinkArgs args) {
  constexpr int NW = kWideShrink;
  __shared__ f32x4 red[NW][4][64];
  const ShrinkGroup& G = args.g[blockIdx.y];
  if (!G.a) return;
  const int t = threadIdx.x, lane = t & 63, li = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int K = G.k, nc = (K + 63) / 64;
  // NT tiles of one adapter, NS of its slabs from s0 on
  auto slabs = [&](const Tile* tiles, int rank, int s0, auto nt_c, auto n_c) {
    constexpr int NT = decltype(nt_c)::value, NS = decltype(n_c)::value;
    constexpr int U = NS * NT <= 2 ? 4 : 2;
    const int id = __builtin_amdgcn_readfirstlane(tiles[0].id);
    const uint16_t* ap = G.a + ((int64_t(id) * G.slabs + s0) * kSlab + li) * K + 8 * lg;
    const uint16_t* xp[NT];
    f32x4 acc[NT][NS];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      xp[i] = G.x + tiles[i].row * G.ldx + 8 * lg;
#pragma unroll
      for (int s = 0; s < NS; ++s) acc[i][s] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    for (int c = wave; c < nc; c += U * NW) {
      uint4 xf[U][2][NT], af[U][2][NS];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        // (past the end: the last chunk once more, left out below)
        const int k0 = 64 * min(c + u * NW, nc - 1), k1 = k0 + 32 < K ? k0 + 32 : k0;
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          xf[u][0][i] = *reinterpret_cast<const uint4*>(xp[i] + k0);
          xf[u][1][i] = *reinterpret_cast<const uint4*>(xp[i] + k1);
        }
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          af[u][0][s] = *reinterpret_cast<const uint4*>(ap + int64_t(s) * kSlab * K + k0);
          af[u][1][s] = *reinterpret_cast<const uint4*>(ap + int64_t(s) * kSlab * K + k1);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (c + u * NW >= nc) break;
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int s = 0; s < NS; ++s) {
            acc[i][s] = mma(af[u][0][s], xf[u][0][i], acc[i][s]);
            if (64 * (c + u * NW) + 32 < K) acc[i][s] = mma(af[u][1][s], xf[u][1][i], acc[i][s]);
          }
      }
    }
    const float scale = G.scale[id];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      __syncthreads();
#pragma unroll
      for (int s = 0; s < NS; ++s) red[wave][s][lane] = acc[i][s];
      __syncthreads();
      for (int s = wave; s < NS; s += NW) {  // a slab per wave
        f32x4 sum = red[0][s][lane];
#pragma unroll
        for (int w = 1; w < NW; ++w) sum += red[w][s][lane];
        if (li < tiles[i].rows)
          store_h(G.h + ((tiles[i].first + li) * G.slabs + s0 + s) * kParts * kSlab + 4 * lg, sum,
                  scale, rank - (s0 + s) * kSlab - 4 * lg, args.last);
      }
    }
  };
  auto run = [&](const Tile* tiles, auto nt_c) {
    const int rank = min(G.rank[tiles[0].id], G.slabs * kSlab), all = (rank + kSlab - 1) / kSlab;
    int s = 0;
    for (; s + 4 <= all; s += 4) slabs(tiles, rank, s, nt_c, std::integral_constant<int, 4>{});
    if (all - s == 3) slabs(tiles, rank, s, nt_c, std::integral_constant<int, 3>{});
    else if (all - s == 2) slabs(tiles, rank, s, nt_c, std::integral_constant<int, 2>{});
    else if (all - s == 1) slabs(tiles, rank, s, nt_c, std::integral_constant<int, 1>{});
  };
  const int64_t first = 2 * int64_t(blockIdx.x);
  Tile tiles[2] = {get_tile(args, G, first, li), {}};
  if (first + 1 < args.ntiles) tiles[1] = get_tile(args, G, first + 1, li);
  if (tiles[0].rows > 0 && tiles[1].rows > 0 && tiles[0].id == tiles[1].id) {
    run(tiles, std::integral_constant<int, 2>{});
    return;
  }
#pragma unroll 1
  for (int i = 0; i < 2; ++i) {
    const Tile one = i == 0 ? tiles[0] : tiles[1];
    if (one.rows > 0) run(&one, std::integral_constant<int, 1>{});
  }
}

// Puts one adapter into its place: A's rows and then zeros (blocks [0, a_blocks)), B's columns in
// slabs of 16 with zeros past the rank, scale and rank. A thread moves 16 bytes of the place.
struct LoadArgs {
  const uint16_t *a, *b;
  uint16_t *to_a, *to_b;
  float* to_scale;
  int32_t* to_rank;
  int64_t lda, ldb;
  float scale;
  int32_t r, k, n, slabs, a_blocks;
};

__global__ __launch_bounds__(256) void adapter_load_kernel(const LoadArgs args) {
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    *args.to_scale = args.scale;
    *args.to_rank = args.r;
  }
  uint16_t v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (int(blockIdx.x) < args.a_blocks) {
    const int64_t i = (int64_t(blockIdx.x) * 256 + threadIdx.x) * 8;  // in [16 slabs][k]
    const int64_t row = i / args.k;
    if (row >= int64_t(kSlab) * args.slabs) return;
    if (row < args.r) {
      const uint16_t* p = args.a + row * args.lda + (i - row * args.k);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = p[e];
    }
    *reinterpret_cast<uint4*>(args.to_a + i) = *reinterpret_cast<const uint4*>(v);
    return;
  }
  const int64_t i = (int64_t(blockIdx.x - args.a_blocks) * 256 + threadIdx.x) * 8;  // [slabs][n][16]
  const int64_t row = i / kSlab % args.n, slab = i / kSlab / args.n;
  if (slab >= args.slabs) return;
  const int64_t col = slab * kSlab + i % kSlab;
  const uint16_t* p = args.b + row * args.ldb + col;
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (col + e < args.r) v[e] = p[e];
  *reinterpret_cast<uint4*>(args.to_b + i) = *reinterpret_cast<const uint4*>(v);
}

int64_t max_tiles(int64_t m, int32_t count) { return m / kSlab + std::min<int64_t>(m, count) + 1; }

// Positions of a plan: the rows, and where the runs of an adapter are aligned the gaps too.
int64_t positions(int64_t m, int32_t count) {
  if (m <= WKV7_ADAPTER_PACKED_ROWS) return m;
  const int64_t runs = std::min<int64_t>(m, int64_t(count) + 1);
  return (m + (kAlign - 1) * runs + kAlign - 1) / kAlign * kAlign;
}

// Whether a plan of m rows over count adapters can be: its positions are 32-bit numbers.
bool plan_fits(int64_t m, int32_t count) {
  return m >= 0 && m <= WKV7_ADAPTER_MAX_ROWS && count >= 0 && positions(m, count) <= INT32_MAX;
}

// Where the plan's parts start, in ints.
int64_t plan_part(int64_t positions, int part) { return part * ((positions + 3) / 4 * 4); }

size_t align256(size_t n) { return (n + 255) & ~size_t(255); }

int check_sets(const wkv7_adapter_set* sets, int32_t ngroups, int32_t count) {
  for (int i = 0; i < ngroups; ++i) {
    const wkv7_adapter_set& s = sets[i];
    if (!s.a) continue;
    if (!s.b || !s.scale || !s.rank || s.count < count || s.slabs < 1 ||
        s.slabs > WKV7_ADAPTER_MAX_RANK / kSlab)
      return WKV7_ERR_ARG;
    if (!aligned16(s.a) || !aligned16(s.b)) return WKV7_ERR_SHAPE;
  }
  return WKV7_OK;
}

// What the wide kernel needs of the products: whole stages of k, and rows that its 32-bit offsets
// reach.
bool wide_fits(int64_t m, const wkv7_proj_group* groups, int ng) {
  for (int i = 0; i < ng; ++i) {
    const int64_t k = groups[i].k;
    if (k % 64 || ((m - 1) * groups[i].ldx + k) * 2 > int64_t(0xffffffff) ||
        ((int64_t(groups[i].n) - 1) * groups[i].ldw + k) * 2 > int64_t(0xffffffff))
      return false;
  }
  return true;
}

// The row tile of the wide kernel (in units of 64 rows), 0 for the others: whichever takes the
// least time by its rounds over the units. Microseconds per round of one tile per unit, measured
// at k = 2048 (they scale together with k): 256 x 256 tiles 79, 128 x 256 47, the other kernel's
// 128 x 64 tiles 16.5. Three products of 2048 columns and 2048 k: 3001 rows 114 in 128 x 256 (127
// in 256 x 256, 165 in 128 x 64), 32,768 rows 910 in 256 x 256 (1187, about 2200). A plan of few
// rows does not align its runs as the wide kernel needs.
int wide_tile(int64_t m, int64_t positions, const wkv7_proj_group* groups, int ng, int cus) {
  if (m <= WKV7_ADAPTER_PACKED_ROWS || !wide_fits(m, groups, ng)) return 0;
  const struct { TileShape shape; int tm; double us; } kinds[] = {
      {{128, 64}, 0, 16.5}, {{128, 256}, 2, 47.}, {{256, 256}, 4, 79.}};
  double best = 0.;
  int tm = 0;
  for (const auto& k : kinds) {
    const int64_t tiles = count_tiles(positions, groups, ng, k.shape);
    const double us = k.us * double((tiles + cus - 1) / cus);
    if (best == 0. || us < best) {
      best = us;
      tm = k.tm;
    }
  }
  return tm;
}

struct Work {
  Plan plan;
  int waves;  // of the thin kernel, 0: the tiled one
  int wide;   // row tile of the wide kernel, 0: another one
  size_t h[WKV7_PROJ_MAX_GROUPS];
  size_t partials, bytes;
};

Work make_work(int64_t rows, int64_t m, const wkv7_proj_group* groups, const wkv7_adapter_set* sets,
               int ng, int cus) {
  Work w{};
  w.waves = thin_waves(m, groups, ng, cus);
  w.wide = wide_tile(rows, m, groups, ng, cus);
  w.plan = make_plan(m, groups, ng, cus);
  // 128 x 64 tiles for at most half of the units and k of 4096 or more: k split over two
  // workgroups per tile, which also share its adapters. 203 rows of a 4096 x 4096 product, 24
  // adapters of 64 ranks: 42 us in place of 49. (At half that k the second launch takes what the
  // split gains, and without adapters the bits are wkv7_proj_grouped's.)
  const int64_t tiles = count_tiles(m, groups, ng, kShapes[2]);
  int kmin = groups[0].k;
  for (int i = 1; i < ng; ++i) kmin = std::min(kmin, groups[i].k);
  if (!w.waves && !w.wide && w.plan.shape == 2 && w.plan.parts == 1 && 2 * tiles <= cus &&
      kmin >= 4096) {
    int64_t cols = 0;
    for (int i = 0; i < ng; ++i) cols += groups[i].n;
    w.plan.parts = 2;
    w.plan.ws_bytes = 2 * size_t(m) * size_t(cols) * sizeof(float);
  }
  for (int i = 0; i < ng; ++i) {
    w.h[i] = w.bytes;
    if (sets[i].a) w.bytes += align256(size_t(m) * sets[i].slabs * kParts * kSlab * sizeof(uint16_t));
  }
  w.partials = w.bytes;
  if (!w.waves && !w.wide) w.bytes += w.plan.ws_bytes;
  return w;
}

}  // namespace
}  // namespace wkv7

using namespace wkv7;

extern "C" int64_t wkv7_adapter_plan_ints(int64_t m, int32_t count) {
  if (!plan_fits(m, count)) return 0;
  return plan_part(positions(m, count), 3) + kTileInts * max_tiles(m, count);
}

extern "C" int wkv7_adapter_plan(const int32_t* ids, int64_t m, int32_t count, int32_t* plan,
                                 int64_t plan_ints) {
  if (!plan_fits(m, count) || !plan || (m > 0 && !ids)) return WKV7_ERR_ARG;
  if (plan_ints < wkv7_adapter_plan_ints(m, count)) return WKV7_ERR_WORKSPACE;
  // (a prompt's rows have one adapter, so rows are taken in runs of equal ids)
  auto run_end = [&](int64_t i) {
    const int32_t a = ids[i];
    while (++i < m && ids[i] == a) {}
    return i;
  };
  for (int64_t i = 0; i < m; i = run_end(i))
    if (ids[i] < -1 || ids[i] >= count) return WKV7_ERR_ARG;
  const int64_t all = positions(m, count);
  const int64_t align = m <= WKV7_ADAPTER_PACKED_ROWS ? 1 : kAlign;
  int32_t* order = plan;
  int32_t* id = plan + plan_part(all, 1);
  int32_t* end = plan + plan_part(all, 2);
  int32_t* tile = plan + plan_part(all, 3);
  int32_t* const last = tile + kTileInts * max_tiles(m, count);
  // Rows by adapter, in their own order within it, those without one last, at the end of the tiles'
  // place (the tiles of the rows before one, 20 ints for at most 16 rows or the rest of a run, end
  // before it): counted in the place of `end`, or sorted where there are more adapters than places.
  int32_t* const sorted = last - m;
  if (count < all) {
    std::fill(end, end + count + 1, 0);
    auto slot = [&](int64_t i) { return ids[i] < 0 ? count : ids[i]; };
    for (int64_t i = 0, e; i < m; i = e) {
      e = run_end(i);
      end[slot(i)] += int32_t(e - i);
    }
    int32_t at = 0;
    for (int32_t a = 0; a <= count; ++a) {
      const int32_t n = end[a];
      end[a] = at;
      at += n;
    }
    for (int64_t i = 0, e; i < m; i = e) {
      e = run_end(i);
      int32_t& at = end[slot(i)];
      std::iota(sorted + at, sorted + at + (e - i), int32_t(i));
      at += int32_t(e - i);
    }
  } else {
    for (int64_t i = 0; i < m; ++i) sorted[i] = int32_t(i);
    std::sort(sorted, sorted + m, [ids](int32_t x, int32_t y) {
      const uint32_t a = uint32_t(ids[x]), b = uint32_t(ids[y]);  // (-1 is the largest)
      return a != b ? a < b : x < y;
    });
  }
  auto gap = [&](int64_t from, int64_t to) {
    std::fill(order + from, order + to, -1);
    std::fill(id + from, id + to, -1);
    std::fill(end + from, end + to, int32_t(to));
  };
  int64_t p = 0;
  for (int64_t i = 0; i < m;) {
    const int32_t a = ids[sorted[i]];
    const int64_t first = (p + align - 1) / align * align;
    gap(p, first);
    for (p = first; i < m && ids[sorted[i]] == a; ++i) order[p++] = sorted[i];
    std::fill(id + first, id + p, a);
    std::fill(end + first, end + p, int32_t(p));
    for (int64_t f = first; a >= 0 && f < p; f += kSlab, tile += kTileInts) {
      const int64_t rows = std::min<int64_t>(kSlab, p - f);
      tile[0] = int32_t(f);
      tile[1] = int32_t(rows);
      tile[2] = a;
      tile[3] = 0;
      std::copy(order + f, order + f + rows, tile + 4);
      std::fill(tile + 4 + rows, tile + kTileInts, order[p - 1]);
    }
  }
  gap(p, all);
  std::fill(tile, last, 0);
  return WKV7_OK;
}

extern "C" int wkv7_adapter_load(const wkv7_adapter_set* set, int32_t index, int32_t n, int32_t k,
                                 const uint16_t* a, int64_t lda, const uint16_t* b, int64_t ldb,
                                 int32_t r, float scale, void* stream) {
  if (!set || !set->a || !set->b || !set->scale || !set->rank || !a || !b) return WKV7_ERR_ARG;
  if (index < 0 || index >= set->count || set->slabs < 1 ||
      set->slabs > WKV7_ADAPTER_MAX_RANK / kSlab || n < 1 || k < 32 || k % 32 || r < 1 ||
      r > set->slabs * kSlab)
    return WKV7_ERR_ARG;
  if (lda < k || ldb < r || !aligned16(set->a) || !aligned16(set->b)) return WKV7_ERR_SHAPE;
  const int64_t size_a = int64_t(kSlab) * set->slabs * k, size_b = int64_t(kSlab) * set->slabs * n;
  const int64_t a_blocks = (size_a + 2047) / 2048, b_blocks = (size_b + 2047) / 2048;
  if (a_blocks + b_blocks > 0x7fffffff) return WKV7_ERR_ARG;
  // (the set's pointers are the bank's own memory, which a launch of this kind may write)
  const LoadArgs args{a,
                      b,
                      const_cast<uint16_t*>(set->a) + index * size_a,
                      const_cast<uint16_t*>(set->b) + index * size_b,
                      const_cast<float*>(set->scale) + index,
                      const_cast<int32_t*>(set->rank) + index,
                      lda,
                      ldb,
                      scale,
                      r,
                      k,
                      n,
                      set->slabs,
                      int32_t(a_blocks)};
  adapter_load_kernel<<<unsigned(a_blocks + b_blocks), 256, 0, as_stream(stream)>>>(args);
  return launch_status();
}

extern "C" size_t wkv7_proj_adapters_workspace_bytes(int64_t m, const wkv7_proj_group* groups,
                                                     const wkv7_adapter_set* sets,
                                                     int32_t ngroups, int32_t count) {
  if (validate(m, groups, ngroups) != WKV7_OK || !sets || m == 0 || !plan_fits(m, count) ||
      check_sets(sets, ngroups, count) != WKV7_OK)
    return 0;
  int cus = 0;
  if (device_cus(&cus) != WKV7_OK) return 0;
  return make_work(m, positions(m, count), groups, sets, ngroups, cus).bytes;
}

extern "C" int wkv7_proj_adapters(int64_t m, const wkv7_proj_group* groups,
                                  const wkv7_adapter_set* sets, int32_t ngroups,
                                  const int32_t* plan, int32_t count, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  int rc = validate(m, groups, ngroups);
  if (rc != WKV7_OK) return rc;
  if (!sets || !plan_fits(m, count) || (m > 0 && !plan)) return WKV7_ERR_ARG;
  rc = check_sets(sets, ngroups, count);
  if (rc != WKV7_OK) return rc;
  if (m == 0) return WKV7_OK;
  if (!aligned16(plan)) return WKV7_ERR_SHAPE;
  int cus = 0;
  rc = device_cus(&cus);
  if (rc != WKV7_OK) return rc;
  const int64_t all = positions(m, count);
  const Work work = make_work(m, all, groups, sets, ngroups, cus);
  if (work.bytes && (!workspace || workspace_bytes < work.bytes || !aligned16(workspace)))
    return WKV7_ERR_WORKSPACE;
  char* ws = static_cast<char*>(workspace);
  hipStream_t s = as_stream(stream);

  Adapters ad{};
  ad.order = plan;
  ad.id = plan + plan_part(all, 1);
  ad.end = plan + plan_part(all, 2);
  ad.rows = m;
  ShrinkArgs sh{};
  sh.tiles = plan + plan_part(all, 3);
  sh.ntiles = int32_t(max_tiles(m, count));
  sh.m = m;
  sh.positions = all;
  sh.last = work.wide ? 1.f : 0.5f;
  int slabs = 0, kmax = 0;
  for (int i = 0; i < ngroups; ++i) {
    const wkv7_adapter_set& set = sets[i];
    if (!set.a) continue;
    uint16_t* h = reinterpret_cast<uint16_t*>(ws + work.h[i]);
    // (only the plan's own ids: a set may hold more adapters than the plan knows)
    sh.g[i] = {groups[i].x, set.a,          set.scale, set.rank, h,
               groups[i].ldx, groups[i].k, count,     set.slabs};
    ad.h[i] = h;
    ad.b[i] = set.b;
    ad.rank[i] = set.rank;
    ad.count[i] = count;
    ad.slabs[i] = set.slabs;
    slabs = std::max(slabs, set.slabs);
    kmax = std::max(kmax, groups[i].k);
  }
  if (slabs && count) {
    if (int64_t(sh.ntiles) * slabs * ngroups <= 8 * int64_t(cus)) {
      const dim3 grid(unsigned(sh.ntiles), unsigned(slabs), unsigned(ngroups));
      if (kmax <= 1024) shrink_thin_kernel<4><<<grid, 256, 0, s>>>(sh);
      else shrink_thin_kernel<8><<<grid, 512, 0, s>>>(sh);
    } else {
      const dim3 grid(unsigned((sh.ntiles + 1) / 2), unsigned(ngroups));
      shrink_wide_kernel<<<grid, 64 * kWideShrink, 0, s>>>(sh);
    }
    rc = launch_status();
    if (rc != WKV7_OK) return rc;
  }
  if (work.wide == 4) return launch_wide<4>(all, groups, ngroups, ad, s);
  if (work.wide == 2) return launch_wide<2>(all, groups, ngroups, ad, s);
  if (work.waves == 4) return launch_thin<4>(all, groups, ngroups, ad, s);
  if (work.waves == 8) return launch_thin<8>(all, groups, ngroups, ad, s);
  return launch_plan(all, groups, ngroups, work.plan, reinterpret_cast<float*>(ws + work.partials),
                     ad, s);
}
