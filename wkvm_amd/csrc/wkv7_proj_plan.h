// Launches of the projection kernels: argument checks, the choice of a tile shape and of a k split.
#pragma once

#include <algorithm>

#include "wkv7_proj_core.h"

namespace wkv7 {
namespace {

struct TileShape {
  int bm, bn;
};

// Tile shapes (fewer re-reads of x and w per output the larger the tile);
// measured on the MI355X inside HIP graphs.
constexpr TileShape kShapes[] = {{64, 64}, {32, 32}, {128, 64}, {64, 32}};

int64_t count_tiles(int64_t m, const wkv7_proj_group* gs, int ng, TileShape sh) {
  int64_t tiles = 0;
  const int64_t tm = (m + sh.bm - 1) / sh.bm;
  for (int i = 0; i < ng; ++i) tiles += tm * ((gs[i].n + sh.bn - 1) / sh.bn);
  return tiles;
}

// kSplits: plans split k over workgroups for this shape.
template <int BM, int BN, int S, int GM, int GN, int BK, bool kSplits, class Extra>
int launch(int64_t m, const wkv7_proj_group* gs, int ng, int parts, float* ws, const Extra& ex,
           hipStream_t s) {
  ProjArgs args{};
  args.m = m;
  args.ngroups = ng;
  args.parts = parts;
  args.ws = ws;
  const int64_t tiles_m = (m + BM - 1) / BM;
  int64_t end = 0, elems = 0;
  for (int i = 0; i < ng; ++i) {
    args.g[i] = gs[i];
    end += tiles_m * ((gs[i].n + BN - 1) / BN) * parts;
    if (end > int64_t(0x7fffffff)) return WKV7_ERR_ARG;
    args.tile_end[i] = int32_t(end);
    args.ws_off[i] = elems * parts;
    elems += m * gs[i].n;
    args.elem_end[i] = elems;
  }
  args.tiles_m = int32_t(tiles_m);
  args.xcd_span = int32_t((end + kXcds - 1) / kXcds);
  const unsigned grid = unsigned(args.xcd_span) * kXcds;
  if constexpr (kSplits) {
    if (parts > 1) {
      const int64_t blocks = (elems + 255) / 256;
      if (blocks > int64_t(0x7fffffff)) return WKV7_ERR_ARG;
      proj_kernel<BM, BN, S, GM, GN, BK, true><<<grid, 64 * GM * GN, 0, s>>>(args, ex);
      const int rc = launch_status();
      if (rc != WKV7_OK) return rc;
      proj_reduce_kernel<<<unsigned(blocks), 256, 0, s>>>(args, ex);
      return launch_status();
    }
  }
  proj_kernel<BM, BN, S, GM, GN, BK, false><<<grid, 64 * GM * GN, 0, s>>>(args, ex);
  return launch_status();
}

template <int NW, class Extra>
int launch_thin(int64_t m, const wkv7_proj_group* gs, int ng, const Extra& ex, hipStream_t s) {
  ProjArgs args{};
  args.m = m;
  args.ngroups = ng;
  int64_t end = 0;
  for (int i = 0; i < ng; ++i) {
    args.g[i] = gs[i];
    end += (int64_t(gs[i].n) + 15) / 16;
    if (end > int64_t(0x7fffffff)) return WKV7_ERR_ARG;
    args.tile_end[i] = int32_t(end);
  }
  proj_thin_kernel<NW><<<unsigned(end), 64 * NW, 0, s>>>(args, ex);
  return launch_status();
}

// Tile shape and k split for a launch (the same decision for the workspace
// query and the launch).
struct Plan {
  int shape;  // index into kShapes
  int parts;  // k parts per tile
  size_t ws_bytes;
};

// One row tile: the thin kernel for few column tiles, where it has no second
// launch, and for short k. Not for many column tiles of long k: every one
// re-reads all of x (1.5B first stage of 16 rows, 407 workgroups, 12.2 us
// against 9.4 in 32 x 32 tiles; o_proj of the 7B shape, 256, 12.2 against 13.5).
// Its waves: 8 for long k, 4 where k has few chunks (LoRA up-projections of the
// 7B shape 5.2 against 6.4 us).
constexpr int kThinShortK = 512;

int thin_waves(int64_t m, const wkv7_proj_group* gs, int ng, int cus) {
  if (m > WKV7_PROJ_FEW_ROWS) return 0;
  int kmax = 0;
  for (int i = 0; i < ng; ++i) kmax = std::max(kmax, gs[i].k);
  if (kmax <= kThinShortK) return 4;
  return count_tiles(m, gs, ng, kShapes[1]) * 2 <= int64_t(cus) ? 8 : 0;
}

// The plan of the tiled kernel. At 16 rows or fewer the thin one runs in its
// place wherever it would split k (at most half a tile per unit of long k), so
// the workspace is never used there.
Plan make_plan(int64_t m, const wkv7_proj_group* gs, int ng, int cus) {
  int kmin = gs[0].k;
  int64_t cols = 0;
  for (int i = 0; i < ng; ++i) {
    kmin = std::min(kmin, gs[i].k);
    cols += gs[i].n;
  }
  // The launch reads (BM + BN) rows of k per tile from L2, which bounds it
  // at a few hundred rows. With long k, the shape whose rounds over the
  // compute units take least; us per round, measured at k = 2048 (128 x 64: 16
  // waves, 3-stage ring of 128-wide k stages, 144 KiB of LDS, one workgroup per
  // unit; 64 x 32: 8 waves, 4-stage ring, 96 KiB, one; 32 x 32: 4 waves,
  // 4-stage ring, 64 KiB, two). The 1.5B first stage: 8 rows 8.1 us in 32 x 32
  // tiles (9.3 in 64 x 32 with 4 waves), 64 rows 9.3 in 64 x 32 (10.3), 256 rows
  // 18.6 in 128 x 64 (19.6 with 8 waves), 512 rows 33.9 (39.5 in 64 x 64);
  // o_proj at 256 rows 9.1 (9.8 with 4 waves), at 512 rows 14.1 (17.0 in 32 x 32).
  // With short k the prologue counts as much as the stages: 64 x 64 tiles (8
  // waves, 2-stage ring) as soon as every unit gets one (LoRA up-projections at
  // 128 rows 5.2 against 7.1 us), else 32 x 32.
  Plan p{1, 1, 0};
  int64_t tiles = count_tiles(m, gs, ng, kShapes[1]);
  const int64_t units = std::max(cus, 1);
  auto rounds = [](int64_t t, int64_t slots) { return double((t + slots - 1) / slots); };
  if (kmin >= 1024) {
    double best = tiles <= units ? 8.2 : 9.6 * rounds(tiles, 2 * units);
    const struct { int shape; double us; } wide[] = {{3, 9.1}, {2, 16.5}};
    for (const auto& w : wide) {
      const int64_t t = count_tiles(m, gs, ng, kShapes[w.shape]);
      const double us = w.us * rounds(t, units);
      if (us < best) {
        best = us;
        p.shape = w.shape;
      }
    }
    tiles = count_tiles(m, gs, ng, kShapes[p.shape]);
  } else if (count_tiles(m, gs, ng, kShapes[0]) >= units) {
    p.shape = 0;
    tiles = count_tiles(m, gs, ng, kShapes[0]);
  }
  // 32 x 32 tiles for at most half of the units and long k: split k so that about two
  // workgroups per unit each walk at least 8 stages. (With more tiles the
  // partials' extra traffic and second launch cost more than they save.)
  const int nk = (kmin + 63) / 64;
  if (p.shape == 1 && tiles * 2 <= int64_t(cus) && nk >= 16) {
    int64_t parts = (2 * int64_t(cus) + tiles / 2) / tiles;
    parts = std::min<int64_t>(parts, std::min(8, nk / 8));
    if (parts >= 2) {
      p.parts = int(parts);
      p.ws_bytes = size_t(parts) * size_t(m) * size_t(cols) * sizeof(float);
    }
  }
  return p;
}

template <class Extra>
int launch_plan(int64_t m, const wkv7_proj_group* gs, int ng, const Plan& p, float* ws,
                const Extra& ex, hipStream_t s) {
  // (128 x 64 tiles are split only with adapters)
  if (p.shape == 0) return launch<64, 64, 2, 2, 4, 128, false>(m, gs, ng, p.parts, ws, ex, s);
  if (p.shape == 2) return launch<128, 64, 3, 8, 2, 128, Extra::kOn>(m, gs, ng, p.parts, ws, ex, s);
  if (p.shape == 3) return launch<64, 32, 4, 4, 2, 128, false>(m, gs, ng, p.parts, ws, ex, s);
  return launch<32, 32, 4, 2, 2, 128, true>(m, gs, ng, p.parts, ws, ex, s);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int validate(int64_t m, const wkv7_proj_group* groups, int32_t ngroups) {
  if (m < 0 || !groups || ngroups < 1 || ngroups > WKV7_PROJ_MAX_GROUPS) return WKV7_ERR_ARG;
  if (m > int64_t(0x7fffffff)) return WKV7_ERR_ARG;
  for (int i = 0; i < ngroups; ++i) {
    const wkv7_proj_group& g = groups[i];
    if (!g.x || !g.w || !g.y || g.n < 1 || g.k < 32 || g.k % 32 != 0) return WKV7_ERR_ARG;
    if (g.act != WKV7_ACT_NONE && g.act != WKV7_ACT_TANH && g.act != WKV7_ACT_SIGMOID)
      return WKV7_ERR_ARG;
    if (g.ldx < g.k || g.ldw < g.k || g.ldy < g.n) return WKV7_ERR_SHAPE;
    if (g.ldx % 8 || g.ldw % 8 || !aligned16(g.x) || !aligned16(g.w)) return WKV7_ERR_SHAPE;
  }
  return WKV7_OK;
}

int device_cus(int* cus) {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess ||
      hipDeviceGetAttribute(cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess)
    return launch_status();
  return WKV7_OK;
}

}  // namespace
}  // namespace wkv7
