// Products with 4-bit weights and group scales: y = act(x W^T + bias), W = s (c - z) with a scale and
// a zero point for each row and group of inputs, and the kernels that lay such weights out.
#include <algorithm>

#include "wkv7_w4_tile.h"

using namespace wkv7;

namespace wkv7 {
namespace {

struct W4Source {
  const uint8_t* codes;
  const void* scale;
  const uint8_t* zero;
  int scale_dtype;
  const uint16_t* w;  // or a bf16 weight to round
  int64_t ldw;
  bool symmetric;
};

// A thread per (row, eight inputs), 16 of them side by side over a block of 128: a group is 4, 8 or 16
// neighbouring lanes. Weights past n and k are zeros. (134 M codes in 59 us, 3.4 TB/s.)
__global__ __launch_bounds__(256) void w4_fill_kernel(const wkv7_w4_weight out, const W4Source src) {
  const int k = out.k, group = out.group;
  const int groups = (k + group - 1) / group, blocks = (k + kW4K - 1) / kW4K;
  const int64_t tile = int64_t(blockIdx.x) / blocks;
  const int block = int(int64_t(blockIdx.x) % blocks);
  const int li = threadIdx.x / 16, t = threadIdx.x % 16;
  const int64_t n = tile * kW4N + li;
  const int i0 = block * kW4K + 8 * t, gi = i0 / group;
  const bool real = n < out.n && i0 < k;
  uint32_t word = 0u, c[8] = {};
  if (src.w) {
    float v[8] = {}, lo = 0.f, hi = 0.f;
    for (int e = 0; e < 8 && real; ++e) {
      v[e] = bf16_to_f32(src.w[n * src.ldw + i0 + e]);
      lo = fminf(lo, v[e]);
      hi = fmaxf(hi, v[e]);
    }
    for (int d = 1; d < group / 8; d *= 2) {
      lo = fminf(lo, __shfl_xor(lo, d));
      hi = fmaxf(hi, __shfl_xor(hi, d));
    }
    // (halves: the range of finite weights may not be)
    const float range = src.symmetric ? fmaxf(-lo, hi) / 7.f : (0.5f * hi - 0.5f * lo) / 7.5f;
    word = __float_as_uint(range) & ~15u;
    const float s = w4_scale(word);
    const float z = src.symmetric ? 8.f : s > 0.f ? fminf(fmaxf(rintf(-lo / s), 0.f), 15.f) : 0.f;
    word |= uint32_t(z);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      c[e] = uint32_t(s > 0.f ? fminf(fmaxf(rintf(v[e] / s) + z, 0.f), 15.f) : z);
  } else if (real) {
    const int64_t at = n * groups + gi;
    const uint16_t bits = static_cast<const uint16_t*>(src.scale)[at];
    const float s = src.scale_dtype == WKV7_SCALE_BF16
                        ? bf16_to_f32(bits)
                        : float(__builtin_bit_cast(_Float16, bits));
    word = (__float_as_uint(s) & ~15u) | (src.zero ? src.zero[at] & 15u : 8u);
    const uint8_t* from = src.codes + n * k + i0;
    uint32_t two[2] = {};
    if (reinterpret_cast<uintptr_t>(src.codes) % 8 == 0) {
      const uint2 v = *reinterpret_cast<const uint2*>(from);
      two[0] = v.x;
      two[1] = v.y;
    } else {
      for (int e = 0; e < 8; ++e) two[e / 4] |= uint32_t(from[e]) << 8 * (e % 4);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) c[e] = two[e / 4] >> 8 * (e % 4) & 15u;
  }
  uint32_t bits = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int at = w4_bit(e);
    bits |= c[e] << at | (at > 28 ? c[e] >> (32 - at) : 0u);
  }
  const int lane = li + 16 * (t & 3);
  out.codes[((tile * blocks + block) * 64 + lane) * 4 + t / 4] = real ? bits : 0u;
  if (i0 % group == 0 && gi < groups)
    out.scales[(tile * groups + gi) * kW4N + li] = n < out.n ? word : 0u;
}

__global__ __launch_bounds__(256) void w4_unpack_kernel(const wkv7_w4_weight w, float* out) {
  const int64_t item = int64_t(blockIdx.x) * 256 + threadIdx.x;  // a word: eight codes
  const int k = w.k, words = k / 8;
  if (item >= int64_t(w.n) * words) return;
  const int64_t n = item / words;
  const int i0 = int(item % words) * 8;
  const int groups = (k + w.group - 1) / w.group, blocks = (k + kW4K - 1) / kW4K;
  const int lane = int(n % kW4N) + 16 * (i0 >> 3 & 3);
  const uint32_t bits = w.codes[(((n / kW4N) * blocks + i0 / kW4K) * 64 + lane) * 4 + (i0 >> 5 & 3)];
  const uint32_t word = w.scales[((n / kW4N) * groups + i0 / w.group) * kW4N + (n % kW4N)];
  for (int e = 0; e < 8; ++e)
    out[n * k + i0 + e] = w4_scale(word) * float(w4_code(bits, e) - w4_zero(word));
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int validate(const wkv7_w4_weight& w) {
  if (!w.codes || !w.scales || w.n < 1 || w.k < 32 || w.k % 32) return WKV7_ERR_ARG;
  if (w.group != 32 && w.group != 64 && w.group != 128) return WKV7_ERR_ARG;
  if (!aligned16(w.codes) || !aligned16(w.scales)) return WKV7_ERR_SHAPE;
  return WKV7_OK;
}

int validate(int64_t m, const wkv7_w4_group* groups, int32_t ngroups) {
  if (m < 0 || m > int64_t(0x7fffffff) || !groups || ngroups < 1 || ngroups > WKV7_PROJ_MAX_GROUPS)
    return WKV7_ERR_ARG;
  for (int i = 0; i < ngroups; ++i) {
    const wkv7_w4_group& g = groups[i];
    const int rc = validate(g.w);
    if (rc != WKV7_OK) return rc;
    if (!g.x || !g.y) return WKV7_ERR_ARG;
    if (g.act != WKV7_ACT_NONE && g.act != WKV7_ACT_TANH && g.act != WKV7_ACT_SIGMOID)
      return WKV7_ERR_ARG;
    if (g.ldx < g.w.k || g.ldy < g.w.n || g.ldx % 8 || !aligned16(g.x)) return WKV7_ERR_SHAPE;
  }
  return WKV7_OK;
}

int fill(const wkv7_w4_weight& w, const W4Source& src, void* stream) {
  const int64_t blocks = (int64_t(w.n) + kW4N - 1) / kW4N * ((w.k + kW4K - 1) / kW4K);
  if (blocks > int64_t(0x7fffffff)) return WKV7_ERR_ARG;
  w4_fill_kernel<<<unsigned(blocks), 256, 0, as_stream(stream)>>>(w, src);
  return launch_status();
}

// Workgroups of the products: one per column tile, or as many as the device holds at once
// (`slots`), dealt by their tiles.
int64_t deal(W4Args& a, int columns, int64_t slots) {
  int64_t tiles = 0;
  for (int i = 0; i < a.ngroups; ++i) tiles += (int64_t(a.g[i].w.n) + columns - 1) / columns;
  int64_t end = 0;
  for (int i = 0; i < a.ngroups; ++i) {
    const int64_t own = (int64_t(a.g[i].w.n) + columns - 1) / columns;
    end += tiles <= slots ? own : std::max<int64_t>(1, own * slots / tiles);
    a.wg_end[i] = int32_t(std::min<int64_t>(end, 0x7fffffff));
  }
  return end;
}

template <int KS>
int launch_thin(int64_t m, const wkv7_w4_group* groups, int n, int cus, hipStream_t s) {
  W4Args a{};
  a.m = m;
  int blocks = 0;
  for (int i = 0; i < n; ++i) {
    if (groups[i].w.group != 32 * KS) continue;
    a.g[a.ngroups++] = groups[i];
    blocks = std::max(blocks, (groups[i].w.k + kW4K - 1) / kW4K);
  }
  if (a.ngroups == 0) return WKV7_OK;
  // A unit holds two workgroups of 8 waves or one of 16 (three products of 4096 x 4096: one row 10.1
  // us in 8 waves of two blocks, twice; 9.5 in 16. 16 rows 20.3 and 14.1). Groups of 32 have too many
  // scales and sums in registers for two blocks at once (12.6 us with one, 22.9 in 16 waves of two).
  const bool wide = blocks > 16 && KS > 1;
  const int64_t wgs = deal(a, kW4N, (wide ? 1 : 2) * int64_t(cus));
  if (wgs > int64_t(0x7fffffff)) return WKV7_ERR_ARG;
  if constexpr (KS > 1) {
    if (wide) w4_thin_kernel<16, 2, KS><<<unsigned(wgs), 1024, 0, s>>>(a);
    else if (blocks > 8) w4_thin_kernel<8, 2, KS><<<unsigned(wgs), 512, 0, s>>>(a);
    if (blocks > 8) return launch_status();
  }
  w4_thin_kernel<8, 1, KS><<<unsigned(wgs), 512, 0, s>>>(a);
  return launch_status();
}

template <int TN, int KS>
int launch_mid(W4Args& a, int cus, hipStream_t s) {
  const int row_tiles = int((a.m + 31) / 32);
  int64_t end = 0;
  for (int i = 0; i < a.ngroups; ++i) {
    end += (int64_t(a.g[i].w.n) + 32 * TN - 1) / (32 * TN) * row_tiles;
    if (end > int64_t(0x7ffffff0)) return WKV7_ERR_ARG;
    a.wg_end[i] = int32_t(end);
  }
  const int span = int((end + kW4Xcds - 1) / kW4Xcds);
  // Eight waves fill a unit, or four twice where there are more tiles than units (three products of 4096
  // x 4096: 32 rows 11.9 us in eight, 13.8 in four; 64 rows 21.3 and 18.8).
  if constexpr (TN == 2 || KS == 1) {  // (else there are at most as many tiles as units)
    if (end > cus) {
      w4_mid_kernel<4, TN, KS><<<unsigned(span) * kW4Xcds, 256, 0, s>>>(a, row_tiles, span);
      return launch_status();
    }
  }
  w4_mid_kernel<8, TN, KS><<<unsigned(span) * kW4Xcds, 512, 0, s>>>(a, row_tiles, span);
  return launch_status();
}

template <int KS>
int launch_mid(int64_t m, const wkv7_w4_group* groups, int n, int cus, hipStream_t s) {
  W4Args a{};
  a.m = m;
  int64_t tiles = 0;
  for (int i = 0; i < n; ++i) {
    if (groups[i].w.group != 32 * KS) continue;
    a.g[a.ngroups++] = groups[i];
    tiles += (int64_t(groups[i].w.n) + 31) / 32 * ((m + 31) / 32);
  }
  if (a.ngroups == 0) return WKV7_OK;
  // 64 columns, which share the reads of x, as soon as 32 would be more tiles than units (three
  // products of 2048 x 2048, 32 rows 6.6 us in 32 columns, 8.1 in 64; 64 rows 9.3 and 8.4). Not for
  // groups of 32, whose sums and scales do not fit the registers then.
  if constexpr (KS > 1) {
    if (tiles > cus) return launch_mid<2, KS>(a, cus, s);
  }
  return launch_mid<1, KS>(a, cus, s);
}

int device_cus(int* cus) {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess ||
      hipDeviceGetAttribute(cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess)
    return launch_status();
  return WKV7_OK;
}

// Which kernel runs. us for three products of 2048 x 2048 (4096 x 4096, one of 65536 x 2048):
//   thin and mid kernel: 1 row 5.0 and 5.9 (9.5 and 10.5, 15.6 and 24.2), 4 rows 5.9 both (11.8 and 10.6,
//   19 and 24), 16 rows 7.8 and 6.1 (14.0 and 10.7, 21 and 25)
//   mid kernel and output tiles, with the sums before them: 128 rows 12.8 and 15.0 (28.9 and 26.8), 192
//   rows 18.9 and 15.6; one product of 2048 x 2048, 256 rows 8.3 and 13.9, 512 rows 12.5 and 14.4
// So a few rows go to the mid kernel where its tiles (32 rows x 64 columns) are one a unit, and many
// where they are two. With more tiles and k past what the thin kernel holds of x at once, it reads x
// again for each: 32768 x 8192, 1 row 37 us (the mid kernel 33), 16 rows 71 (32).
enum class W4Kernel { kThin, kMid, kTiles };
W4Kernel choose(int64_t m, const wkv7_w4_group* groups, int n, int cus) {
  int64_t tiles = 0;
  int k = 0;
  for (int i = 0; i < n; ++i) {
    tiles += (int64_t(groups[i].w.n) + 63) / 64 * ((m + 31) / 32);
    k = std::max(k, groups[i].w.k);
  }
  if (m <= (tiles <= cus ? 3 : k <= 4096 ? 16 : 0)) return W4Kernel::kThin;
  return m <= WKV7_W4_NO_WORKSPACE_ROWS || tiles <= 2 * int64_t(cus) ? W4Kernel::kMid
                                                                     : W4Kernel::kTiles;
}

// Workspace of the tile kernel: the sums of every product's x over its groups.
size_t sums_bytes(int64_t m, const wkv7_w4_group& g) {
  return size_t(m + 31) / 32 * 32 * 3 * w4_padded_groups(g.w.k, g.w.group) * sizeof(uint16_t);
}

size_t workspace_bytes_of(int64_t m, const wkv7_w4_group* groups, int n) {
  if (m <= WKV7_W4_NO_WORKSPACE_ROWS) return 0;
  size_t bytes = 0;
  for (int i = 0; i < n; ++i) bytes += sums_bytes(m, groups[i]);
  return bytes;
}

int64_t count_tiles(const W4TileArgs& a, int bm, int bn) {
  int64_t tiles = 0;
  for (int i = 0; i < a.ngroups; ++i)
    tiles += (a.m + bm - 1) / bm * ((int64_t(a.g[i].w.n) + bn - 1) / bn);
  return tiles;
}

template <int GM, int GN, int TM, int TN, int KH, int S, int KS>
int launch_tiles(W4TileArgs& a, hipStream_t s) {
  constexpr int BM = 32 * TM * GM, BN = 32 * TN * GN;
  int64_t end = 0;
  for (int i = 0; i < a.ngroups; ++i) {
    end += (a.m + BM - 1) / BM * ((int64_t(a.g[i].w.n) + BN - 1) / BN);
    if (end > int64_t(0x7ffffff0)) return WKV7_ERR_ARG;
    a.tile_end[i] = int32_t(end);
  }
  a.span = int32_t((end + kW4Xcds - 1) / kW4Xcds);
  w4_tile_kernel<GM, GN, TM, TN, KH, S, KS>
      <<<unsigned(a.span) * kW4Xcds, 64 * GM * GN * KH, 0, s>>>(a);
  return launch_status();
}

// The products of groups of 32 KS inputs: sums of x, then output tiles.
template <int KS>
int launch_tiled(int64_t m, const wkv7_w4_group* groups, int n, uint16_t*& ws, int cus,
                 hipStream_t s) {
  W4SumArgs sums{};
  W4TileArgs tiles{};
  sums.m = tiles.m = m;
  int64_t waves = 0;
  int distinct = 0;
  for (int i = 0; i < n; ++i) {
    const wkv7_w4_group& g = groups[i];
    if (g.w.group != 32 * KS) continue;
    const int at = tiles.ngroups++;
    tiles.g[at] = g;
    int same = 0;  // products of one x share its sums
    while (same < distinct &&
           (sums.x[same] != g.x || sums.ldx[same] != g.ldx || sums.k[same] != g.w.k))
      ++same;
    if (same == distinct) {
      sums.sums[distinct] = ws;
      sums.x[distinct] = g.x;
      sums.ldx[distinct] = g.ldx;
      sums.k[distinct++] = g.w.k;
      waves = std::max(waves, (m + 31) / 32 * 32 *
                                  ((w4_padded_groups(g.w.k, 32 * KS) * 32 * KS + 511) / 512));
      ws += sums_bytes(m, g) / sizeof(uint16_t);
    }
    tiles.sums[at] = sums.sums[same];
  }
  if (tiles.ngroups == 0) return WKV7_OK;
  if ((waves + 3) / 4 > int64_t(0x7fffffff)) return WKV7_ERR_ARG;
  w4_sums_kernel<KS><<<dim3(unsigned((waves + 3) / 4), distinct), 256, 0, s>>>(sums);
  const int rc = launch_status();
  if (rc != WKV7_OK) return rc;
  // Four waves side by side, two workgroups on a unit, but for the second shape, of eight waves that
  // take turns in k. us with the sums, three products of 2048 x 2048 (4096 x 4096) by rows, in tiles of
  // 32 x 128, of 64 x 128 in two parts, of 64 x 128 and of 64 x 256:
  //   128 rows 15.5, 15.0, 18.5, 22.7 (30.7, 26.9, 31.6, 43.4)
  //   256 rows 19.6, 17.3, 19.7, 25.3 (45.6, 48.0, 44.2, 46.7)
  //   1024 rows 46.9, 44.7, 42.9, 40.9 (164, 152, 143, 119); 4096 rows (610, 567, 510, 420)
  // The parts' workgroups fill a unit, and a launch of 256 of them leaves some units with two and some
  // with none (36 us, and 22 for 224 of the same length).
  const int64_t tiles64 = count_tiles(tiles, 64, 128);
  if (8 * tiles64 <= 7 * int64_t(cus)) return launch_tiles<1, 4, 2, 1, 2, 2, KS>(tiles, s);
  if (count_tiles(tiles, 64, 256) > cus) return launch_tiles<1, 4, 2, 2, 1, 2, KS>(tiles, s);
  // An odd number of tiles of 32 rows, without the last half of a tile of 64 (two products of 8960 x
  // 1536, 96 rows: 18.2 us and 21.6).
  if (count_tiles(tiles, 32, 128) < 2 * tiles64) return launch_tiles<1, 4, 1, 1, 1, 3, KS>(tiles, s);
  return launch_tiles<1, 4, 2, 1, 1, 3, KS>(tiles, s);
}

}  // namespace
}  // namespace wkv7

extern "C" size_t wkv7_w4_code_bytes(int32_t n, int32_t k) {
  if (n < 1 || k < 1) return 0;
  return (size_t(n) + kW4N - 1) / kW4N * ((size_t(k) + kW4K - 1) / kW4K) * 1024;
}

extern "C" size_t wkv7_w4_scale_bytes(int32_t n, int32_t k, int32_t group) {
  if (n < 1 || k < 1 || group < 1) return 0;
  return (size_t(n) + kW4N - 1) / kW4N * ((size_t(k) + group - 1) / group) * (kW4N * 4);
}

extern "C" int wkv7_w4_pack(const wkv7_w4_weight* weight, const uint8_t* codes, const void* scale,
                            int32_t scale_dtype, const uint8_t* zero, void* stream) {
  if (!weight || !codes || !scale) return WKV7_ERR_ARG;
  if (scale_dtype != WKV7_SCALE_BF16 && scale_dtype != WKV7_SCALE_F16) return WKV7_ERR_ARG;
  const int rc = validate(*weight);
  if (rc != WKV7_OK) return rc;
  if (reinterpret_cast<uintptr_t>(scale) & 1u) return WKV7_ERR_SHAPE;
  return fill(*weight, W4Source{codes, scale, zero, scale_dtype, nullptr, 0, false}, stream);
}

extern "C" int wkv7_w4_quantize(const wkv7_w4_weight* weight, const uint16_t* w, int64_t ldw,
                                int32_t symmetric, void* stream) {
  if (!weight || !w) return WKV7_ERR_ARG;
  const int rc = validate(*weight);
  if (rc != WKV7_OK) return rc;
  if (ldw < weight->k || (reinterpret_cast<uintptr_t>(w) & 1u)) return WKV7_ERR_SHAPE;
  return fill(*weight, W4Source{nullptr, nullptr, nullptr, 0, w, ldw, symmetric != 0}, stream);
}

extern "C" int wkv7_w4_unpack(const wkv7_w4_weight* weight, float* w, void* stream) {
  if (!weight || !w) return WKV7_ERR_ARG;
  const int rc = validate(*weight);
  if (rc != WKV7_OK) return rc;
  if (reinterpret_cast<uintptr_t>(w) & 3u) return WKV7_ERR_SHAPE;
  const int64_t blocks = (int64_t(weight->n) * (weight->k / 8) + 255) / 256;
  if (blocks > int64_t(0x7fffffff)) return WKV7_ERR_ARG;
  w4_unpack_kernel<<<unsigned(blocks), 256, 0, as_stream(stream)>>>(*weight, w);
  return launch_status();
}

extern "C" size_t wkv7_proj_w4_workspace_bytes(int64_t m, const wkv7_w4_group* groups,
                                               int32_t ngroups) {
  return validate(m, groups, ngroups) == WKV7_OK ? workspace_bytes_of(m, groups, ngroups) : 0;
}

extern "C" int wkv7_proj_w4(int64_t m, const wkv7_w4_group* groups, int32_t ngroups,
                            void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = validate(m, groups, ngroups);
  if (rc != WKV7_OK) return rc;
  if (m == 0) return WKV7_OK;
  hipStream_t st = as_stream(stream);
  if (m > WKV7_W4_NO_WORKSPACE_ROWS) {
    if (!workspace || workspace_bytes < workspace_bytes_of(m, groups, ngroups))
      return WKV7_ERR_WORKSPACE;
    if (!aligned16(workspace)) return WKV7_ERR_SHAPE;
  }
  int cus = 0;
  int done = device_cus(&cus);
  if (done != WKV7_OK) return done;
  switch (choose(m, groups, ngroups, cus)) {
    case W4Kernel::kThin:
      done = launch_thin<4>(m, groups, ngroups, cus, st);
      if (done == WKV7_OK) done = launch_thin<2>(m, groups, ngroups, cus, st);
      if (done == WKV7_OK) done = launch_thin<1>(m, groups, ngroups, cus, st);
      return done;
    case W4Kernel::kMid:
      done = launch_mid<4>(m, groups, ngroups, cus, st);
      if (done == WKV7_OK) done = launch_mid<2>(m, groups, ngroups, cus, st);
      if (done == WKV7_OK) done = launch_mid<1>(m, groups, ngroups, cus, st);
      return done;
    case W4Kernel::kTiles: break;
  }
  uint16_t* ws = static_cast<uint16_t*>(workspace);
  done = launch_tiled<4>(m, groups, ngroups, ws, cus, st);
  if (done == WKV7_OK) done = launch_tiled<2>(m, groups, ngroups, ws, cus, st);
  if (done == WKV7_OK) done = launch_tiled<1>(m, groups, ngroups, ws, cus, st);
  return done;
}
