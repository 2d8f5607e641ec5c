// Sampling of each row's next token by temperature, top-k, top-p and min-p, from
// given random numbers, with the token's log-probability.
//
// With M = max x, w_i = exp((x_i - M) / T) and the order "larger logit first, ties
// by lower index", every filter keeps a prefix of that order: top-k its first k
// tokens, top-p the shortest prefix whose weight reaches p of what top-k left,
// min-p the tokens with w_i >= min_p. So the kept set is one cut in the order,
// a pair (key, index), and rarely more than a few hundred tokens are near it.
//
// Two launches. The scan, a wave per 2,048 tokens, reads the logits once and leaves
// sums, group weights and the maxima of runs of 32 tokens; the finish, a workgroup
// per row, reads again only the runs that can hold kept tokens, sorts those, and
// draws. Where top-p's share reaches far down it goes over the row twice more: once
// for a histogram of the weights, once for the tokens of the bin that the cut is in.
// One workgroup per row for all of it would leave a lone row on one unit (161 us for
// 65,536 logits with every filter, 20 now). 256 rows of 65,536 fp32 logits in a HIP
// graph: temperature alone 22.9 us (2.9 TB/s; the scan by itself 4.1), greedy 20.4, min-p
// 0.05 23.1, top-k 50 and top-p 0.95 28, top-p 0.95 alone 57.4, rows of mixed settings 48.7,
// top-k 5,000 (more than there are runs: radix passes over the whole row) 139.
//
// The draw is an exponential race in two levels: with positive exponential variates
// e, group j of 256 consecutive tokens arrives at e / W_j (W_j the kept weight in it)
// and the first arrival wins with probability W_j / W; the tokens of that group
// race the same way. A row needs 256 + V / 256 variates instead of V, and
// the outcome depends on ratios of the two earliest arrivals, which rounding
// disturbs in about one row of 10^6; a uniform through the cumulated sum would fall
// across one of its V borders thousands of times as often.
//
// Weights that are added in an order that varies (LDS atomics) are fixed-point
// numbers, of 42 fraction bits (w <= 1) or, in the histogram of a whole row, of 31 bits
// of the weight where the token's bins start: the sums are exact and the token does not
// depend on the order. Plain sums are fp32 per thread, joined in a fixed order.
#include "wkv7_common.h"

namespace wkv7 {
namespace {

typedef unsigned long long u64;

constexpr int kGroup = WKV7_SAMPLE_GROUP;
constexpr int kChunk = 2048;              // tokens of one wave of the scan
constexpr int kSub = 32;                  // tokens whose maximum the scan keeps
constexpr int kChunkSubs = kChunk / kSub;
constexpr int kChunkGroups = kChunk / kGroup;
constexpr int kScanThreads = 256;

constexpr int kThreads = 512;             // of the finish: two workgroups share a unit
constexpr int kWaves = kThreads / kWave;
constexpr int kBins = 2048;
constexpr int kList = 4096;               // candidates held in LDS
constexpr int kSubs = 4096;               // runs of kSub tokens that may hold candidates
constexpr int kFarBins = 8192;            // of a whole row's weights
// The candidate list's group weights take the place of the histogram.
constexpr int kListGroups = kBins + kBins / 2;

struct SampleArgs {
  const void* logits;
  int64_t stride;
  const float* noise;
  int64_t noise_stride;
  const float *temperature, *top_p, *min_p;  // per row, or NULL: the value below
  const int32_t* top_k;
  float temperature1, top_p1, min_p1;
  int32_t top_k1;
  int32_t V, rows, chunks;
  int32_t* tokens;
  float* logprobs;
  // what the scan leaves for the finish, per row
  float* sub_max;   // [chunks * kChunkSubs]
  float* mass;      // [chunks * kChunkGroups]: group weights relative to the chunk's maximum
  float2* chunk;    // [chunks]: maximum, sum of exp(x - maximum)
};

struct Settings {
  float c;        // log2(e) / temperature
  float top_p;
  float floor_z;  // min-p: the least (x - M) c
  int32_t top_k;
  bool greedy, by_k, by_p;
};

__device__ __forceinline__ Settings settings(const SampleArgs& a, int64_t b) {
  const float temp = a.temperature ? a.temperature[b] : a.temperature1;
  const float min_p = a.min_p ? a.min_p[b] : a.min_p1;
  Settings s;
  s.top_p = a.top_p ? a.top_p[b] : a.top_p1;
  s.top_k = a.top_k ? a.top_k[b] : a.top_k1;
  // the clamp keeps c and every product a number
  s.c = 1.44269504088896340736f / fminf(fmaxf(temp, 0x1p-60f), 0x1p60f);
  s.floor_z = min_p > 0.f ? log2f(fminf(min_p, 1.f)) : -INFINITY;
  s.greedy = !(temp > 0.f);
  s.by_k = s.top_k > 0 && s.top_k < a.V;
  s.by_p = s.top_p < 1.f;
  return s;
}

// Ascending in the order of the tokens: the largest logit has the smallest key.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);  // (-0 and +0 are equal)
  return (u >> 31) ? u : ~u & 0x7fffffffu;
}
__device__ __forceinline__ float key_logit(uint32_t k) {
  return __uint_as_float((k >> 31) ? k : ~k & 0x7fffffffu);
}

// NaN counts as -inf, +inf as the largest finite number.
__device__ __forceinline__ float clean(float x) {
  return fminf(fmaxf(x, -INFINITY), 3.402823466e38f);
}

__device__ __forceinline__ float load_one(const float* p) { return clean(*p); }
__device__ __forceinline__ float load_one(const uint16_t* p) { return clean(bf16_to_f32(*p)); }

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// 42 fraction bits of w in [0, 2^22).
__device__ __forceinline__ u64 fixed(float w) {
  const float hi = w * 0x1p10f;
  return u64(uint32_t(hi)) << 32 | uint32_t(__builtin_amdgcn_fractf(hi) * 0x1p32f);
}

// Lane exchanges inside 16 lanes; after the smaller steps the mirrors act as xor 4 and xor 8.
constexpr int kXor1 = 0xb1, kXor2 = 0x4e, kXor4 = 0x141, kXor8 = 0x140;
template <int kCtrl>
__device__ __forceinline__ float dpp(float v) {
  return __uint_as_float(__builtin_amdgcn_update_dpp(0u, __float_as_uint(v), kCtrl, 0xf, 0xf, true));
}

__device__ __forceinline__ float wave_max(float v) {
  v = fmaxf(v, dpp<kXor1>(v));
  v = fmaxf(v, dpp<kXor2>(v));
  v = fmaxf(v, dpp<kXor4>(v));
  v = fmaxf(v, dpp<kXor8>(v));
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
// The sum over the 2^kLog lanes around a lane.
template <int kLog>
__device__ __forceinline__ float lanes_sum(float v) {
  v += dpp<kXor1>(v);
  v += dpp<kXor2>(v);
  v += dpp<kXor4>(v);
  if constexpr (kLog > 3) v += dpp<kXor8>(v);
  if constexpr (kLog > 4) v += __shfl_xor(v, 16);
  if constexpr (kLog > 5) v += __shfl_xor(v, 32);
  return v;
}

// Elements of one 16-byte load, as they lie in memory.
template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr int N = 4;
  typedef float Raw __attribute__((ext_vector_type(4), aligned(4)));
  Raw x;
  __device__ __forceinline__ float raw(int e) const { return x[e]; }
  __device__ __forceinline__ float get(int e) const { return clean(raw(e)); }
};
template <> struct Vec<uint16_t> {
  static constexpr int N = 8;
  typedef uint32_t Raw __attribute__((ext_vector_type(4), aligned(2)));
  Raw x;
  __device__ __forceinline__ float raw(int e) const {
    return (e & 1) ? bf16_hi(x[e / 2]) : bf16_lo(x[e / 2]);
  }
  __device__ __forceinline__ float get(int e) const { return clean(raw(e)); }
};

template <typename T>
__device__ __forceinline__ Vec<T> load_full(const T* p) {
  return {*reinterpret_cast<const typename Vec<T>::Raw*>(p)};
}
// The vector at element i of a row of n; elements past the end are -inf.
template <typename T>
__device__ __forceinline__ Vec<T> load_part(const T* row, int i, int n) {
  if (i + Vec<T>::N <= n) return load_full(row + i);
  Vec<T> v;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (sizeof(T) == 4) {
      v.x[e] = i + e < n ? row[i + e] : -INFINITY;
    } else {
      const uint32_t lo = i + 2 * e < n ? row[i + 2 * e] : 0xff80u;
      const uint32_t hi = i + 2 * e + 1 < n ? row[i + 2 * e + 1] : 0xff80u;
      v.x[e] = lo | hi << 16;
    }
  }
  return v;
}

// -- the scan: one wave per chunk of 2,048 tokens, one pass over the logits -----------------------

// Bound by the one pass over the logits: 256 rows of 65,536 fp32 logits 15.6 us (4.3 TB/s, where a
// large copy reaches 4.8), 512 rows of 131,077 in bf16 34 us (4.0 TB/s, with half of that time's
// instructions in the two exponentials per logit).
//
// Of every chunk: its maximum and sum of exponentials; of every 32 tokens the maximum, for the
// finish to know where the largest logits are; and, where no filter applies or top-p alone needs the
// row's weight, the weight of every group. Everything is relative to the chunk's own
// maximum, so the chunks need nothing of each other.
template <typename T>
__global__ __launch_bounds__(kScanThreads) void sample_scan_kernel(const SampleArgs args) {
  constexpr int N = Vec<T>::N;
  constexpr int kSteps = kChunk / (kWave * N);
  constexpr int kSubLanes = kSub / N;      // 8 or 4 lanes hold 32 tokens
  constexpr int kGroupLanes = kGroup / N;  // 64 or 32 lanes hold a group
  const int64_t id = int64_t(blockIdx.x) * (kScanThreads / kWave) +
                     __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  if (id >= int64_t(args.rows) * args.chunks) return;
  const int64_t b = id / args.chunks;
  const int first = int(id - b * args.chunks) * kChunk;
  const int lane = threadIdx.x & (kWave - 1);
  const int V = args.V;
  const T* row = static_cast<const T*>(args.logits) + b * args.stride;
  Vec<T> v[kSteps];
  if (first + kChunk <= V) {
#pragma unroll
    for (int j = 0; j < kSteps; ++j) v[j] = load_full(row + first + (j * kWave + lane) * N);
  } else {
#pragma unroll
    for (int j = 0; j < kSteps; ++j) v[j] = load_part(row, first + (j * kWave + lane) * N, V);
  }
  const Settings set = settings(args, b);
  float x[kSteps][N];
  float top = -INFINITY;
  float* sub = args.sub_max + id * kChunkSubs;
#pragma unroll
  for (int j = 0; j < kSteps; ++j) {
    float m = -INFINITY;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      x[j][e] = v[j].get(e);
      m = fmaxf(m, x[j][e]);
    }
    top = fmaxf(top, m);
    m = fmaxf(m, dpp<kXor1>(m));
    m = fmaxf(m, dpp<kXor2>(m));
    if constexpr (kSubLanes == 8) m = fmaxf(m, dpp<kXor4>(m));
    if (lane % kSubLanes == 0) sub[(j * kWave + lane) / kSubLanes] = m;
  }
  top = wave_max(top);
  float raw = 0.f;
  // (a chunk of nothing but -inf: its sums stay zero)
  const float base = top == -INFINITY ? 0.f : top;
  if (args.logprobs) {
    const float c = 1.44269504088896340736f;
#pragma unroll
    for (int j = 0; j < kSteps; ++j)
#pragma unroll
      for (int e = 0; e < N; ++e) raw += exp2_hw((x[j][e] - base) * c);
    raw = lanes_sum<6>(raw);
  }
  if (lane == 0) args.chunk[id] = make_float2(top, raw);
  // group weights: for the race where no filter applies, and for top-p's total
  if (set.greedy || set.by_k || (!set.by_p && set.floor_z > -INFINITY)) return;
  float w[kSteps];
#pragma unroll
  for (int j = 0; j < kSteps; ++j) {
    w[j] = 0.f;
#pragma unroll
    for (int e = 0; e < N; ++e) w[j] += exp2_hw((x[j][e] - base) * set.c);
  }
  float* mass = args.mass + id * kChunkGroups;
#pragma unroll
  for (int j = 0; j < kSteps; ++j) {
    const float s = kGroupLanes == 64 ? lanes_sum<6>(w[j]) : lanes_sum<5>(w[j]);
    if (lane % kGroupLanes == 0) mass[(j * kWave + lane) / kGroupLanes] = s;
  }
}

// -- the finish: one workgroup per row ----------------------------------------------------------------
//
// A chain of short steps with a barrier after each, so latency bounds it: about 5 us where nothing is
// cut off, 12 for top-k 40 (sums 2, histogram of run maxima 4, gathering 2, order 2, race 2) and 16
// for top-k 200. A top-p that reaches far down (65,536 fp32 logits: 32 us for a row) is bound by the
// work per token of its two passes: about 12 us for the histogram, 7 for the bin's tokens. Workgroups of
// 512 threads, two of which share a unit, so that one works while the other waits. Tried and slower:
// fp32 LDS atomics, and bins of each thread's own, for the histograms.

struct Found {
  uint32_t bin, before_cnt, cnt;
  u64 before_wgt, wgt;
};

struct alignas(16) Shared {
  union {
    struct {
      u64 wgt[kBins];
      uint32_t cnt[kBins];
      uint2 list[kList];  // logit bits, index
      uint16_t subs[kSubs];
    };
    u64 mass[kListGroups];           // takes the place of the histogram
    u64 far[kFarBins + kWave];       // the last 64 take what is in no bin, each from one lane
    float row_mass[WKV7_SAMPLE_MAX_VOCAB / kGroup];
  };
  uint32_t n_list, n_subs;
  Found found;
  u64 first;
  u64 red[kWaves];
  uint32_t wave_cnt[kWaves];
  u64 wave_wgt[kWaves];
};

struct MaxF { __device__ float operator()(float a, float b) const { return fmaxf(a, b); } };
struct AddD { __device__ double operator()(double a, double b) const { return a + b; } };
struct AddU { __device__ u64 operator()(u64 a, u64 b) const { return a + b; } };
struct MinU { __device__ u64 operator()(u64 a, u64 b) const { return a < b ? a : b; } };

// Reduction over the block; every thread gets the result.
template <typename V, typename Op>
__device__ __forceinline__ V block_all(V v, Op op, Shared& sm) {
  static_assert(sizeof(V) <= sizeof(u64), "fits a slot");
  V* slot = reinterpret_cast<V*>(sm.red);
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) v = op(v, __shfl_xor(v, o));
  __syncthreads();
  if ((threadIdx.x & (kWave - 1)) == 0) slot[threadIdx.x / kWave] = v;
  __syncthreads();
  V r = slot[threadIdx.x & (kWaves - 1)];
#pragma unroll
  for (int o = 1; o < kWaves; o <<= 1) r = op(r, __shfl_xor(r, o));
  return r;
}

// An arrival time (not negative) with its index: the smaller time wins, then the lower index.
__device__ __forceinline__ u64 arrival(float t, uint32_t i) {
  return (u64(__float_as_uint(t)) << 32) | i;
}

// A row that every pass reads again: f(logit, index) for the tokens of this thread.
template <typename T>
struct Row {
  static constexpr int N = Vec<T>::N;
  static constexpr int kStep = kThreads * N;
  const T* p;
  int n;

  // f(vector, index of its first element); every thread makes the same calls. The next U vectors
  // are under way while f works on U. The one that the row may end in is read apart: the code of
  // its guarded loads is long, and a workgroup runs through most of the kernel's code once.
  template <typename F>
  __device__ __forceinline__ void vectors(F f) const {
    constexpr int U = 4;
    const int i = int(threadIdx.x) * N, whole = n / kStep * kStep;
    Vec<T> v[U], w[U], last;
    auto fetch = [&](Vec<T>(&to)[U], int at) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (at + u * kStep < whole) to[u] = load_full(p + at + u * kStep + i);
    };
    if (whole < n) last = load_part(p, whole + i, n);
    fetch(v, 0);
    for (int at = 0; at < whole; at += U * kStep) {
      fetch(w, at + U * kStep);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (at + u * kStep < whole) f(v[u], at + u * kStep + i);
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = w[u];
    }
    if (whole < n) f(last, whole + i);
  }
  template <typename F>
  __device__ __forceinline__ void operator()(F f) const {
    vectors([&](const Vec<T>& x, int i) {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (i + e < n) f(x.get(e), uint32_t(i + e));
    });
  }
};

struct ListRow {
  const Shared& sm;
  uint32_t n;
  template <typename F>
  __device__ __forceinline__ void operator()(F f) const {
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
      const uint2 c = sm.list[i];
      f(__uint_as_float(c.x), c.y);
    }
  }
};

__device__ __forceinline__ void clear_bins(Shared& sm) {
  __syncthreads();
  for (int i = threadIdx.x; i < kBins; i += kThreads) {
    sm.cnt[i] = 0;
    sm.wgt[i] = 0;
  }
  __syncthreads();
}

// Inclusive sums over the block, in thread order.
__device__ __forceinline__ void block_scan(uint32_t& c, u64& w, uint32_t& all_c, u64& all_w,
                                           Shared& sm) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const uint32_t cu = __shfl_up(c, o);
    const u64 wu = __shfl_up(w, o);
    if (lane >= o) {
      c += cu;
      w += wu;
    }
  }
  __syncthreads();
  if (lane == kWave - 1) {
    sm.wave_cnt[wave] = c;
    sm.wave_wgt[wave] = w;
  }
  __syncthreads();
  all_c = 0;
  all_w = 0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    if (i < wave) {
      c += sm.wave_cnt[i];
      w += sm.wave_wgt[i];
    }
    all_c += sm.wave_cnt[i];
    all_w += sm.wave_wgt[i];
  }
}

// The bin in which the cumulated count (or weight) reaches target >= 1; the last bin that
// holds anything where it never does.
__device__ __forceinline__ Found find_bin(Shared& sm, bool by_weight, u64 target) {
  constexpr int kEach = kBins / kThreads;
  const int t = threadIdx.x;
  __syncthreads();
  uint32_t c[kEach], cb = 0, all_c;
  u64 w[kEach], wb = 0, all_w;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    c[i] = sm.cnt[kEach * t + i];
    w[i] = sm.wgt[kEach * t + i];
    cb += c[i];
    wb += w[i];
  }
  const uint32_t mine_c = cb;
  const u64 mine_w = wb;
  block_scan(cb, wb, all_c, all_w, sm);
  cb -= mine_c;  // before this thread's bins
  wb -= mine_w;
  const u64 goal = min(target, by_weight ? all_w : u64(all_c));
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const u64 before = by_weight ? wb : u64(cb), here = by_weight ? w[i] : u64(c[i]);
    if (before < goal && before + here >= goal)
      sm.found = {uint32_t(kEach * t + i), cb, c[i], wb, w[i]};
    cb += c[i];
    wb += w[i];
  }
  __syncthreads();
  return sm.found;
}

// The same over the far bins, which hold weights alone: kFarEach neighbouring bins in 31 fraction bits
// of what a token at the start of the first of them weighs, 2^-(width * that bin) of the largest.
constexpr int kFarEach = kFarBins / kThreads;

__device__ __forceinline__ Found find_far(Shared& sm, float width, u64 target) {
  const int t = threadIdx.x;
  __syncthreads();
  uint32_t none = 0, all_c;
  u64 mine = 0, all_w;
  // (each lane starts at another bin of its own, lest they all read the same banks)
#pragma unroll
  for (int i = 0; i < kFarEach; ++i) mine += sm.far[kFarEach * t + (i + t) % kFarEach];
  const float unit = exp2_hw(fmaf(-width, float(kFarEach * t), -31.f));
  auto weight = [unit](u64 sum) {
    return fixed(fmaf(float(uint32_t(sum >> 32)), 0x1p32f, float(uint32_t(sum))) * unit);
  };
  mine = weight(mine);
  u64 before = mine;
  block_scan(none, before, all_c, all_w, sm);
  before -= mine;
  const u64 goal = min(target, all_w);
  if (before < goal && before + mine >= goal) {
    uint32_t bin = kFarEach * t;
    u64 sum = sm.far[bin], upto = 0;
    for (; before + weight(sum) < goal; sum += sm.far[++bin]) upto = sum;
    sm.found = {bin, 0, 0, before + weight(upto), weight(sum) - weight(upto)};
  }
  __syncthreads();
  return sm.found;
}

// A cut in the order: what lies before it or on it is kept.
struct Cut {
  uint32_t key, index;
  float x;  // the key's logit
  __device__ __forceinline__ Cut(uint32_t k, uint32_t i) : key(k), index(i), x(key_logit(k)) {}
  __device__ __forceinline__ bool keeps(float v, uint32_t i) const {
    return v > x || (v == x && i <= index);
  }
};

// The cut after the tokens whose count (or weight) reaches target, among those of `rows`
// that pred takes; `upto` gets the weight up to it (where weights are wanted).
template <typename Rows, typename Pred, typename Weight>
__device__ __forceinline__ Cut descend(const Rows& rows, Pred pred, Weight weight, bool want_weight,
                                    bool by_weight, u64 target, u64* upto, Shared& sm) {
  uint32_t prefix = 0, before_cnt = 0;
  u64 before_wgt = 0;
  Found f{};
#pragma unroll 1
  for (int level = 0; level < 3; ++level) {
    const int shift = level == 0 ? 21 : level == 1 ? 10 : 0;
    const uint32_t mask = level == 2 ? 1023u : 2047u;
    const int above = level == 0 ? 32 : level == 1 ? 21 : 10;
    clear_bins(sm);
    rows([&](float x, uint32_t i) {
      if (!pred(x, i)) return;
      const uint32_t k = order_key(x);
      if (level && (k >> above) != prefix) return;
      const uint32_t b = (k >> shift) & mask;
      atomicAdd(&sm.cnt[b], 1u);
      if (want_weight) atomicAdd(&sm.wgt[b], fixed(weight(x)));
    });
    f = find_bin(sm, by_weight, target - (by_weight ? before_wgt : u64(before_cnt)));
    before_cnt += f.before_cnt;
    before_wgt += f.before_wgt;
    prefix = level == 0 ? f.bin : (prefix << (level == 1 ? 11 : 10)) | f.bin;
  }
  // f.cnt tokens share the key: how many of them belong before the cut
  const u64 each = f.cnt ? f.wgt / f.cnt : 0;
  const u64 rest = target - (by_weight ? before_wgt : u64(before_cnt));
  u64 ties = by_weight ? (each ? (rest + each - 1) / each : 1) : rest;
  ties = max(u64(1), min(ties, u64(f.cnt)));
  if (upto) *upto = before_wgt + ties * each;
  Cut cut(prefix, 0xffffffffu);
  if (ties >= f.cnt) return cut;
  // the lowest `ties` indices among them
  uint32_t before = 0, high = 0;
#pragma unroll 1
  for (int level = 0; level < 2; ++level) {
    clear_bins(sm);
    rows([&](float x, uint32_t i) {
      if (!pred(x, i) || order_key(x) != cut.key) return;
      if (level && (i >> 11) != high) return;
      atomicAdd(&sm.cnt[level ? i & 2047u : i >> 11], 1u);
    });
    f = find_bin(sm, false, ties - before);
    before += f.before_cnt;
    if (level == 0) high = f.bin;
  }
  cut.index = high << 11 | f.bin;
  return cut;
}

// Top-k's and top-p's cut among the tokens of `rows`. `total`: the weight that top-p's share is
// of, where top-k does not give it.
template <typename Rows, typename Weight>
__device__ __forceinline__ Cut cut_rows(const Rows& rows, const Settings& set, double total,
                                        Weight weight, Shared& sm) {
  Cut cut(order_key(-INFINITY), 0xffffffffu);
  if (set.by_k) {
    u64 upto = 0;
    cut = descend(rows, [](float, uint32_t) { return true; }, weight, set.by_p, false,
                  u64(set.top_k), &upto, sm);
    total = double(upto) * 0x1p-42;
  }
  if (set.by_p) {
    const Cut outer = cut;
    const u64 target = max(u64(1), u64(ceil(fmax(double(set.top_p), 0.) * total * 0x1p42)));
    cut = descend(rows, [outer](float x, uint32_t i) { return outer.keeps(x, i); }, weight, true,
                  true, target, static_cast<u64*>(nullptr), sm);
    // (all of a key's tokens: all that top-k left of them)
    if (cut.key == outer.key) cut.index = min(cut.index, outer.index);
  }
  return cut;
}

// The race over the candidates that `kept` takes.
template <typename Kept, typename Weight>
__device__ __forceinline__ uint32_t race_list(const ListRow& rows, Kept kept, Weight weight,
                                              const float* noise, int groups, Shared& sm) {
  __syncthreads();
  for (int g = threadIdx.x; g < groups; g += kThreads) sm.mass[g] = 0;
  __syncthreads();
  rows([&](float x, uint32_t i) {
    if (kept(x, i)) atomicAdd(&sm.mass[i / kGroup], fixed(weight(x)));
  });
  __syncthreads();
  u64 best = ~0ull;
  for (int g = threadIdx.x; g < groups; g += kThreads)
    if (sm.mass[g]) best = min(best, arrival(noise[kGroup + g] / float(sm.mass[g]), uint32_t(g)));
  const uint32_t group = uint32_t(block_all(best, MinU(), sm));
  best = ~0ull;
  rows([&](float x, uint32_t i) {
    if (i / kGroup == group && kept(x, i))
      best = min(best, arrival(noise[i % kGroup] / weight(x), i));
  });
  return uint32_t(block_all(best, MinU(), sm));
}

// The race inside a group, over the tokens that `kept` takes.
template <typename T, typename Kept, typename Weight>
__device__ __forceinline__ uint32_t race_group(const Row<T>& row, uint32_t group, Kept kept,
                                               Weight weight, const float* noise, Shared& sm) {
  u64 best = ~0ull;
  const int i = int(min(group, uint32_t(row.n - 1) / kGroup)) * kGroup + int(threadIdx.x);
  if (threadIdx.x < kGroup && i < row.n) {
    const float x = load_one(row.p + i);
    if (kept(x, uint32_t(i))) best = arrival(noise[threadIdx.x] / weight(x), uint32_t(i));
  }
  return uint32_t(block_all(best, MinU(), sm));
}

// The race over the whole row. A group is the vectors of 256 / N neighbouring lanes; its weight
// goes through LDS, so that the variates are read in one go.
template <typename T, typename Kept, typename Weight>
__device__ __forceinline__ uint32_t race_row(const Row<T>& row, Kept kept, Weight weight,
                                             const float* noise, Shared& sm) {
  constexpr int kLanes = kGroup / Vec<T>::N;
  const int groups = (row.n + kGroup - 1) / kGroup;
  __syncthreads();
  row.vectors([&](const Vec<T>& x, int i) {
    float w = 0.f;
#pragma unroll
    for (int e = 0; e < Vec<T>::N; ++e) {
      const float v = x.get(e);
      w += kept(v, uint32_t(i + e)) ? weight(v) : 0.f;
    }
    w = kLanes == 64 ? lanes_sum<6>(w) : lanes_sum<5>(w);
    if ((threadIdx.x & (kLanes - 1)) == 0 && i < row.n) sm.row_mass[i / kGroup] = w;
  });
  __syncthreads();
  u64 best = ~0ull;
  for (int g = threadIdx.x; g < groups; g += kThreads) {
    const float w = sm.row_mass[g];
    if (w > 0.f) best = min(best, arrival(noise[kGroup + g] / w, uint32_t(g)));
  }
  const uint32_t group = uint32_t(block_all(best, MinU(), sm));
  return race_group(row, group, kept, weight, noise, sm);
}

// The same where the scan has left the groups' whole weights: a group's first arrival is no earlier
// than its whole weight says, so only groups that could still be first are looked at, in place of
// the whole row: about as many as the row weighs more than what is kept. Every wave has its own
// share of the groups; what one of them has found ends the others.
template <typename T, typename Kept, typename Weight, typename Whole>
__device__ __forceinline__ uint32_t race_bounded(const Row<T>& row, Kept kept, Weight weight,
                                                 Whole whole, const float* noise, Shared& sm) {
  const int groups = (row.n + kGroup - 1) / kGroup;
  const int lane = threadIdx.x & (kWave - 1);
  u64 best = ~0ull, seen = 0;
  __syncthreads();
  if (threadIdx.x == 0) sm.first = ~0ull;
  __syncthreads();
#pragma unroll 1
  for (;;) {
    u64 next = ~0ull;  // the earliest possible arrival that has not been looked at
    for (int g = threadIdx.x; g < groups; g += kThreads) {
      const float w = whole(g) * (1.f + 0x1p-12f);  // (more than the two sums' rounding)
      if (!(w > 0.f)) continue;
      const u64 a = arrival(noise[kGroup + g] / w, uint32_t(g)) + 1;
      if (a > seen) next = min(next, a);
    }
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) next = min(next, __shfl_xor(next, o));
    if (next >= __hip_atomic_load(&sm.first, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP)) break;
    seen = next;
    const uint32_t g = uint32_t(next - 1);
    float w = 0.f;
#pragma unroll
    for (int e = 0; e < kGroup / kWave; ++e) {
      const int i = int(g) * kGroup + e * kWave + lane;
      const float x = i < row.n ? load_one(row.p + i) : -INFINITY;
      w += kept(x, uint32_t(i)) ? weight(x) : 0.f;
    }
    w = lanes_sum<6>(w);
    if (!(w > 0.f)) continue;
    best = min(best, arrival(noise[kGroup + g] / w, g));
    if (lane == 0) atomicMin(&sm.first, best);
  }
  const uint32_t group = uint32_t(block_all(best, MinU(), sm));
  return race_group(row, group, kept, weight, noise, sm);
}

// The candidates of the list (at most one per thread) in order: thread t gets the t-th key, then its
// index, ~0 past the end. Each counts the keys before its own, which all lanes of a wave read at
// once: n steps that wait for nothing, where the barriers and lane exchanges of a sorting network
// took 5 us for 41 keys and 9 for 210 (so 2 and 3.7, with the sums after it).
__device__ __forceinline__ u64 sorted_candidate(uint32_t n, Shared& sm) {
  static_assert(2 * kThreads <= kBins, "keys, and keys in order");
  constexpr int kAtOnce = 16;  // (past n they are ~0, up to kThreads)
  const uint32_t t = threadIdx.x;
  u64 v = ~0ull;
  if (t < n) v = u64(order_key(__uint_as_float(sm.list[t].x))) << 32 | sm.list[t].y;
  __syncthreads();
  sm.wgt[t] = v;
  __syncthreads();
  if (__builtin_amdgcn_readfirstlane(t) < n) {
    uint32_t before = 0;
    for (uint32_t j = 0; j < n; j += kAtOnce) {
      ulonglong2 k[kAtOnce / 2];
#pragma unroll
      for (int i = 0; i < kAtOnce / 2; ++i)
        k[i] = reinterpret_cast<const ulonglong2*>(sm.wgt + j)[i];
#pragma unroll
      for (int i = 0; i < kAtOnce / 2; ++i) before += (k[i].x < v) + (k[i].y < v);
    }
    if (t < n) sm.wgt[kThreads + before] = v;
  }
  __syncthreads();
  return t < n ? sm.wgt[kThreads + t] : ~0ull;
}

// Candidates: every token whose logit `takes` accepts (a condition that holds for every larger
// logit too), found through the maxima of the runs of 32 tokens. False where they are too many.
template <typename T, typename Takes>
__device__ __forceinline__ bool gather(const Row<T>& row, const float* sub_max, int n_sub,
                                       Takes takes, Shared& sm) {
  constexpr int N = Vec<T>::N, kLanes = kSub / N;
  __syncthreads();
  if (threadIdx.x == 0) sm.n_list = sm.n_subs = 0;
  __syncthreads();
  for (int s = threadIdx.x; s < n_sub; s += kThreads) {
    if (takes(sub_max[s])) {
      const uint32_t at = atomicAdd(&sm.n_subs, 1u);
      if (at < kSubs) sm.subs[at] = uint16_t(s);
    }
  }
  __syncthreads();
  const uint32_t n = sm.n_subs;
  if (n > kSubs) return false;
  for (uint32_t at = threadIdx.x / kLanes; at < n; at += kThreads / kLanes) {
    const int i = int(sm.subs[at]) * kSub + int(threadIdx.x % kLanes) * N;
    const Vec<T> v = load_part(row.p, i, row.n);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float x = v.get(e);
      if (i + e < row.n && takes(x)) {
        const uint32_t to = atomicAdd(&sm.n_list, 1u);
        if (to < kList) sm.list[to] = make_uint2(__float_as_uint(x), uint32_t(i + e));
      }
    }
  }
  __syncthreads();
  return sm.n_list <= kList;
}

template <typename T>
__global__ __launch_bounds__(kThreads, 4) void sample_finish_kernel(const SampleArgs args) {
  __shared__ Shared sm;
  const int64_t b = blockIdx.x;
  const int t = threadIdx.x, V = args.V, chunks = args.chunks;
  const Row<T> row{static_cast<const T*>(args.logits) + b * args.stride, V};
  const float* noise = args.noise + b * args.noise_stride;
  const Settings set = settings(args, b);
  const float2* chunk = args.chunk + b * chunks;
  const float* sub_max = args.sub_max + b * chunks * kChunkSubs;
  const float* mass = args.mass + b * chunks * kChunkGroups;
  const int groups = (V + kGroup - 1) / kGroup, n_sub = (V + kSub - 1) / kSub;

  float m = -INFINITY;
  for (int i = t; i < chunks; i += kThreads) m = fmaxf(m, chunk[i].x);
  const float top = block_all(m, MaxF(), sm);
  if (top == -INFINITY) {  // nothing to choose from
    if (t == 0) {
      args.tokens[b] = -1;
      if (args.logprobs) args.logprobs[b] = -INFINITY;
    }
    return;
  }
  auto weight = [top, c = set.c](float x) { return exp2_hw((x - top) * c); };
  auto over_floor = [top, c = set.c, z = set.floor_z](float x) { return (x - top) * c >= z; };
  double raw = 0.;
  if (args.logprobs) {
    for (int i = t; i < chunks; i += kThreads) {
      const float2 h = chunk[i];
      raw += double(h.y) * double(exp2_hw((h.x - top) * 1.44269504088896340736f));
    }
    raw = block_all(raw, AddD(), sm);
  }
  // a group's weight relative to the row's maximum
  auto group_weight = [&](int g) {
    return mass[g] * exp2_hw((chunk[g / kChunkGroups].x - top) * set.c);
  };

  uint32_t token;
  if (set.greedy) {
    u64 best = ~0ull;  // the first run that holds the maximum, and the first such token in it
    for (int s = t; s < n_sub; s += kThreads)
      if (sub_max[s] == top) best = min(best, u64(s));
    const int i = int(block_all(best, MinU(), sm)) * kSub + t;
    best = t < kSub && i < V && load_one(row.p + i) == top ? u64(i) : ~0ull;
    token = uint32_t(block_all(best, MinU(), sm));
  } else if (!set.by_k && !set.by_p && set.floor_z == -INFINITY) {
    u64 best = ~0ull;
    for (int g = t; g < groups; g += kThreads) {
      const float w = group_weight(g);
      if (w > 0.f) best = min(best, arrival(noise[kGroup + g] / w, uint32_t(g)));
    }
    const uint32_t group = uint32_t(block_all(best, MinU(), sm));
    token = race_group(row, group, [](float, uint32_t) { return true; }, weight, noise, sm);
  } else {
    double total = 0.;
    if (set.by_p && !set.by_k) {
      for (int g = t; g < groups; g += kThreads) total += double(group_weight(g));
      total = block_all(total, AddD(), sm);
    }
    const u64 share = max(u64(1), u64(ceil(fmax(double(set.top_p), 0.) * total * 0x1p42)));
    // Every token that top-p keeps of all weighs more than (1 - p) / V of the row: those that weigh
    // less add up to less than 1 - p. In log2 of the weight:
    const float rest_of = (1.f - fmaxf(set.top_p, 0.f)) * float(total) / float(V);
    const float low = fminf(log2f(fmaxf(rest_of, 0x1p-80f)), 0.f) - 0.01f;
    bool done = false;
    if (groups > kListGroups) {
      // (no room for the candidates' group weights)
    } else if (!set.by_k && !set.by_p) {
      if (gather(row, sub_max, n_sub, over_floor, sm)) {
        token = race_list(ListRow{sm, sm.n_list}, [](float, uint32_t) { return true; }, weight,
                          noise, groups, sm);
        done = true;
      }
    } else {
      // Distance from the maximum in 2,048 steps: the histogram of the run maxima says from which
      // step on there are enough tokens, for the maxima alone are that many, or weigh that much.
      // For top-k the steps are 1/128 of a logit or, where the last one would hold its end,
      // coarser; for top-p alone they end where its tokens end. min-p may thin the candidates
      // only where top-p's share does not count them.
      const bool thin = !set.by_p;
      float scale = set.by_k ? 128.f * fminf(set.c, 1.f) : float(kBins - 1) / -low * set.c;
      uint32_t last = kBins - 1;
      bool enough = set.by_k && set.top_k > n_sub;  // (more tokens than runs: all of them)
      for (int j = 0; !enough && j < 5; ++j, scale *= 0.0625f) {
        clear_bins(sm);
        for (int s = t; s < n_sub; s += kThreads) {
          const float x = sub_max[s];
          const int bin = int(fminf((top - x) * scale, float(kBins - 1)));
          if (bin == kBins - 1) continue;  // (too far, and most of the runs of a steep row)
          atomicAdd(&sm.cnt[bin], 1u);
          if (!set.by_k) atomicAdd(&sm.wgt[bin], fixed(weight(x)));
        }
        const Found f = find_bin(sm, !set.by_k, set.by_k ? u64(set.top_k) : share);
        enough = set.by_k ? f.before_cnt + f.cnt >= uint32_t(set.top_k)
                          : f.before_wgt + f.wgt >= share;
        last = enough ? f.bin : kBins - 1;
        if (enough || !set.by_k) break;
      }
      // (top-k among tokens of the last step of the coarsest scale: every token is a candidate)
      if (set.by_k) enough = true;
      if (V <= kList && !enough) {
        enough = true;
        last = kBins - 1;
      }
      if (enough && gather(row, sub_max, n_sub, [=](float x) {
            return uint32_t(fminf((top - x) * scale, float(kBins - 1))) <= last &&
                   (!thin || over_floor(x));
          }, sm)) {
        const uint32_t n = sm.n_list;
        done = true;
        if (n <= kThreads) {
          const uint64_t limit = set.by_k ? uint64_t(set.top_k) : ~0ull;
          const u64 v = sorted_candidate(n, sm);
          const float x = key_logit(uint32_t(v >> 32));
          const bool mine = uint32_t(t) < n && uint64_t(t) < limit;
          const u64 w = mine ? fixed(weight(x)) : 0;
          u64 upto = w, all;
          uint32_t one = 0, none;
          block_scan(one, upto, none, all, sm);
          const u64 target =
              set.by_k ? max(u64(1), u64(ceil(fmax(double(set.top_p), 0.) * double(all)))) : share;
          const bool kept = mine && (t == 0 || !set.by_p || upto - w < target);
          if (kept) sm.list[t] = make_uint2(__float_as_uint(x), uint32_t(v));
          const ListRow first{sm, uint32_t(__syncthreads_count(kept))};
          token = race_list(first, [=](float x, uint32_t) { return over_floor(x); }, weight,
                            noise, groups, sm);
        } else {
          const ListRow rows{sm, n};
          const Cut cut = cut_rows(rows, set, total, weight, sm);
          token = race_list(rows, [=](float x, uint32_t i) {
            return cut.keeps(x, i) && over_floor(x); }, weight, noise, groups, sm);
        }
      }
    }
    // (a row with +inf in it, whose distance to the largest finite number is negative, is left to
    // the last resort)
    if (!done && set.by_p && !set.by_k && top < 3.402823466e38f) {
      // Top-p's share reaches far down: a pass over 8,192 bins of its tokens' range in log weight
      // leaves one short run of the order to look at closely. What bounds the pass is the work per
      // token, half instructions and half LDS atomics; the bins are many lest the run be long (2,048
      // of them, and a branch per token: 256 rows of mixed settings 63 us where this took 53). A
      // token adds its weight relative to its bins' start, to 2^-31 of itself, so that many tokens of
      // one weight, or a tail far below 2^-32 of the largest, count as what they are (42 bits of the
      // largest in place of that: 512 rows of 131,077 118.6 us, 116.1 so).
      const float width = fmaxf(-low, 1.f) / float(kFarBins);  // of a bin, in log2
      const float steps = set.c / width;                       // bins per logit
      constexpr float kRun = kFarEach;                         // bins of one start
      __syncthreads();
      for (int i = t; i < kFarBins; i += kThreads) sm.far[i] = 0;
      __syncthreads();
      row.vectors([&](const Vec<T>& v, int) {
        constexpr int N = Vec<T>::N;
        uint32_t bin[N], w[N];
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float r = (top - v.raw(e)) * (steps / kRun), d = r * kRun;
          const bool in = d < float(kFarBins);  // (not NaN, nor -inf past the row's end)
          const float rel = exp2_hw(-kRun * width * __builtin_amdgcn_fractf(r));
          w[e] = in ? uint32_t(fmaf(rel, 0x1p31f, 0.5f)) : 0u;
          bin[e] = in ? uint32_t(d) : kFarBins + (threadIdx.x & (kWave - 1));
          // (in straight lines: a branch per token leaves nothing to do while one waits)
          asm volatile("" : "+v"(w[e]), "+v"(bin[e]));
        }
#pragma unroll
        for (int e = 0; e < N; ++e) atomicAdd(&sm.far[bin[e]], u64(w[e]));
      });
      const Found f = find_far(sm, width, share);
      if (t == 0) sm.n_list = 0;
      __syncthreads();
      // The bin's tokens: first those in a range of logits that surely holds the bin (d is within
      // 0.01 of the exact quotient, the range's ends within 2^-21 of top's and their own size); of
      // them the others become -inf.
      const float down = top - (float(f.bin) + 1.02f) / steps;
      const float up = top - (float(f.bin) - 0.02f) / steps;
      const float slack = (fabsf(top) + fabsf(down)) * 0x1p-21f;
      const float least = down - slack, most = up + slack;
      row.vectors([&](const Vec<T>& v, int i) {
        uint32_t in = 0;
#pragma unroll
        for (int e = 0; e < Vec<T>::N; ++e)
          in |= ((v.raw(e) >= least) & (v.raw(e) <= most)) ? 1u << e : 0u;
        for (; in; in &= in - 1) {
          const uint32_t to = atomicAdd(&sm.n_list, 1u);
          if (to < kList) sm.list[to].y = uint32_t(i + __builtin_ctz(in));
        }
      });
      __syncthreads();
      for (uint32_t i = t; i < min(sm.n_list, uint32_t(kList)); i += kThreads) {
        const uint32_t token = sm.list[i].y;
        const float x = token < uint32_t(V) ? load_one(row.p + token) : -INFINITY;
        const float d = (top - x) * (steps / kRun) * kRun;
        const bool in = d < float(kFarBins) && uint32_t(d) == f.bin;
        sm.list[i].x = __float_as_uint(in ? x : -INFINITY);
      }
      __syncthreads();
      const uint32_t n = sm.n_list;
      if (n > 0 && n <= kList) {
        const u64 rest = share > f.before_wgt ? share - f.before_wgt : 1;
        Cut cut(0u, 0u);
        if (n <= kThreads) {
          const u64 v = sorted_candidate(n, sm);
          const u64 w = uint32_t(t) < n ? fixed(weight(key_logit(uint32_t(v >> 32)))) : 0;
          u64 upto = w, all;
          uint32_t one = 0, none;
          block_scan(one, upto, none, all, sm);
          // the last token that still begins before the share is reached
          const bool kept = uint32_t(t) < n && v >> 32 != order_key(-INFINITY) &&
                            (t == 0 || upto - w < rest);
          const int last = __syncthreads_count(kept) - 1;
          if (t == max(last, 0)) sm.red[0] = v;
          __syncthreads();
          cut = Cut(uint32_t(sm.red[0] >> 32), uint32_t(sm.red[0]));
          __syncthreads();
        } else {
          cut = descend(ListRow{sm, n}, [](float x, uint32_t) { return x > -INFINITY; }, weight,
                        true, true, rest, static_cast<u64*>(nullptr), sm);
        }
        auto kept = [=](float x, uint32_t i) { return cut.keeps(x, i) && over_floor(x); };
        token = set.floor_z > -INFINITY  // (which may leave little of what the groups weigh)
                    ? race_row(row, kept, weight, noise, sm)
                    : race_bounded(row, kept, weight, group_weight, noise, sm);
        done = true;
      }
    }
    if (!done) {
      const Cut cut = cut_rows(row, set, total, weight, sm);
      token = race_row(row, [=](float x, uint32_t i) {
        return cut.keeps(x, i) && over_floor(x); }, weight, noise, sm);
    }
  }
  if (t == 0) {
    token = min(token, uint32_t(V - 1));  // (whatever the variates are)
    args.tokens[b] = int32_t(token);
    if (args.logprobs)
      args.logprobs[b] = float(double(load_one(row.p + token) - top) - log(raw));
  }
}

size_t align256(size_t n) { return (n + 255) & ~size_t(255); }

struct Layout {
  size_t sub_max, mass, chunk, bytes;
  int32_t chunks;
};

Layout layout(int64_t rows, int32_t vocab) {
  Layout l;
  l.chunks = (vocab + kChunk - 1) / kChunk;
  const size_t n = size_t(rows) * l.chunks;
  l.sub_max = 0;
  l.mass = align256(n * kChunkSubs * sizeof(float));
  l.chunk = l.mass + align256(n * kChunkGroups * sizeof(float));
  l.bytes = l.chunk + align256(n * sizeof(float2));
  return l;
}

template <typename T>
int launch(const SampleArgs& args, hipStream_t s) {
  const int64_t waves = int64_t(args.rows) * args.chunks;
  const int64_t blocks = (waves * kWave + kScanThreads - 1) / kScanThreads;
  if (blocks > 0x7fffffff) return WKV7_ERR_ARG;
  sample_scan_kernel<T><<<unsigned(blocks), kScanThreads, 0, s>>>(args);
  const int rc = launch_status();
  if (rc != WKV7_OK) return rc;
  sample_finish_kernel<T><<<unsigned(args.rows), kThreads, 0, s>>>(args);
  return launch_status();
}

}  // namespace
}  // namespace wkv7

using namespace wkv7;

extern "C" size_t wkv7_sample_workspace_bytes(int32_t rows, int32_t vocab) {
  if (rows < 1 || vocab < 1 || vocab > WKV7_SAMPLE_MAX_VOCAB) return 0;
  return layout(rows, vocab).bytes;
}

extern "C" int wkv7_sample_tokens(const void* logits, int32_t logits_dtype, int32_t rows,
                                  int32_t vocab, int64_t row_stride, const float* noise,
                                  int64_t noise_stride, const struct wkv7_sample_params* params,
                                  int32_t* tokens, float* logprobs, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  if (rows < 0 || vocab < 1 || !params) return WKV7_ERR_ARG;
  if (logits_dtype != WKV7_Y_BF16 && logits_dtype != WKV7_Y_F32) return WKV7_ERR_ARG;
  if (rows == 0) return WKV7_OK;
  if (!logits || !noise || !tokens) return WKV7_ERR_ARG;
  if (vocab > WKV7_SAMPLE_MAX_VOCAB || row_stride < vocab ||
      noise_stride < WKV7_SAMPLE_GROUP + (int64_t(vocab) + kGroup - 1) / kGroup)
    return WKV7_ERR_SHAPE;
  const size_t width = logits_dtype == WKV7_Y_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(logits) % width || reinterpret_cast<uintptr_t>(noise) % 4)
    return WKV7_ERR_SHAPE;
  const Layout l = layout(rows, vocab);
  if (!workspace || workspace_bytes < l.bytes || reinterpret_cast<uintptr_t>(workspace) % 16)
    return WKV7_ERR_WORKSPACE;
  char* ws = static_cast<char*>(workspace);
  const SampleArgs args{logits,
                        row_stride,
                        noise,
                        noise_stride,
                        params->temperature,
                        params->top_p,
                        params->min_p,
                        params->top_k,
                        params->temperature1,
                        params->top_p1,
                        params->min_p1,
                        params->top_k1,
                        vocab,
                        rows,
                        l.chunks,
                        tokens,
                        logprobs,
                        reinterpret_cast<float*>(ws + l.sub_max),
                        reinterpret_cast<float*>(ws + l.mass),
                        reinterpret_cast<float2*>(ws + l.chunk)};
  return logits_dtype == WKV7_Y_F32 ? launch<float>(args, as_stream(stream))
                                    : launch<uint16_t>(args, as_stream(stream));
}
