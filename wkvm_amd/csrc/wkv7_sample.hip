// Sampling of each row's next token by temperature, top-k, top-p and min-p, from
// given random numbers, with the token's log-probability.
//
// With M = max x, w_i = exp((x_i - M) / T) and the order "larger logit first, ties
// by lower index", every filter keeps a prefix of that order: top-k its first k
// tokens, top-p the shortest prefix whose weight reaches p of what top-k left,
// min-p the tokens with w_i >= min_p. So the kept set is one cut in the order,
// a pair (key, index), found by a radix descent over histograms of counts and
// weights; nothing is sorted.
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
// numbers of 42 fraction bits (w <= 1), so every sum is exact and the token does
// not depend on the order; plain sums are fp32 per thread, joined in a fixed order.
#include <algorithm>

#include "wkv7_common.h"

namespace wkv7 {
namespace {

typedef unsigned long long u64;

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / kWave;
constexpr int kBins = 2048;
constexpr int kGroup = WKV7_SAMPLE_GROUP;
constexpr float kLog2e = 1.44269504088896340736f;

struct SampleArgs {
  const void* logits;
  int64_t stride;
  const float* noise;
  int64_t noise_stride;
  const float *temperature, *top_p, *min_p;  // per row, or NULL: the value below
  const int32_t* top_k;
  float temperature1, top_p1, min_p1;
  int32_t top_k1;
  int32_t V;
  int32_t* tokens;
  float* logprobs;
};

struct Found {
  uint32_t bin, before_cnt, cnt;
  u64 before_wgt, wgt;
};

struct Shared {
  uint32_t cnt[kBins];
  u64 wgt[kBins];
  Found found;
  u64 red[kWaves];
  uint32_t wave_cnt[kWaves];
  u64 wave_wgt[kWaves];
};

// Ascending in the order of the tokens: the largest logit has the smallest key.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);  // (-0 and +0 are equal)
  return (u >> 31) ? u : ~u & 0x7fffffffu;
}

// NaN counts as -inf, +inf as the largest finite number.
__device__ __forceinline__ float clean(float x) {
  return fminf(fmaxf(x, -INFINITY), 3.402823466e38f);
}

// 42 fraction bits of w in [0, 1].
__device__ __forceinline__ u64 fixed(float w) {
  const float hi = truncf(w * 2097152.f);
  const float lo = (w * 2097152.f - hi) * 2097152.f;
  return (u64(uint32_t(hi)) << 21) + uint32_t(lo);
}

template <typename V, typename Op>
__device__ __forceinline__ V wave_all(V v, Op op) {
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) v = op(v, __shfl_xor(v, o));
  return v;
}

// Reduction over the block; every thread gets the result.
template <typename V, typename Op>
__device__ __forceinline__ V block_all(V v, Op op, Shared& sm) {
  static_assert(sizeof(V) <= sizeof(u64), "fits a slot");
  V* slot = reinterpret_cast<V*>(sm.red);
  v = wave_all(v, op);
  __syncthreads();
  if ((threadIdx.x & (kWave - 1)) == 0) slot[threadIdx.x / kWave] = v;
  __syncthreads();
  V r = slot[0];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) r = op(r, slot[i]);
  return r;
}

struct MaxF { __device__ float operator()(float a, float b) const { return fmaxf(a, b); } };
struct AddD { __device__ double operator()(double a, double b) const { return a + b; } };
struct MinU { __device__ u64 operator()(u64 a, u64 b) const { return a < b ? a : b; } };

// An arrival time (not negative) with its index: the smaller time wins, then the lower index.
__device__ __forceinline__ u64 arrival(float t, uint32_t i) {
  return (u64(__float_as_uint(t)) << 32) | i;
}

// Elements of one 16-byte load.
template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr int N = 4;
  float x[4];
  __device__ float get(int e) const { return clean(x[e]); }
};
template <> struct Vec<uint16_t> {
  static constexpr int N = 8;
  uint32_t x[4];
  __device__ float get(int e) const {
    return clean((e & 1) ? bf16_hi(x[e / 2]) : bf16_lo(x[e / 2]));
  }
};

template <typename T> struct Unaligned;
template <> struct Unaligned<float> {
  typedef float type __attribute__((ext_vector_type(4), aligned(4)));
};
template <> struct Unaligned<uint16_t> {
  typedef uint32_t type __attribute__((ext_vector_type(4), aligned(2)));
};

// The vector at element i of a row of n; elements past the end are -inf.
template <typename T>
__device__ __forceinline__ Vec<T> load_vec(const T* row, int i, int n) {
  Vec<T> v;
  if (i + Vec<T>::N <= n) {
    const auto r = *reinterpret_cast<const typename Unaligned<T>::type*>(row + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) v.x[e] = r[e];
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v.x[e] = i + e < n ? row[i + e] : -INFINITY;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t lo = i + 2 * e < n ? row[i + 2 * e] : 0xff80u;
      const uint32_t hi = i + 2 * e + 1 < n ? row[i + 2 * e + 1] : 0xff80u;
      v.x[e] = lo | hi << 16;
    }
  }
  return v;
}

// A row: R > 0 vectors per thread held in registers, or R = 0, read again by every pass.
template <typename T, int R>
struct Row {
  static constexpr int N = Vec<T>::N;
  static constexpr int kStep = kThreads * N;
  const T* p;
  int n;
  Vec<T> v[R > 0 ? R : 1];

  __device__ void load(const T* row, int len) {
    p = row;
    n = len;
    if constexpr (R > 0) {
#pragma unroll
      for (int j = 0; j < R; ++j)
        if (j * kStep < n) v[j] = load_vec(p, j * kStep + int(threadIdx.x) * N, n);
    }
  }
  // f(vector, index of its first element); every thread makes the same calls.
  template <typename F>
  __device__ __forceinline__ void vectors(F f) const {
    if constexpr (R > 0) {
#pragma unroll
      for (int j = 0; j < R; ++j)
        if (j * kStep < n) f(v[j], j * kStep + int(threadIdx.x) * N);
    } else {
      for (int j = 0; j * kStep < n; ++j) {
        const int i = j * kStep + int(threadIdx.x) * N;
        f(load_vec(p, i, n), i);
      }
    }
  }
  // f(logit, index) for the tokens of this thread
  template <typename F>
  __device__ __forceinline__ void operator()(F f) const {
    vectors([&](const Vec<T>& x, int i) {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (i + e < n) f(x.get(e), uint32_t(i + e));
    });
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

// The bin in which the cumulated count (or weight) reaches target >= 1; the last bin that
// holds anything where it never does.
__device__ __forceinline__ Found find_bin(Shared& sm, bool by_weight, u64 target) {
  const int t = threadIdx.x, lane = t & (kWave - 1), wave = t / kWave;
  __syncthreads();
  const uint32_t c0 = sm.cnt[2 * t], c1 = sm.cnt[2 * t + 1];
  const u64 w0 = sm.wgt[2 * t], w1 = sm.wgt[2 * t + 1];
  uint32_t c = c0 + c1;
  u64 w = w0 + w1;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const uint32_t cu = __shfl_up(c, o);
    const u64 wu = __shfl_up(w, o);
    if (lane >= o) {
      c += cu;
      w += wu;
    }
  }
  if (lane == kWave - 1) {
    sm.wave_cnt[wave] = c;
    sm.wave_wgt[wave] = w;
  }
  __syncthreads();
  uint32_t cb = 0, ct = 0;
  u64 wb = 0, wt = 0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    if (i < wave) {
      cb += sm.wave_cnt[i];
      wb += sm.wave_wgt[i];
    }
    ct += sm.wave_cnt[i];
    wt += sm.wave_wgt[i];
  }
  const u64 goal = min(target, by_weight ? wt : u64(ct));
  cb += c - c0 - c1;  // before bin 2 t
  wb += w - w0 - w1;
  const u64 b0 = by_weight ? wb : cb, v0 = by_weight ? w0 : c0, v1 = by_weight ? w1 : c1;
  if (b0 < goal && b0 + v0 >= goal) sm.found = {uint32_t(2 * t), cb, c0, wb, w0};
  if (b0 + v0 < goal && b0 + v0 + v1 >= goal)
    sm.found = {uint32_t(2 * t + 1), cb + c0, c1, wb + w0, w1};
  __syncthreads();
  return sm.found;
}

// A cut in the order: what lies before it or on it is kept.
struct Cut {
  uint32_t key, index;
  __device__ __forceinline__ bool keeps(float x, uint32_t i) const {
    const uint32_t k = order_key(x);
    return k < key || (k == key && i <= index);
  }
};

// The cut after the tokens whose count (or weight) reaches target, among those of `rows`
// that pred takes; `upto` gets the weight up to it (where weights are wanted).
template <typename Rows, typename Pred, typename Weight>
__device__ __forceinline__ Cut descend(const Rows& rows, Pred pred, Weight weight,
                                       bool want_weight, bool by_weight, u64 target, u64* upto,
                                       Shared& sm) {
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
  Cut cut{prefix, 0xffffffffu};
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

// The race over the tokens that `kept` takes. A group is the vectors of 256 / N neighbouring
// lanes.
template <typename T, int R, typename Kept, typename Weight>
__device__ __forceinline__ uint32_t race_row(const Row<T, R>& row, Kept kept, Weight weight,
                                             const float* noise, Shared& sm) {
  constexpr int kLanes = kGroup / Vec<T>::N;
  u64 best = ~0ull;
  row.vectors([&](const Vec<T>& x, int i) {
    float w = 0.f;
#pragma unroll
    for (int e = 0; e < Vec<T>::N; ++e) {
      const float v = x.get(e);
      if (i + e < row.n && kept(v, uint32_t(i + e))) w += weight(v);
    }
#pragma unroll
    for (int o = 1; o < kLanes; o <<= 1) w += __shfl_xor(w, o);
    if (w > 0.f && (threadIdx.x & (kLanes - 1)) == 0) {
      const int g = i / kGroup;
      best = min(best, arrival(noise[kGroup + g] / w, uint32_t(g)));
    }
  });
  const uint32_t group = uint32_t(block_all(best, MinU(), sm));
  best = ~0ull;
  const int i = int(group) * kGroup + int(threadIdx.x);
  if (threadIdx.x < kGroup && i < row.n) {
    float v;
    if constexpr (sizeof(T) == 4) v = clean(row.p[i]);
    else v = clean(bf16_to_f32(row.p[i]));
    if (kept(v, uint32_t(i))) best = arrival(noise[threadIdx.x] / weight(v), uint32_t(i));
  }
  return uint32_t(block_all(best, MinU(), sm));
}

template <typename T, int R>
__global__ __launch_bounds__(kThreads) void sample_kernel(const SampleArgs args) {
  __shared__ Shared sm;
  const int64_t b = blockIdx.x;
  const int V = args.V;
  Row<T, R> row;
  row.load(static_cast<const T*>(args.logits) + b * args.stride, V);
  const float* noise = args.noise + b * args.noise_stride;
  const float temp = args.temperature ? args.temperature[b] : args.temperature1;
  const float top_p = args.top_p ? args.top_p[b] : args.top_p1;
  const float min_p = args.min_p ? args.min_p[b] : args.min_p1;
  const int32_t top_k = args.top_k ? args.top_k[b] : args.top_k1;
  const bool greedy = !(temp > 0.f);
  const bool by_k = top_k > 0 && top_k < V;
  const bool by_p = top_p < 1.f;

  float tmax = -INFINITY;
  row([&](float x, uint32_t) { tmax = fmaxf(tmax, x); });
  const float top = block_all(tmax, MaxF(), sm);
  if (top == -INFINITY) {  // nothing to choose from
    if (threadIdx.x == 0) {
      args.tokens[b] = -1;
      if (args.logprobs) args.logprobs[b] = -INFINITY;
    }
    return;
  }
  // w = 2^((x - top) c); the clamp keeps c and every product a number
  const float c = kLog2e / fminf(fmaxf(temp, 0x1p-60f), 0x1p60f);
  auto weight = [&](float x) { return __builtin_amdgcn_exp2f((x - top) * c); };
  const float floor_z = min_p > 0.f ? log2f(fminf(min_p, 1.f)) : -INFINITY;
  auto over_floor = [&](float x) { return (x - top) * c >= floor_z; };

  double total = 0., raw = 0.;
  if (args.logprobs) {
    float s = 0.f;
    row([&](float x, uint32_t) { s += __builtin_amdgcn_exp2f((x - top) * kLog2e); });
    raw = block_all(double(s), AddD(), sm);
  }
  uint32_t token;
  if (greedy) {
    u64 best = ~0ull;
    row([&](float x, uint32_t i) { best = min(best, u64(order_key(x)) << 32 | i); });
    token = uint32_t(block_all(best, MinU(), sm));
  } else if (!by_k && !by_p) {
    token = race_row(row, [&](float x, uint32_t) { return over_floor(x); }, weight, noise, sm);
  } else {
    if (by_p && !by_k) {
      float s = 0.f;
      row([&](float x, uint32_t) { s += weight(x); });
      total = block_all(double(s), AddD(), sm);
    }
    auto all = [](float, uint32_t) { return true; };
    Cut cut{0xffffffffu, 0xffffffffu};
    if (by_k) {
      u64 upto = 0;
      cut = descend(row, all, weight, by_p, false, u64(top_k), &upto, sm);
      total = double(upto) * 0x1p-42;
    }
    if (by_p) {
      const Cut outer = cut;
      const u64 target = max(u64(1), u64(ceil(fmax(double(top_p), 0.) * total * 0x1p42)));
      cut = descend(row, [&](float x, uint32_t i) { return outer.keeps(x, i); }, weight, true,
                    true, target, static_cast<u64*>(nullptr), sm);
      // (all of a key's tokens: all that top-k left of them)
      if (cut.key == outer.key) cut.index = min(cut.index, outer.index);
    }
    token = race_row(row, [&](float x, uint32_t i) { return cut.keeps(x, i) && over_floor(x); },
                     weight, noise, sm);
  }
  if (threadIdx.x == 0) {
    args.tokens[b] = int32_t(token);
    if (args.logprobs) {
      const T* p = static_cast<const T*>(args.logits) + b * args.stride;
      float x;
      if constexpr (sizeof(T) == 4) x = clean(p[token]);
      else x = clean(bf16_to_f32(p[token]));
      args.logprobs[b] = float(double(x - top) - log(raw));
    }
  }
}

template <typename T>
int launch(const SampleArgs& args, int32_t rows, hipStream_t s) {
  constexpr int kStep = Row<T, 0>::kStep;
  if (args.V <= 16 * kStep) sample_kernel<T, 16><<<rows, kThreads, 0, s>>>(args);
  else sample_kernel<T, 0><<<rows, kThreads, 0, s>>>(args);
  return launch_status();
}

}  // namespace
}  // namespace wkv7

using namespace wkv7;

extern "C" int wkv7_sample_tokens(const void* logits, int32_t logits_dtype, int32_t rows,
                                  int32_t vocab, int64_t row_stride, const float* noise,
                                  int64_t noise_stride, const struct wkv7_sample_params* params,
                                  int32_t* tokens, float* logprobs, void* stream) {
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
                        tokens,
                        logprobs};
  return logits_dtype == WKV7_Y_F32 ? launch<float>(args, rows, as_stream(stream))
                                    : launch<uint16_t>(args, rows, as_stream(stream));
}
