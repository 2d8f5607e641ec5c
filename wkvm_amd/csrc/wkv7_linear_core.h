// Device code of the chunked linear attention (wkv7_linear_prefill).
//
// A workgroup of four waves walks one piece of one sequence for one head and 64 value columns, 64
// tokens at a time, its state in accumulator registers. With v_mfma_f32_16x16x32_bf16 (lane l, li =
// l % 16, lg = l / 16: an A or B lane holds row or column li at 8 lg .. 8 lg + 7 of a 32-wide block,
// a result lane D[4 lg + i][li]):
//   * wave w owns the chunk's tokens 16 w .. 16 w + 15 for the outputs, which are computed
//     transposed (D rows are value columns), and K / 4 key rows of the state
//   * the rows of a result tile are named so that the registers of two tiles are an operand of the
//     next product as they stand: keys and tokens 32 p + 8 (m / 4) + 4 half + m % 4 for row m of
//     tile (p, half), and value columns likewise. Scores therefore never leave their wave; of the
//     state a bf16 split goes through LDS, each lane's own words
//   * q, k and v come by direct loads into LDS, one chunk ahead; k and v are read transposed
// The operands that are not bf16 to begin with (scores under their decays, decayed keys, the state)
// are split into bf16 parts: three where an fp32 result is kept (the state, an fp32 y), two
// (2^-17 of each term) for a y that is rounded to bf16.
#pragma once

#include "wkv7_mfma.h"

namespace wkv7 {
namespace {

constexpr int kChunk = 64;          // tokens of a chunk
constexpr int kLinearThreads = 256;
constexpr int kLinearXcds = 8;      // workgroups are dealt round-robin over 8 XCDs
constexpr int kMinPiece = 512;      // tokens of the shortest piece that a sequence is cut into
constexpr int kChainThreads = 256;
constexpr int kChainElems = 4 * kChainThreads;
constexpr double kLog2e = 1.4426950408889634;

struct LinearSeqs {
  float* state;
  int64_t rows;
  const int32_t* slot_ids;
  const int32_t* cu;
  int32_t nseq;
  bool zero_init;
  int64_t tokens;
  // Piece g of sequence s, tokens [cu[s] + g piece, ..), is number cu[s] / piece + s + g of `slots`;
  // piece 0: a sequence is one piece, number s.
  int64_t piece, slots;
  int64_t span;    // work items per XCD
  float* pieces;   // [slots][H][K][V]: local final states, then the pieces' initial states
  double* sums;    // [slots][H]: sums of log2 decays
};

typedef __attribute__((address_space(3))) uint4 lds_u4;
typedef __attribute__((address_space(3))) float lds_f32;

__device__ __forceinline__ uint32_t lds_at(const uint4* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const lds_u4*)p));
}
__device__ __forceinline__ uint32_t lds_at(const float* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const lds_f32*)p));
}

// Direct loads, lane l's 16 (4) bytes to lds + 16 l (4 l). The compiler does not see them: every
// wait for them is one of the barriers below.
__device__ __forceinline__ void to_lds16(const void* src, uint32_t lds) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "{m0}"(lds), "v"(src) : "memory");
}
__device__ __forceinline__ void to_lds4(const void* src, uint32_t lds) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dword %1, off" : : "{m0}"(lds), "v"(src) : "memory");
}
// At most N vector memory operations of this wave pending, then the workgroup barrier. (They
// complete in order, stores among them.)
template <int N>
__device__ __forceinline__ void barrier_vm() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(N) : "memory");
}
__device__ __forceinline__ void barrier_lds() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory");
}

// Two values as N packed bf16 parts, the largest first.
template <int N>
__device__ __forceinline__ void split_pair(float a, float b, uint32_t (&out)[N], const Neg& n) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    out[i] = pack_bf16(a, b);
    if (i + 1 < N) {
      a = sub_bf16(a, out[i], n.lo);
      b = sub_bf16(b, out[i], n.hi);
    }
  }
}

template <int N>
__device__ __forceinline__ void split_eight(const float (&x)[8], uint4 (&out)[N], const Neg& n) {
  uint32_t w[4][N];
#pragma unroll
  for (int i = 0; i < 4; ++i) split_pair<N>(x[2 * i], x[2 * i + 1], w[i], n);
#pragma unroll
  for (int i = 0; i < N; ++i) out[i] = make_uint4(w[0][i], w[1][i], w[2][i], w[3][i]);
}

// Sequence and tokens of piece number `slot`; false where it has none. (Offsets that break their
// contract give some tokens in [0, tokens).)
struct Piece {
  int seq;
  int64_t beg, end;  // its tokens
  bool first, last;
};

__device__ __forceinline__ int64_t offset_at(const LinearSeqs& a, int s) {
  return min(max(int64_t(a.cu[s]), int64_t(0)), a.tokens);
}

__device__ __forceinline__ bool find_piece(const LinearSeqs& a, int64_t slot, Piece& p) {
  int s = int(slot);
  int64_t index = 0;
  if (a.piece) {
    // the last sequence whose first piece is at most `slot`, 64 of them at a time
    const int lane = threadIdx.x & 63;
    int n = 0;
    for (int i = 0; i < a.nseq; i += 64) {
      const int at = i + lane;
      const bool in = at < a.nseq && offset_at(a, at) / a.piece + at <= slot;
      const uint64_t votes = __ballot(in);
      n += __popcll(votes);
      if (votes != ~uint64_t(0)) break;
    }
    s = n - 1;
    if (s < 0) return false;
    index = slot - (offset_at(a, s) / a.piece + s);
  }
  const int64_t beg = offset_at(a, s), end = max(offset_at(a, s + 1), beg);
  if (index < 0 || (index > 0 && beg + index * a.piece >= end)) return false;
  p.seq = s;
  p.beg = beg + index * a.piece;
  p.end = a.piece ? min(p.beg + a.piece, end) : end;
  p.first = index == 0;
  p.last = p.end == end;
  return true;
}

template <int KD, bool kStates>
struct LinearStage {
  uint4 q[kStates ? 1 : kChunk * KD / 8];
  uint4 k[kChunk * KD / 8];
  uint4 v[kChunk * 8];
  float g[4][kChunk];  // every wave's own copy
};

// element offset of channel e of row r of a [row][W] array, whose 16-byte chunks are swizzled by row
template <int W>
__device__ __forceinline__ int at(int r, int e) {
  return r * W + ((((e >> 3) ^ r) & (W / 8 - 1)) << 3) + (e & 7);
}

// kStates: only the piece's final state from zero and the sum of its decays, for a piece that is
// not its sequence's last.
template <int KD, bool kF32, bool kStates>
__global__ __launch_bounds__(kLinearThreads) void linear_prefill_kernel(const LinearSeqs a,
                                                                         const wkv7_linear_io io) {
  constexpr int RT = KD / 64;          // state tiles of a wave by 16 key rows
  constexpr int NP = KD / 32;          // blocks of 32 keys
  constexpr int YP = kF32 ? 3 : 2;     // bf16 parts of the state and the scores in y
  constexpr int KL = KD / 32;          // direct loads of a wave for its share of q or k
  constexpr int kLoads = (kStates ? KL : 2 * KL) + 2 + 1;
  __shared__ LinearStage<KD, kStates> ring[2];
  __shared__ uint4 s_state[kStates ? 1 : YP * NP * 4 * 64];
  __shared__ float s_hi[4][kChunk], s_lo[4][kChunk], s_dec[4][kChunk];
  __shared__ float s_part[2][4][64];
  __shared__ int s_bad[2];

  const int lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tiles = io.V / 64;
  // neighbouring items (the tiles and heads that share q and k) on one XCD
  int64_t item = int64_t(blockIdx.x % kLinearXcds) * a.span + blockIdx.x / kLinearXcds;
  if (item >= a.slots * io.H * tiles) return;
  const int vt = int(item % tiles);
  item /= tiles;
  const int head = int(item % io.H);
  const int64_t slot_no = item / io.H;
  Piece pc;
  if (!find_piece(a, slot_no, pc)) return;
  const int64_t row = a.slot_ids[pc.seq];
  const int64_t V = io.V;
  const int col0 = 64 * vt;
  if (kStates && pc.last) return;
  if (row < 0 || row >= a.rows) {  // no state is touched, the outputs are zero
    if (!kStates)
      for (int64_t t = pc.beg + wave; t < pc.end; t += 4) {
        const int64_t o = (t * io.H + head) * V + col0 + lane;
        if (kF32) static_cast<float*>(io.y)[o] = 0.f;
        else static_cast<uint16_t*>(io.y)[o] = 0;
      }
    return;
  }

  // state: key(rt, i) and column(c) of this lane's accumulators
  const int kp = RT == 1 ? wave >> 1 : wave;  // the wave's block of 32 keys
  auto half_of = [&](int rt) { return RT == 1 ? wave & 1 : rt; };
  auto key0 = [&](int rt) { return 32 * kp + 8 * lg + 4 * half_of(rt); };
  auto col_of = [&](int c) { return 32 * (c >> 1) + 8 * (li >> 2) + 4 * (c & 1) + (li & 3); };
  float* slot_state = a.state + (row * io.H + head) * (KD * V) + col0;
  float* piece_state = a.piece ? a.pieces + (slot_no * io.H + head) * (KD * V) + col0 : nullptr;

  f32x4 S[RT][4];
  const float* from = kStates ? nullptr
                      : a.piece ? piece_state
                      : a.zero_init ? nullptr : slot_state;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        S[rt][c][i] = from && pc.end > pc.beg ? from[(key0(rt) + i) * V + col_of(c)] : 0.f;

  auto store_state = [&](float* to) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) to[(key0(rt) + i) * V + col_of(c)] = S[rt][c][i];
  };
  if (pc.end == pc.beg) {
    if (!kStates && a.zero_init) store_state(slot_state);
    return;
  }

  const int hq = head / (io.H / io.Hq);
  const uint16_t* qp = io.q + hq * KD;
  const uint16_t* kptr = io.k + hq * KD;
  const uint16_t* vp = io.v + int64_t(head) * V + col0;
  const float* gp = io.log_decay + head;

  // The direct loads of chunk c; rows behind the piece read its last token again (their decays are
  // taken as 0 and their keys are dropped from the state).
  auto issue = [&](int64_t c, LinearStage<KD, kStates>& st) {
    const int64_t t0 = pc.beg + kChunk * c, lastt = pc.end - 1;
    constexpr int R = 64 / (KD / 8);  // rows of a load
#pragma unroll
    for (int i = 0; i < KL; ++i) {
      const int r = R * (4 * i + wave) + lane / (KD / 8);
      const int ch = ((lane % (KD / 8)) ^ r) & (KD / 8 - 1);
      const int64_t t = min(t0 + r, lastt);
      if (!kStates) to_lds16(qp + t * io.ldq + 8 * ch, lds_at(st.q) + 1024 * (4 * i + wave));
      to_lds16(kptr + t * io.ldk + 8 * ch, lds_at(st.k) + 1024 * (4 * i + wave));
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = 8 * (4 * i + wave) + lane / 8;
      const int ch = ((lane % 8) ^ r) & 7;
      to_lds16(vp + min(t0 + r, lastt) * io.ldv + 8 * ch, lds_at(st.v) + 1024 * (4 * i + wave));
    }
    to_lds4(gp + min(t0 + lane, lastt) * io.ld_decay, lds_at(&st.g[wave][0]));
  };

  const Neg neg = neg_consts();
  const int64_t chunks = (pc.end - pc.beg + kChunk - 1) / kChunk;
  f32x4 y[4];           // the last chunk's outputs, stored behind the next one's first barrier
  bool pending = false;
  double sum = 0.;      // log2 decays of the piece so far

  auto store_y = [&](int64_t c) {
    const int64_t t = pc.beg + kChunk * c + 16 * wave + li;
    if (t >= pc.end) return;
    const int64_t o = (t * io.H + head) * V + col0 + 8 * lg;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const f32x4 &x0 = y[2 * h], &x1 = y[2 * h + 1];
      if (kF32) {
        f32x4* p = reinterpret_cast<f32x4*>(static_cast<float*>(io.y) + o + 32 * h);
        p[0] = x0;
        p[1] = x1;
      } else {
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(io.y) + o + 32 * h) =
            make_uint4(pack_bf16(x0[0], x0[1]), pack_bf16(x0[2], x0[3]), pack_bf16(x1[0], x1[1]),
                       pack_bf16(x1[2], x1[3]));
      }
    }
  };

  issue(0, ring[0]);
  for (int64_t c = 0; c < chunks; ++c) {
    LinearStage<KD, kStates>& st = ring[c & 1];
    const bool more = c + 1 < chunks;
    const int n = int(min(int64_t(kChunk), pc.end - pc.beg - kChunk * c));  // its tokens
    if (more) issue(c + 1, ring[(c + 1) & 1]);
    if (!kStates) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int ct = 0; ct < 4; ++ct) {
          uint32_t lo[YP], hi[YP];
          split_pair<YP>(S[rt][ct][0], S[rt][ct][1], lo, neg);
          split_pair<YP>(S[rt][ct][2], S[rt][ct][3], hi, neg);
#pragma unroll
          for (int p = 0; p < YP; ++p)
            reinterpret_cast<uint2*>(&s_state[((p * NP + kp) * 4 + ct) * 64 + lane])[half_of(rt)] =
                make_uint2(lo[p], hi[p]);
        }
    }
    if (threadIdx.x == 0) s_bad[c & 1] = 0;
    if (more) barrier_vm<kLoads>();
    else barrier_vm<0>();
    if (!kStates && pending) store_y(c - 1);

    // G: sums of log2 decays up to each token, in 64 bits, then as two floats
    double G = 0.;
    if (lane < n) {
      const float g = st.g[wave][lane];
      G = double(g < -1e4f ? -1e4f : g) * kLog2e;
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const double before = __shfl_up(G, d);
      if (lane >= d) G += before;
    }
    const double Glast = __shfl(G, 63);
    const float Ghi = float(G);
    s_hi[wave][lane] = Ghi;
    s_lo[wave][lane] = float(G - double(Ghi));
    s_dec[wave][lane] = lane < n ? __builtin_amdgcn_exp2f(float(Glast - G)) : 0.f;
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    const float all = __builtin_amdgcn_exp2f(float(Glast));

    const uint16_t* sq = reinterpret_cast<const uint16_t*>(st.q);
    const uint16_t* sk = reinterpret_cast<const uint16_t*>(st.k);
    const uint16_t* sv = reinterpret_cast<const uint16_t*>(st.v);
    uint4 vf[2][4];  // V: columns li of tile c, tokens 32 b + 8 lg ..
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int ct = 0; ct < 4; ++ct) {
        const int col = 32 * (ct >> 1) + 4 * (ct & 1) + 8 * (li & 3);
        const uint2 x = ld_tr(sv + at<64>(32 * b + 8 * lg + (li >> 2), col));
        const uint2 z = ld_tr(sv + at<64>(32 * b + 8 * lg + 4 + (li >> 2), col));
        vf[b][ct] = make_uint4(x.x, x.y, z.x, z.y);
      }

    float wrong = 0.f;  // NaN as soon as a result is not finite
    if (!kStates) {
      const int t = 16 * wave + li;
      uint4 qf[NP];
#pragma unroll
      for (int p = 0; p < NP; ++p) qf[p] = ld16(sq + at<KD>(t, 32 * p + 8 * lg));
#pragma unroll
      for (int ct = 0; ct < 4; ++ct) y[ct] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int part = YP - 1; part >= 0; --part)
#pragma unroll
        for (int p = 0; p < NP; ++p)
#pragma unroll
          for (int ct = 0; ct < 4; ++ct)
            y[ct] = mma32(s_state[((part * NP + p) * 4 + ct) * 64 + lane], qf[p], y[ct]);
      const float thi = s_hi[wave][t], tlo = s_lo[wave][t];
      const float es = __builtin_amdgcn_exp2f(thi + tlo) * io.scale;
#pragma unroll
      for (int ct = 0; ct < 4; ++ct)
#pragma unroll
        for (int i = 0; i < 4; ++i) y[ct][i] *= es;
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        if (b > (wave >> 1)) break;  // (uniform) behind every token of the wave
        float p8[8];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          f32x4 sc = {0.f, 0.f, 0.f, 0.f};
          const int kr = 32 * b + 8 * (li >> 2) + 4 * h + (li & 3);
#pragma unroll
          for (int p = 0; p < NP; ++p) sc = mma32(ld16(sk + at<KD>(kr, 32 * p + 8 * lg)), qf[p], sc);
          const int s0 = 32 * b + 8 * lg + 4 * h;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float e =
                __builtin_amdgcn_exp2f((thi - s_hi[wave][s0 + i]) + (tlo - s_lo[wave][s0 + i]));
            p8[4 * h + i] = s0 + i <= t ? sc[i] * io.scale * e : 0.f;
          }
        }
        uint4 pf[YP];
        split_eight<YP>(p8, pf, neg);
#pragma unroll
        for (int part = YP - 1; part >= 0; --part)
#pragma unroll
          for (int ct = 0; ct < 4; ++ct) y[ct] = mma32(vf[b][ct], pf[part], y[ct]);
      }
      if (t < n)
#pragma unroll
        for (int ct = 0; ct < 4; ++ct)
#pragma unroll
          for (int i = 0; i < 4; ++i) wrong = fmaf(y[ct][i], 0.f, wrong);
    }

    f32x4 next[RT][4];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
      for (int ct = 0; ct < 4; ++ct)
#pragma unroll
        for (int i = 0; i < 4; ++i) next[rt][ct][i] = S[rt][ct][i] * all;
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int key = 32 * kp + 4 * half_of(rt) + 8 * (li & 3);
        const uint2 x = ld_tr(sk + at<KD>(32 * b + 8 * lg + (li >> 2), key));
        const uint2 z = ld_tr(sk + at<KD>(32 * b + 8 * lg + 4 + (li >> 2), key));
        const uint4 kt = make_uint4(x.x, x.y, z.x, z.y);
        float kd[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) kd[j] = elem(kt, j) * s_dec[wave][32 * b + 8 * lg + j];
        uint4 kf[3];
        split_eight<3>(kd, kf, neg);
#pragma unroll
        for (int part = 2; part >= 0; --part)
#pragma unroll
          for (int ct = 0; ct < 4; ++ct)
            next[rt][ct] = mma32(kf[part], vf[b][ct], next[rt][ct]);
      }
#pragma unroll
      for (int ct = 0; ct < 4; ++ct)
#pragma unroll
        for (int i = 0; i < 4; ++i) wrong = fmaf(next[rt][ct][i], 0.f, wrong);
    }
    if (__ballot(wrong != wrong) && lane == 0) s_bad[c & 1] = 1;
    barrier_lds();
    sum += Glast;
    pending = true;
    if (!s_bad[c & 1]) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int ct = 0; ct < 4; ++ct) S[rt][ct] = next[rt][ct];
      continue;
    }
    // Something in the chunk is not finite: products of whole tiles would carry it to tokens before
    // it (0 times infinity). Token by token instead, as the formula is written.
    pending = false;
    for (int t = 0; t < n; ++t) {
      const float d = expf(st.g[wave][t]);
      float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float kv = bf16_to_f32(sk[at<KD>(t, key0(rt) + i)]);
          const float qv = kStates ? 0.f : bf16_to_f32(sq[at<KD>(t, key0(rt) + i)]) * io.scale;
#pragma unroll
          for (int ct = 0; ct < 4; ++ct) {
            const float v = bf16_to_f32(sv[at<64>(t, col_of(ct))]);
            S[rt][ct][i] = fmaf(d, S[rt][ct][i], kv * v);
            if (!kStates) part[ct] = fmaf(qv, S[rt][ct][i], part[ct]);
          }
        }
      if (kStates) continue;
#pragma unroll
      for (int ct = 0; ct < 4; ++ct) {
        part[ct] += __shfl_xor(part[ct], 16);
        part[ct] += __shfl_xor(part[ct], 32);
        if (lg == 0) s_part[t & 1][wave][col_of(ct)] = part[ct];
      }
      barrier_lds();
      if (wave == 0) {
        const float (*p)[64] = s_part[t & 1];
        const float v = (p[0][lane] + p[1][lane]) + (p[2][lane] + p[3][lane]);
        const int64_t o = ((pc.beg + kChunk * c + t) * io.H + head) * V + col0 + lane;
        if (kF32) static_cast<float*>(io.y)[o] = v;
        else static_cast<uint16_t*>(io.y)[o] = f32_to_bf16(v);
      }
    }
    barrier_lds();  // the stage is free for the next loads
  }
  if (kStates) {
    store_state(piece_state);
    if (vt == 0 && threadIdx.x == 0) a.sums[slot_no * io.H + head] = sum;
    return;
  }
  if (pending) store_y(chunks - 1);
  if (pc.last) store_state(slot_state);
}

// From the pieces' local final states to their initial states, in order, four entries per thread:
// S_in(0) is the sequence's initial state, S_in(g + 1) = e^(sum of g) S_in(g) + S_local(g).
template <int KD>
__global__ __launch_bounds__(kChainThreads) void linear_chain_kernel(const LinearSeqs a,
                                                                      const wkv7_linear_io io) {
  const int64_t size = int64_t(KD) * io.V;
  const int blocks = int(size / kChainElems);
  int64_t item = blockIdx.x;
  const int64_t e = (item % blocks) * kChainElems + 4 * threadIdx.x;
  item /= blocks;
  const int head = int(item % io.H);
  const int s = int(item / io.H);
  const int64_t row = a.slot_ids[s];
  if (row < 0 || row >= a.rows) return;
  const int64_t beg = offset_at(a, s), end = max(offset_at(a, s + 1), beg);
  const int64_t n = (end - beg + a.piece - 1) / a.piece;
  if (n == 0) return;
  f32x4 run = {0.f, 0.f, 0.f, 0.f};
  if (!a.zero_init)
    run = *reinterpret_cast<const f32x4*>(a.state + (row * io.H + head) * size + e);
  const int64_t first = beg / a.piece + s;
  float* p = a.pieces + (first * io.H + head) * size + e;
  const double* sums = a.sums + first * io.H + head;
  f32x4 local = run;
  if (n > 1) local = *reinterpret_cast<const f32x4*>(p);
  for (int64_t g = 0; g < n; ++g) {
    f32x4 ahead = run;
    if (g + 2 < n) ahead = *reinterpret_cast<const f32x4*>(p + io.H * size);
    *reinterpret_cast<f32x4*>(p) = run;
    if (g + 1 < n) {
      const double sum = sums[g * io.H];
      const float f = exp2f(float(sum));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // an infinite entry stays so, however small the factor, unless a token forgot the state
        const bool inf = fabsf(run[i]) == INFINITY && f == 0.f && sum > -1e4;
        run[i] = inf ? run[i] + local[i] : fmaf(f, run[i], local[i]);
      }
    }
    local = ahead;
    p += io.H * size;
  }
}

}  // namespace
}  // namespace wkv7
