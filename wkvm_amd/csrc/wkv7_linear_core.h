// Device code of the chunked linear attention (wkv7_linear_prefill).
//
// A workgroup walks one piece of one sequence for one head and a tile of VT value columns, 64 tokens
// at a time ("chunk"), its state in the accumulator registers of four state waves, each of which owns
// K / 4 key rows. Two groups of four output waves take the chunks in turn, 16 tokens to a wave. With
// v_mfma_f32_16x16x32_bf16 (lane l, li = l % 16, lg = l / 16: an A or B lane holds row or column li at
// 8 lg .. 8 lg + 7 of a 32-wide block, a result lane D[4 lg + i][li]), the rows of a result tile are
// named so that the registers of two tiles are an operand of the next product as they stand: keys,
// tokens and value columns 32 p + 8 (m / 4) + 4 half + m % 4 for row m of tile (p, half). Scores
// therefore never leave their wave; of the state a bf16 split goes through LDS, each lane's own words.
//
// In tick c, with one barrier at its end:
//   state waves    write the split of the state before chunk c, ask for the k and v rows of chunk
//                  c + kAhead + 1 (direct loads into an LDS ring), add chunk c to the state, decay
//                  the keys of chunk c + 1
//   one group      chunk c - 1: the state's part of the outputs, scores of the wave's own block
//   the other      chunk c - 2: the other scores, their products with the values, the outputs; sums
//                  of the decays of chunk c + 2
// The operands that are not bf16 to begin with (scores under their decays, decayed keys, the state)
// are split into three bf16 parts, which hold all of an fp32 number: a bf16 y is the fp32 one rounded
// once. (With two parts, 2^-18 of each term, 8 x 4,096 tokens x 32 heads take 132.7 us on a card where
// three take 138.4, and 134.6 on one where three take 133.4; 16,384 tokens x 12 heads 50.6 and 53.8.)
#pragma once

#include "wkv7_mfma.h"

namespace wkv7 {
namespace {

constexpr int kChunk = 64;          // tokens of a chunk
constexpr int kLinearXcds = 8;      // workgroups are dealt round-robin over 8 XCDs
constexpr int kMinPiece = 256;      // tokens of the shortest piece that a sequence is cut into
constexpr int kChainThreads = 64;
constexpr int kChainElems = 4 * kChainThreads;
constexpr int kParts = 3;           // bf16 parts of an fp32 operand
constexpr double kLog2e = 1.4426950408889634;

struct LinearSeqs {
  float* state;
  int64_t rows;
  const int32_t* slot_ids;
  const int32_t* cu;
  int32_t nseq;
  bool zero_init;
  int64_t tokens;
  // Piece g of sequence s, tokens [cu[s] + g piece, ..), is number first_piece(s) + g of `slots`; piece
  // 0: a sequence is one piece, number s.
  int64_t piece, slots;
  const int32_t* order;  // of whole sequences (or null): the one to start as number i
  bool longest_first;    // without an order, and nseq < 64: by length
  float* pieces;   // [slots][H][K][V]: local final states, then the pieces' initial states
  double* sums;    // [slots][H]: sums of log2 decays, -infinity where a token forgets the state
};

typedef __attribute__((address_space(3))) uint4 lds_u4;

__device__ __forceinline__ uint32_t lds_at(const uint4* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const lds_u4*)p));
}
// Direct load: 16 bytes per lane from base + offset to lds + 16 l. The compiler does not see it:
// every wait for it is one of the barriers below. kOnce: lines that are not read again are not kept
// in the caches (19 ragged prompts of 128 channels 104.7 us, 108.1 without; 8 x 4,096 tokens x 32 heads
// 135.4 and 136.3. The queries, whose lines are read in parts, and the outputs' stores are slower so).
template <bool kOnce>
__device__ __forceinline__ void to_lds16(const void* base, uint32_t offset, uint32_t lds) {
  if constexpr (kOnce) {
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt"
                 :
                 : "{m0}"(lds), "v"(offset), "s"(base)
                 : "memory");
  } else {
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :
                 : "{m0}"(lds), "v"(offset), "s"(base)
                 : "memory");
  }
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

// At least one number further for the next sequence, and at least as many as this one has pieces: an
// empty sequence has a number too, whose workgroups clear its state where it begins at zero.
__device__ __forceinline__ int64_t first_piece(const LinearSeqs& a, int s) {
  return offset_at(a, s) / a.piece + s;
}

__device__ __forceinline__ bool find_piece(const LinearSeqs& a, int64_t slot, Piece& p) {
  int s = int(slot);
  int64_t index = 0;
  if (a.longest_first) {
    // lane i has the offset and the length of sequence i; the one with `slot` longer ones (of two of
    // one length the first counts as longer) is it
    const int lane = threadIdx.x & 63;
    const int at = int(offset_at(a, min(lane, a.nseq)));
    const int length = __shfl_down(at, 1) - at;
    int longer = 0;
    for (int i = 0; i < a.nseq; ++i) {
      const int other = __builtin_amdgcn_readlane(length, i);
      longer += other > length || (other == length && i < lane);
    }
    s = __builtin_ctzll(__ballot(lane < a.nseq && longer == s));
    p.seq = s;
    p.beg = __builtin_amdgcn_readlane(at, s);
    p.end = max(int64_t(__builtin_amdgcn_readlane(at, s + 1)), p.beg);
    p.first = p.last = true;
    return true;
  }
  if (!a.piece && a.order) {
    s = a.order[s];
    if (s < 0 || s >= a.nseq) return false;
  }
  if (a.piece) {
    // the last sequence whose first piece is at most `slot`, 64 of them at a time
    const int lane = threadIdx.x & 63;
    int n = 0;
    for (int i = 0; i < a.nseq; i += 64) {
      const int at = i + lane;
      const bool in = at < a.nseq && first_piece(a, at) <= slot;
      const uint64_t votes = __ballot(in);
      n += __popcll(votes);
      if (votes != ~uint64_t(0)) break;
    }
    s = n - 1;
    if (s < 0) return false;
    index = slot - first_piece(a, s);
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

// The 16-byte chunks of a [row][W] array's rows are swizzled by the row, W / 8 chunks a row: chunk c
// of row r sits at c ^ turn(r). An operand read touches chunks 4 x + 0 .. 3 of rows 8 a + 0 .. 3 (a = 0
// .. 3; half of each chunk where the read transposes), or one chunk per lane group of 16 such rows:
// either way every 16 bytes of the 256-byte bank row equally often.
template <int W>
__device__ __forceinline__ int turn(int r) {
  return W == 128 ? (r & 3) << 2 | (r >> 3 & 3) : W == 64 ? (r & 3) | (r >> 1 & 4) : 0;
}
// element offset of channel e of row r
template <int W>
__device__ __forceinline__ int at(int r, int e) {
  return r * W + (((e >> 3) ^ turn<W>(r)) << 3) + (e & 7);
}

// LDS of a workgroup. Chunk c of k and v sits in ring[c % R].
template <int KD, int VT, bool kOutputs, int R>
struct LinearLds {
  static constexpr int NP = KD / 32, NC = VT / 16;
  static constexpr int kDecays = 5;
  struct Stage {
    uint4 k[kChunk * KD / 8];
    uint4 v[kChunk * VT / 8];
  } ring[R];
  uint4 state[2][kOutputs ? kParts * NP * NC * 64 : 1];  // [c % 2]: parts of the state before chunk c
  // of chunk c at [c % kDecays]: its tokens' sums of log2 decays G as two floats each,
  // e^(G_last - G), the decays themselves, e^G_last
  struct Decays {
    alignas(16) float hi[kChunk];
    alignas(16) float lo[kChunk];
    alignas(16) float left[kChunk];
    float raw[kChunk], all;
  } decays[kDecays];
  float part[2][4][VT];
  int bad[4];  // [c % 4]: something in chunk c is not finite
  int again;   // some output of another chunk is not
};

// The state waves' share of a piece: `mine` 0 .. 3.
template <int KD, int VT, bool kOutputs, int R>
struct StateWave {
  using Lds = LinearLds<KD, VT, kOutputs, R>;
  static constexpr int RT = KD / 64, NC = VT / 16, NP = KD / 32;
  static constexpr int KL = KD / 32, VL = VT / 32;  // direct loads of a wave per chunk
  static constexpr int kLoads = KL + VL;
  Lds& lds;
  int mine, li, lg, kp;
  f32x4 S[RT][NC], next[RT][NC];
  uint4 keys[RT][2][kParts];  // the chunk's keys under their decays, transposed, in parts
  Neg neg;
  const uint16_t *knext, *vnext;  // of the first token that no load has asked for (uniform)
  int64_t ldk, ldv;
  bool keys_once;  // no other workgroup reads these keys
  uint32_t koff[KL], voff[VL];

  __device__ __forceinline__ StateWave(Lds& l, int wave) : lds(l), mine(wave) {
    const int lane = threadIdx.x & 63;
    li = lane & 15;
    lg = lane >> 4;
    kp = RT == 1 ? wave >> 1 : wave;  // the wave's block of 32 keys
    neg = neg_consts();
  }
  __device__ __forceinline__ int half_of(int rt) const { return RT == 1 ? mine & 1 : rt; }
  __device__ __forceinline__ int key0(int rt) const { return 32 * kp + 8 * lg + 4 * half_of(rt); }
  __device__ __forceinline__ int col_of(int c) const {
    return 32 * (c >> 1) + 8 * (li >> 2) + 4 * (c & 1) + (li & 3);
  }
  __device__ __forceinline__ void load(const float* from, int64_t V) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          S[rt][c][i] = from ? from[(key0(rt) + i) * V + col_of(c)] : 0.f;
  }
  __device__ __forceinline__ void store(float* to, int64_t V) const {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) to[(key0(rt) + i) * V + col_of(c)] = S[rt][c][i];
  }

  // The rows that this wave's direct loads bring, from the piece's first token on.
  __device__ __forceinline__ void aim(const uint16_t* k, const uint16_t* v, int64_t lk, int64_t lv,
                                      bool once) {
    knext = k;
    vnext = v;
    ldk = lk;
    ldv = lv;
    keys_once = once;
#pragma unroll
    for (int i = 0; i < KL; ++i) koff[i] = key_offset(i, kChunk);
#pragma unroll
    for (int i = 0; i < VL; ++i) voff[i] = value_offset(i, kChunk);
  }
  // Bytes from a chunk's first row to the lane's part of load i; of a chunk of n tokens rows behind them
  // read the last token again (their keys are dropped from the state).
  __device__ __forceinline__ uint32_t key_offset(int i, int n) const {
    const int lane = threadIdx.x & 63, r = 64 / (KD / 8) * (4 * i + mine) + lane / (KD / 8);
    return 2 * (min(r, n - 1) * uint32_t(ldk) + 8 * ((lane % (KD / 8)) ^ turn<KD>(r)));
  }
  __device__ __forceinline__ uint32_t value_offset(int i, int n) const {
    const int lane = threadIdx.x & 63, r = 64 / (VT / 8) * (4 * i + mine) + lane / (VT / 8);
    return 2 * (min(r, n - 1) * uint32_t(ldv) + 8 * ((lane % (VT / 8)) ^ turn<VT>(r)));
  }
  // The direct loads of the next chunk, which has n tokens and goes to ring slot `slot`.
  __device__ __forceinline__ void issue(int slot, int n) {
    auto& st = lds.ring[slot];
    if (n < kChunk) {  // (a piece's last one)
#pragma unroll
      for (int i = 0; i < KL; ++i) koff[i] = key_offset(i, n);
#pragma unroll
      for (int i = 0; i < VL; ++i) voff[i] = value_offset(i, n);
    }
    const uint32_t to = lds_at(st.k) + 1024 * mine;
    if (kOutputs && keys_once) {
#pragma unroll
      for (int i = 0; i < KL; ++i) to_lds16<true>(knext, koff[i], to + 4096 * i);
    } else {
#pragma unroll
      for (int i = 0; i < KL; ++i) to_lds16<false>(knext, koff[i], to + 4096 * i);
    }
#pragma unroll
    for (int i = 0; i < VL; ++i)
      to_lds16<kOutputs>(vnext, voff[i], lds_at(st.v) + 1024 * mine + 4096 * i);
    knext += kChunk * ldk;
    vnext += kChunk * ldv;
  }

  // The state's bf16 parts, before chunk c.
  __device__ __forceinline__ void publish(int c) {
    uint4* to = lds.state[c & 1];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int ct = 0; ct < NC; ++ct) {
        uint32_t a[kParts], b[kParts];
        split_pair<kParts>(S[rt][ct][0], S[rt][ct][1], a, neg);
        split_pair<kParts>(S[rt][ct][2], S[rt][ct][3], b, neg);
#pragma unroll
        for (int p = 0; p < kParts; ++p)
          reinterpret_cast<uint2*>(
              &to[((p * NP + kp) * NC + ct) * 64 + (threadIdx.x & 63)])[half_of(rt)] =
              make_uint2(a[p], b[p]);
      }
  }

  // The decayed keys of chunk c.
  __device__ __forceinline__ void prepare(int c) {
    const uint16_t* sk = reinterpret_cast<const uint16_t*>(lds.ring[unsigned(c) % R].k);
    const auto& dec = lds.decays[unsigned(c) % Lds::kDecays];
    uint2 kt[RT][2][2];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int r = 32 * b + 8 * lg + (li >> 2);
        const int key = 32 * kp + 4 * half_of(rt) + 8 * (li & 3);
        kt[rt][b][0] = ld_tr(sk + at<KD>(r, key));
        kt[rt][b][1] = ld_tr(sk + at<KD>(r + 4, key));
      }
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const f32x4 l0 = *reinterpret_cast<const f32x4*>(&dec.left[32 * b + 8 * lg]);
      const f32x4 l1 = *reinterpret_cast<const f32x4*>(&dec.left[32 * b + 8 * lg + 4]);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const uint4 k8 = make_uint4(kt[rt][b][0].x, kt[rt][b][0].y, kt[rt][b][1].x, kt[rt][b][1].y);
        float kd[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) kd[j] = elem(k8, j) * (j < 4 ? l0[j & 3] : l1[j & 3]);
        split_eight<kParts>(kd, keys[rt][b], neg);
      }
    }
  }

  // next = the state behind chunk c; false in some lane where it is not finite.
  __device__ __forceinline__ bool add(int c) {
    const uint16_t* sv = reinterpret_cast<const uint16_t*>(lds.ring[unsigned(c) % R].v);
    const float all = lds.decays[unsigned(c) % Lds::kDecays].all;
    uint4 vf[2][NC];  // V: columns li of tile ct, tokens 32 b + 8 lg ..
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int ct = 0; ct < NC; ++ct) {
        const int r = 32 * b + 8 * lg + (li >> 2);
        const int col = 32 * (ct >> 1) + 4 * (ct & 1) + 8 * (li & 3);
        const uint2 x = ld_tr(sv + at<VT>(r, col)), z = ld_tr(sv + at<VT>(r + 4, col));
        vf[b][ct] = make_uint4(x.x, x.y, z.x, z.y);
      }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int ct = 0; ct < NC; ++ct)
#pragma unroll
        for (int i = 0; i < 4; ++i) next[rt][ct][i] = S[rt][ct][i] * all;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int part = kParts - 1; part >= 0; --part)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int ct = 0; ct < NC; ++ct)
            next[rt][ct] = mma32(keys[rt][b][part], vf[b][ct], next[rt][ct]);
    f32x4 wrong = {0.f, 0.f, 0.f, 0.f};  // NaN as soon as an entry is not finite
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int ct = 0; ct < NC; ++ct)
#pragma unroll
        for (int i = 0; i < 4; ++i) wrong[i] = fmaf(next[rt][ct][i], 0.f, wrong[i]);
    const float any = (wrong[0] + wrong[1]) + (wrong[2] + wrong[3]);
    return any == any;
  }
  __device__ __forceinline__ void accept() {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int ct = 0; ct < NC; ++ct) S[rt][ct] = next[rt][ct];
  }
};

// A piece's place in the launch: false where there is nothing to do.
struct LinearItem {
  Piece pc;
  int64_t no, row;
  int head, tile;
};

template <int VT>
__device__ __forceinline__ bool find_item(const LinearSeqs& a, const wkv7_linear_io& io,
                                          LinearItem& it) {
  // Runs of neighbouring items (the tiles and heads that share q, k or a line of decays) on one XCD,
  // the runs dealt to the XCDs in turn: pieces that turn out empty are as many on each.
  const int tiles = io.V / VT;
  const int own = io.H / io.Hq * tiles, run = own * ((3 + own) / own);
  const unsigned at = blockIdx.x / kLinearXcds;
  int64_t item = (int64_t(at / run) * kLinearXcds + blockIdx.x % kLinearXcds) * run + at % run;
  if (item >= a.slots * io.H * tiles) return false;
  it.tile = int(item % tiles);
  item /= tiles;
  it.head = int(item % io.H);
  it.no = item / io.H;
  if (!find_piece(a, it.no, it.pc)) return false;
  it.row = a.slot_ids[it.pc.seq];
  return true;
}

// The value that a DPP control brings to this lane, or 0 where it brings none or the row is masked.
template <int kCtrl, int kRows = 0xf>
__device__ __forceinline__ double from_lane(double x) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, int(b), kCtrl, kRows, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, int(b >> 32), kCtrl, kRows, 0xf, false);
  return __builtin_bit_cast(double, uint64_t(hi) << 32 | lo);
}
__device__ __forceinline__ double lane_value(double x, int lane) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_readlane(int(b), lane);
  const uint32_t hi = __builtin_amdgcn_readlane(int(b >> 32), lane);
  return __builtin_bit_cast(double, uint64_t(hi) << 32 | lo);
}

// The decays of a chunk with n tokens, g the lane's token's: by one wave. Returns G_last. The sums
// are 64-bit, so that their differences are right for decays of any size.
template <class Decays>
__device__ __forceinline__ double sum_decays(Decays& d, float g, int n) {
  const int lane = threadIdx.x & 63;
  double G = lane < n ? double(g < -1e4f ? -1e4f : g) * kLog2e : 0.;
  G += from_lane<0x111>(G);  // 1, 2, 4, 8 lanes up within rows of 16
  G += from_lane<0x112>(G);
  G += from_lane<0x114>(G);
  G += from_lane<0x118>(G);
  G += from_lane<0x142, 0xa>(G);  // the last lane of a row to the next, of two rows to the next two
  G += from_lane<0x143, 0xc>(G);
  const double last = lane_value(G, 63);
  const float hi = float(G);
  d.hi[lane] = hi;
  d.lo[lane] = float(G - double(hi));
  d.left[lane] = lane < n ? __builtin_amdgcn_exp2f(float(last - G)) : 0.f;
  d.raw[lane] = g;
  if (lane == 0) d.all = __builtin_amdgcn_exp2f(float(last));
  return last;
}

// A piece once more, token by token as the formula is written, by the four state waves: where a product
// passed fp32 before its decay (a query with a key or with the state, or a factor of growth), which the
// formula need not. A thread has a column and KD / P keys, whose states are in LDS. One barrier and
// then one for each token, as the output waves have. (1.0 us a token of 64 keys, 1.8 of 128.)
template <int KD, int VT, bool kF32>
__device__ __forceinline__ void one_by_one(float* lds, const wkv7_linear_io& io, const Piece& pc,
                                           int head, int col0, const float* initial, float* state) {
  constexpr int P = 256 / VT, J = KD / P;
  const int col = threadIdx.x % VT, key0 = threadIdx.x / VT * J;
  float* S = lds + key0 * VT + col;
  barrier_vm<0>();  // (what other threads have stored, before it is stored again)
#pragma unroll 1
  for (int j = 0; j < J; ++j) S[j * VT] = initial ? initial[int64_t(key0 + j) * io.V + col] : 0.f;
  const int64_t ko = head / (io.H / io.Hq) * KD + key0, vo = int64_t(head) * io.V + col0 + col;
#pragma unroll 1
  for (int64_t t = pc.beg; t < pc.end; ++t) {
    const float d = expf(io.log_decay[t * io.ld_decay + head]);
    const float v = bf16_to_f32(io.v[t * io.ldv + vo]);
    float y = 0.f;
#pragma unroll 1
    for (int j = 0; j < J; ++j) {
      const float s = fmaf(d, S[j * VT], bf16_to_f32(io.k[t * io.ldk + ko + j]) * v);
      y = fmaf(bf16_to_f32(io.q[t * io.ldq + ko + j]) * io.scale, s, y);
      S[j * VT] = s;
    }
    float* sums = lds + KD * VT + (t & 1) * (P * VT) + col;
    sums[threadIdx.x / VT * VT] = y;
    barrier_lds();
    if (threadIdx.x >= VT) continue;
    for (int p = 1; p < P; ++p) y += sums[p * VT];
    const int64_t o = t * io.H * io.V + vo;
    if (kF32) static_cast<float*>(io.y)[o] = y;
    else static_cast<uint16_t*>(io.y)[o] = f32_to_bf16(y);
  }
#pragma unroll 1
  for (int j = 0; j < J && pc.last; ++j) state[int64_t(key0 + j) * io.V + col] = S[j * VT];
}

// Outputs. Waves 0 .. 3 are the state waves, 4 .. 7 and 8 .. 11 the output waves of the even and of
// the odd chunks. Few workgroups: a tick of 1.2 us (64 keys, 32 columns) is the state waves' chain of
// split, products and decayed keys. All units busy: memory, in rows of 128 bytes a token (8 x 4,096 tokens
// x 32 heads 134 to 141 us by card, 4 TB/s of q, k, v and y; vector units busy for 48 and matrix units
// for 27 % of the cycles, at 2.2 GHz; an earlier form took a third less without the outputs and no less
// without the chain). With one group of output waves and two workgroups on a unit the state waves wait for the outputs (a
// third slower).
template <int KD, int VT, bool kF32, int R>
__global__ __launch_bounds__(768) void linear_prefill_kernel(const LinearSeqs a,
                                                             const wkv7_linear_io io) {
  using State = StateWave<KD, VT, true, R>;
  using Lds = typename State::Lds;
  constexpr int NP = State::NP, NC = State::NC, RT = State::RT;
  // Chunk c is asked for in tick c - 1 - kAhead, has landed when tick c - 2 ends (its keys are read
  // from tick c - 1) and is read until tick c + 2.
  constexpr int kAhead = R - 4;
  __shared__ Lds lds;

  const int lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  LinearItem it;
  if (!find_item<VT>(a, io, it)) return;
  const Piece& pc = it.pc;
  const int64_t V = io.V, row = it.row, head = it.head;
  const int col0 = VT * it.tile;
  if (row < 0 || row >= a.rows) {  // no state is touched, the outputs are zero
    for (int64_t t = pc.beg + wave; t < pc.end; t += 12) {
      const int64_t o = (t * io.H + head) * V + col0 + lane;
      if (lane >= VT) continue;
      if (kF32) static_cast<float*>(io.y)[o] = 0.f;
      else static_cast<uint16_t*>(io.y)[o] = 0;
    }
    return;
  }
  float* slot_state = a.state + (row * io.H + head) * (KD * V) + col0;
  const int tokens = int(pc.end - pc.beg);
  const int chunks = (tokens + kChunk - 1) / kChunk;
  auto count = [&](int c) { return min(kChunk, tokens - kChunk * c); };
  const int hq = it.head / (io.H / io.Hq);
  const uint16_t* qbase = io.q + pc.beg * io.ldq + hq * KD;

  if (wave < 4) {
    State sw(lds, wave);
    if (tokens == 0) {
      if (a.zero_init) {
        sw.load(nullptr, V);
        sw.store(slot_state, V);
      }
      return;
    }
    sw.aim(io.k + pc.beg * io.ldk + hq * KD, io.v + pc.beg * io.ldv + head * V + col0, io.ldk, io.ldv,
           io.H == io.Hq && V == VT);
    if (threadIdx.x < 4) lds.bad[threadIdx.x] = 0;
    if (threadIdx.x == 0) lds.again = 0;
#pragma unroll
    for (int c = 0; c <= kAhead; ++c)
      if (c < chunks) sw.issue(c, count(c));
    const float* initial = a.piece ? a.pieces + (it.no * io.H + head) * (KD * V) + col0
                                   : a.zero_init ? nullptr : slot_state;
    sw.load(initial, V);
    barrier_vm<0>();
    sw.prepare(0);
    for (int c = 0; c < chunks; ++c) {
      const bool more = c + 1 + kAhead < chunks;
      if (more) sw.issue(int(unsigned(c + 1 + kAhead) % R), count(c + 1 + kAhead));
      sw.publish(c);
      if (threadIdx.x == 0) lds.bad[(c + 2) & 3] = 0;
      if (__ballot(!sw.add(c)) && lane == 0) lds.bad[c & 3] = 1;
      if (c + 1 < chunks) sw.prepare(c + 1);
      if (more) barrier_vm<(kAhead - 1) * State::kLoads>();
      else barrier_vm<0>();
      if (!__builtin_amdgcn_readfirstlane(lds.bad[c & 3])) {
        sw.accept();
        continue;
      }
      // Something in the chunk is not finite: products of whole tiles would carry it to tokens
      // before it (0 times infinity). Token by token instead, as the formula is written.
      const auto& st = lds.ring[unsigned(c) % R];
      const uint16_t* sk = reinterpret_cast<const uint16_t*>(st.k);
      const uint16_t* sv = reinterpret_cast<const uint16_t*>(st.v);
      const int n = count(c);
      for (int t = 0; t < n; ++t) {
        const float d = expf(lds.decays[unsigned(c) % Lds::kDecays].raw[t]);
        const uint16_t* q = qbase + (int64_t(kChunk) * c + t) * io.ldq;
        float part[NC] = {};
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = sw.key0(rt) + i;
            const float kv = bf16_to_f32(sk[at<KD>(t, key)]);
            const float qv = bf16_to_f32(q[key]) * io.scale;
#pragma unroll
            for (int ct = 0; ct < NC; ++ct) {
              const float v = bf16_to_f32(sv[at<VT>(t, sw.col_of(ct))]);
              sw.S[rt][ct][i] = fmaf(d, sw.S[rt][ct][i], kv * v);
              part[ct] = fmaf(qv, sw.S[rt][ct][i], part[ct]);
            }
          }
#pragma unroll
        for (int ct = 0; ct < NC; ++ct) {
          part[ct] += __shfl_xor(part[ct], 16);
          part[ct] += __shfl_xor(part[ct], 32);
          if (lg == 0) lds.part[t & 1][wave][sw.col_of(ct)] = part[ct];
        }
        barrier_lds();
        if (threadIdx.x < VT) {
          const float(*p)[VT] = lds.part[t & 1];
          const float v = (p[0][lane] + p[1][lane]) + (p[2][lane] + p[3][lane]);
          const int64_t o = ((pc.beg + int64_t(kChunk) * c + t) * io.H + head) * V + col0 + lane;
          if (kF32) static_cast<float*>(io.y)[o] = v;
          else static_cast<uint16_t*>(io.y)[o] = f32_to_bf16(v);
        }
      }
    }
    // The state is stored before all outputs are known to stand, unless it replaces the one they
    // began with.
    if (pc.last && initial != slot_state) sw.store(slot_state, V);
    barrier_lds();
    if (__builtin_amdgcn_readfirstlane(lds.again))
      one_by_one<KD, VT, kF32>(reinterpret_cast<float*>(lds.ring), io, pc, it.head, col0, initial,
                               slot_state);
    else if (pc.last && initial == slot_state)
      sw.store(slot_state, V);
    return;
  }

  // -- output waves --------------------------------------------------------------------------
  if (tokens == 0) return;
  const int group = (wave - 4) >> 2, w = wave & 3;
  const int tw = 16 * w + li;  // the lane's token of a chunk
  const float* gbase = io.log_decay + pc.beg * io.ld_decay + head;
  const int64_t lastt = tokens - 1;
  auto load_g = [&](int c) { return gbase[min(int64_t(kChunk) * c + lane, lastt) * io.ld_decay]; };
  const Neg neg = neg_consts();
  float g = 0.f;  // the lane's decay in the group's next chunk
  if (w == 0) {
    const float now = load_g(group);
    g = load_g(group + 2);
    if (group < chunks) sum_decays(lds.decays[group], now, count(group));
  }
  uint4 qf[NP], qn[NP];  // the lane's query row of the group's chunk and of its next one
  auto load_q = [&](uint4 (&to)[NP], int c) {
    const uint16_t* q = qbase + min(int64_t(kChunk) * c + tw, lastt) * io.ldq + 8 * lg;
#pragma unroll
    for (int p = 0; p < NP; ++p) to[p] = ld16(q + 32 * p);
  };
  // The end of tick c; true if the state waves have written the outputs of chunk c.
  auto end_tick = [&](int c) {
    barrier_lds();
    const bool bad = __builtin_amdgcn_readfirstlane(lds.bad[c & 3]);
    if (bad)
      for (int i = 0; i < count(c); ++i) barrier_lds();
    return bad;
  };
  load_q(qn, group);
  barrier_lds();
  if (group == 1) end_tick(0);

  f32x4 y[NC];
  uint4 own[kParts];  // the parts of the scores with the wave's own block of 32 tokens
  const int blk = w >> 1;
  bool skip = true;  // nothing to finish
  f32x4 wrong = {0.f, 0.f, 0.f, 0.f};  // NaN as soon as an output is not finite
  // Scores with the 32 tokens of block b of chunk c, as an operand's rows.
  auto scores = [&](const uint16_t* sk, int b, f32x4 (&sc)[2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      sc[h] = f32x4{0.f, 0.f, 0.f, 0.f};
      const int kr = 32 * b + 8 * (li >> 2) + 4 * h + (li & 3);
#pragma unroll
      for (int p = 0; p < NP; ++p)
        sc[h] = mma32(ld16(sk + at<KD>(kr, 32 * p + 8 * lg)), qf[p], sc[h]);
    }
  };
  auto begin = [&](int c) {
    const auto& dec = lds.decays[unsigned(c) % Lds::kDecays];
    const uint16_t* sk = reinterpret_cast<const uint16_t*>(lds.ring[unsigned(c) % R].k);
    const uint4* sp = lds.state[c & 1];
    f32x4 sc[2];
    scores(sk, blk, sc);
#pragma unroll
    for (int ct = 0; ct < NC; ++ct) y[ct] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int part = kParts - 1; part >= 0; --part)
#pragma unroll
      for (int p = 0; p < NP; ++p)
#pragma unroll
        for (int ct = 0; ct < NC; ++ct)
          y[ct] = mma32(sp[((part * NP + p) * NC + ct) * 64 + lane], qf[p], y[ct]);
    const float thi = dec.hi[tw], tlo = dec.lo[tw];
    float p8[8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int s0 = 32 * blk + 8 * lg + 4 * h;
      const f32x4 shi = *reinterpret_cast<const f32x4*>(&dec.hi[s0]);
      const f32x4 slo = *reinterpret_cast<const f32x4*>(&dec.lo[s0]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float e = __builtin_amdgcn_exp2f((thi - shi[i]) + (tlo - slo[i]));
        const float x = sc[h][i] * io.scale * e;
        p8[4 * h + i] = s0 + i <= tw ? x : 0.f;
      }
    }
    split_eight<kParts>(p8, own, neg);
    const float es = __builtin_amdgcn_exp2f(thi + tlo) * io.scale;
#pragma unroll
    for (int ct = 0; ct < NC; ++ct)
#pragma unroll
      for (int i = 0; i < 4; ++i) y[ct][i] *= es;
  };
  auto finish = [&](int c) {
    const auto& st = lds.ring[unsigned(c) % R];
    const auto& dec = lds.decays[unsigned(c) % Lds::kDecays];
    const uint16_t* sk = reinterpret_cast<const uint16_t*>(st.k);
    const uint16_t* sv = reinterpret_cast<const uint16_t*>(st.v);
    auto values = [&](int b, const uint4 (&pf)[kParts]) {
      const int r = 32 * b + 8 * lg + (li >> 2);
#pragma unroll
      for (int ct = 0; ct < NC; ++ct) {
        const int col = 32 * (ct >> 1) + 4 * (ct & 1) + 8 * (li & 3);
        const uint2 x = ld_tr(sv + at<VT>(r, col)), z = ld_tr(sv + at<VT>(r + 4, col));
        const uint4 vf = make_uint4(x.x, x.y, z.x, z.y);
#pragma unroll
        for (int part = kParts - 1; part >= 0; --part) y[ct] = mma32(vf, pf[part], y[ct]);
      }
    };
    values(blk, own);
    if (blk) {  // the first block, all of it before the wave's tokens
      f32x4 sc[2];
      float p8[8];
      uint4 before[kParts];
      scores(sk, 0, sc);
      const float thi = dec.hi[tw], tlo = dec.lo[tw];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const f32x4 shi = *reinterpret_cast<const f32x4*>(&dec.hi[8 * lg + 4 * h]);
        const f32x4 slo = *reinterpret_cast<const f32x4*>(&dec.lo[8 * lg + 4 * h]);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          p8[4 * h + i] = sc[h][i] * io.scale *
                          __builtin_amdgcn_exp2f((thi - shi[i]) + (tlo - slo[i]));
      }
      split_eight<kParts>(p8, before, neg);
      values(0, before);
    }
    uint4 out[NC / 2];
#pragma unroll
    for (int h = 0; h < NC / 2; ++h) {
      const f32x4 &x0 = y[2 * h], &x1 = y[2 * h + 1];
      out[h] = make_uint4(pack_bf16(x0[0], x0[1]), pack_bf16(x0[2], x0[3]),
                          pack_bf16(x1[0], x1[1]), pack_bf16(x1[2], x1[3]));
      wrong = mma32(out[h], make_uint4(0, 0, 0, 0), wrong);
    }
    const int t = kChunk * c + tw;
    if (t < tokens) {
      const int64_t o = ((pc.beg + t) * io.H + head) * V + col0 + 8 * lg;
#pragma unroll
      for (int h = 0; h < NC / 2; ++h) {
        if (kF32) {
          f32x4* p = reinterpret_cast<f32x4*>(static_cast<float*>(io.y) + o + 32 * h);
          p[0] = y[2 * h];
          p[1] = y[2 * h + 1];
        } else {
          *reinterpret_cast<uint4*>(static_cast<uint16_t*>(io.y) + o + 32 * h) = out[h];
        }
      }
    }
  };
  for (int c = group; c < chunks; c += 2) {
    // tick c
    if (!skip) finish(c - 2);
#pragma unroll
    for (int p = 0; p < NP; ++p) qf[p] = qn[p];
    if (w == 0 && c + 2 < chunks) {
      sum_decays(lds.decays[unsigned(c + 2) % Lds::kDecays], g, count(c + 2));
      g = load_g(c + 4);
    }
    // an infinite or NaN query: its products with the state's parts are not the formula's
    f32x4 zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int p = 0; p < NP; ++p) zero = mma32(qf[p], make_uint4(0, 0, 0, 0), zero);
    const float any = (zero[0] + zero[1]) + (zero[2] + zero[3]);
    if (__ballot(any != any) && lane == 0) lds.bad[c & 3] = 1;
    skip = end_tick(c);
    // tick c + 1
    load_q(qn, c + 2);
    if (!skip) begin(c);
    if (c + 1 < chunks) end_tick(c + 1);
  }
  if (!skip) finish(chunks - 1 - ((chunks - 1 - group) & 1));
  const float any = (wrong[0] + wrong[1]) + (wrong[2] + wrong[3]);
  if (any != any) lds.again = 1;
  barrier_lds();
  if (__builtin_amdgcn_readfirstlane(lds.again)) {
    barrier_vm<0>();  // (the outputs' stores before those of the state waves)
    for (int t = 0; t < tokens; ++t) barrier_lds();
  }
}

// A piece's final state from zero and the sum of its decays, for a piece that is not its sequence's
// last: the four state waves and one for the decays. With no outputs to wait for, the decayed keys of
// chunk c + 1 are made behind the products of chunk c (1 x 16,384 tokens x 12 heads, pieces of 832: 18.6
// us, 1.0 per chunk and a fill of 5).
template <int KD, int VT, int R>
__global__ __launch_bounds__(320) void linear_states_kernel(const LinearSeqs a,
                                                            const wkv7_linear_io io) {
  using State = StateWave<KD, VT, false, R>;
  constexpr int kAhead = R - 2;  // (as for the outputs, without their ticks behind)
  __shared__ typename State::Lds lds;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  LinearItem it;
  if (!find_item<VT>(a, io, it)) return;
  const Piece& pc = it.pc;
  if (pc.last || it.row < 0 || it.row >= a.rows) return;
  const int64_t V = io.V, head = it.head;
  const int col0 = VT * it.tile;
  const int tokens = int(pc.end - pc.beg);  // (a whole piece)
  const int chunks = (tokens + kChunk - 1) / kChunk;
  auto count = [&](int c) { return min(kChunk, tokens - kChunk * c); };
  if (wave < 4) {
    const int hq = it.head / (io.H / io.Hq);
    State sw(lds, wave);
    sw.aim(io.k + pc.beg * io.ldk + hq * KD, io.v + pc.beg * io.ldv + head * V + col0, io.ldk, io.ldv,
           false);
#pragma unroll
    for (int c = 0; c <= kAhead; ++c)
      if (c < chunks) sw.issue(c, count(c));
    sw.load(nullptr, V);
    barrier_vm<0>();
    sw.prepare(0);
    for (int c = 0; c < chunks; ++c) {
      const bool more = c + 1 + kAhead < chunks;
      if (more) sw.issue(int(unsigned(c + 1 + kAhead) % R), count(c + 1 + kAhead));
      // (as for the outputs, but a wave's keys are its own: it decides by itself)
      const bool bad = __ballot(!sw.add(c));
      if (c + 1 < chunks) sw.prepare(c + 1);
      if (!bad) sw.accept();
      const auto& st = lds.ring[unsigned(c) % R];
      const uint16_t* sk = reinterpret_cast<const uint16_t*>(st.k);
      const uint16_t* sv = reinterpret_cast<const uint16_t*>(st.v);
      for (int t = 0; bad && t < count(c); ++t) {
        const float d = expf(lds.decays[unsigned(c) % State::Lds::kDecays].raw[t]);
#pragma unroll
        for (int rt = 0; rt < State::RT; ++rt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float kv = bf16_to_f32(sk[at<KD>(t, sw.key0(rt) + i)]);
#pragma unroll
            for (int ct = 0; ct < State::NC; ++ct)
              sw.S[rt][ct][i] = fmaf(d, sw.S[rt][ct][i],
                                     kv * bf16_to_f32(sv[at<VT>(t, sw.col_of(ct))]));
          }
      }
      if (more) barrier_vm<(kAhead - 1) * State::kLoads>();
      else barrier_vm<0>();
    }
    sw.store(a.pieces + (it.no * io.H + head) * (KD * V) + col0, V);
    return;
  }
  const float* gbase = io.log_decay + pc.beg * io.ld_decay + head;
  auto load_g = [&](int c) {
    return gbase[min(int64_t(kChunk) * c + lane, int64_t(tokens - 1)) * io.ld_decay];
  };
  const float now[2] = {load_g(0), load_g(1)};
  float g = load_g(2), after = load_g(3);  // (64 lines of memory: they may take longer than a tick)
  double sum = sum_decays(lds.decays[0], now[0], count(0));
  // some token's factor is 0 in fp32 (lanes past a chunk's end have the last token's)
  bool forgets = expf(now[0]) == 0.f || expf(now[1]) == 0.f;
  if (chunks > 1) sum += sum_decays(lds.decays[1], now[1], count(1));
  barrier_lds();
  for (int c = 0; c < chunks; ++c) {
    if (c + 2 < chunks) {
      sum += sum_decays(lds.decays[unsigned(c + 2) % State::Lds::kDecays], g, count(c + 2));
      forgets |= expf(g) == 0.f;
      g = after;
      after = load_g(c + 4);
    }
    barrier_lds();
  }
  const bool any = __ballot(forgets);
  if (it.tile == 0 && lane == 0) a.sums[it.no * io.H + head] = any ? -INFINITY : sum;
}

// e^(sum) x + add for a sum of log2 decays over any number of tokens (-infinity: a token forgot x). The
// power of two is applied by itself, so that the factor passes no range that x or the result does not;
// an infinite x stays so under any decay, but not behind a token that forgot it (0 times infinity).
__device__ __forceinline__ float decayed(float x, double sum, float add) {
  if (sum == -INFINITY) return fmaf(0.f, x, add);
  const double in = fmin(fmax(sum, -400.), 400.), whole = __builtin_floor(in);
  const float part = sum == sum ? __builtin_amdgcn_exp2f(float(in - whole)) : NAN;
  return fmaf(part, ldexpf(x, int(whole)), add);
}

// From the pieces' local final states to their initial states, in order, four entries per thread:
// S_in(0) is the sequence's initial state, S_in(g + 1) = e^(sum of g) S_in(g) + S_local(g). Eight
// pieces' states are read at once: it is a chain of waits for memory (20 pieces of 12 heads 7.4 us).
template <int KD>
__global__ __launch_bounds__(kChainThreads) void linear_chain_kernel(const LinearSeqs a,
                                                                      const wkv7_linear_io io) {
  constexpr int U = 8;
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
  const int64_t first = first_piece(a, s), step = io.H * size;
  float* p = a.pieces + (first * io.H + head) * size + e;
  const double* sums = a.sums + first * io.H + head;
  for (int64_t g0 = 0; g0 < n; g0 += U) {
    f32x4 local[U];
    double sum[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t g = min(g0 + u, n - 1);
      const bool whole = g + 1 < n;  // (the last piece's are not computed)
      local[u] = whole ? *reinterpret_cast<const f32x4*>(p + g * step) : run;
      sum[u] = whole ? sums[g * io.H] : 0.;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (g0 + u >= n) break;
      *reinterpret_cast<f32x4*>(p + (g0 + u) * step) = run;
#pragma unroll
      for (int i = 0; i < 4; ++i) run[i] = decayed(run[i], sum[u], local[u][i]);
    }
  }
}

}  // namespace
}  // namespace wkv7
