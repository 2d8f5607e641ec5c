// Linear attention with a decay for each head, over the slot pool: per token and head
//   S <- e^g S + k v^T,   y = scale q^T S        (S [K, V] fp32, q, k, v bf16)
//
// wkv7_linear_decode: one token per slot, in place. wkv7_linear_prefill: ragged sequences, in
// chunks of 64 tokens on the matrix cores. With G_t the sum of the chunk's log-decays up to token t,
//   P[t][s] = scale (q_t . k_s) e^(G_t - G_s)  for s <= t, else 0
//   y       = P V + scale e^(G_t) Q S
//   S'      = e^(G_last) S + (e^(G_last - G_s) k_s)^T V
// Every exponent is a difference of sums inside the chunk, taken in 64 bits. Where a product passes
// fp32 before its decay, which the formula need not, the sequence's outputs are computed once more
// token by token, as are those of a chunk with an infinity or NaN.
#include <algorithm>

#include "wkv7_linear_core.h"

using namespace wkv7;

namespace wkv7 {
namespace {

constexpr int kDecodeWaves = 4;
constexpr int64_t kLinearMaxLd = int64_t(1) << 24;

// One (batch row, head, 64 value columns) of a decode step: lane i owns a column, wave w K / 4 key
// rows, so that every access of the state is a whole 256-byte run. The state is read and written
// once, without being kept in the caches. HBM bounds it: 256 rows x 32 heads of 64 x 64 in 44.6 us, 6.1
// TB/s of state; 61 rows x 16 heads of 128 x 128 in 23 us, 5.6 TB/s.
template <int KD, bool kF32>
__global__ __launch_bounds__(64 * kDecodeWaves) void linear_decode_kernel(
    float* __restrict__ state, int64_t rows, const int32_t* __restrict__ slot_ids,
    const int32_t* __restrict__ row_order, int B, const wkv7_linear_io io) {
  constexpr int KR = KD / kDecodeWaves;  // key rows of a wave
  __shared__ float2 s_kq[KD];            // (k, scale q)
  __shared__ float s_y[kDecodeWaves][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int tiles = io.V / 64;
  int64_t item = blockIdx.x;
  const int tile = int(item % tiles);
  item /= tiles;
  const int head = int(item % io.H);
  int64_t row = item / io.H;
  if (row_order) {
    row = row_order[row];
    if (row < 0 || row >= B) return;  // uniform: the whole block skips
  }
  const int64_t slot = slot_ids[row];
  const int col = 64 * tile + lane;
  const int64_t out = (row * io.H + head) * io.V + col;
  if (slot < 0 || slot >= rows) {  // uniform: no state is touched, the output is zero
    if (wave == 0) {
      if (kF32) static_cast<float*>(io.y)[out] = 0.f;
      else static_cast<uint16_t*>(io.y)[out] = 0;
    }
    return;
  }
  // the vectors before the state, whose arrival the arithmetic on them then does not wait for
  const int j0 = KR * wave;
  const int hq = head / (io.H / io.Hq);
  const int64_t jo = int64_t(hq) * KD + j0 + (lane & (KR - 1));
  const uint16_t qb = io.q[row * io.ldq + jo], kb = io.k[row * io.ldk + jo];
  const uint16_t vb = io.v[row * io.ldv + int64_t(head) * io.V + col];
  const float g = io.log_decay[row * io.ld_decay + head];
  __builtin_amdgcn_sched_barrier(0);
  float* hp = state + ((slot * io.H + head) * KD + j0) * io.V + col;
  float h[KR];
#pragma unroll
  for (int j = 0; j < KR; ++j) h[j] = __builtin_nontemporal_load(hp + int64_t(j) * io.V);
  asm volatile("" ::"v"(qb), "v"(kb), "v"(vb), "v"(g));
  if (lane < KR)  // (its own wave's rows: no barrier)
    s_kq[j0 + lane] = make_float2(bf16_to_f32(kb), bf16_to_f32(qb) * io.scale);
  const float d = expf(g), v = bf16_to_f32(vb);
  __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
  float y0 = 0.f, y1 = 0.f;
#pragma unroll
  for (int j = 0; j < KR; ++j) {
    const float2 c = s_kq[j0 + j];
    const float hn = fmaf(d, h[j], c.x * v);
    __builtin_nontemporal_store(hn, hp + int64_t(j) * io.V);
    if (j & 1) y1 = fmaf(c.y, hn, y1);
    else y0 = fmaf(c.y, hn, y0);
  }
  s_y[wave][lane] = y0 + y1;
  __syncthreads();
  if (wave == 0) {
    const float y = (s_y[0][lane] + s_y[1][lane]) + (s_y[2][lane] + s_y[3][lane]);
    if (kF32) static_cast<float*>(io.y)[out] = y;
    else static_cast<uint16_t*>(io.y)[out] = f32_to_bf16(y);
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// The checks of both entry points, for `tokens` > 0 where the pointers are needed.
int validate(const float* state, int64_t rows, int64_t tokens, const wkv7_linear_io* io) {
  if (!io || rows < 1 || tokens < 0) return WKV7_ERR_ARG;
  if (io->H < 1 || io->Hq < 1 || io->H % io->Hq) return WKV7_ERR_ARG;
  if (io->y_dtype != WKV7_Y_BF16 && io->y_dtype != WKV7_Y_F32) return WKV7_ERR_ARG;
  if ((io->K != 64 && io->K != 128) || io->V < 64 || io->V % 64 || io->V > WKV7_LINEAR_MAX_V)
    return WKV7_ERR_SHAPE;
  if (!state) return WKV7_ERR_ARG;
  if (!aligned16(state)) return WKV7_ERR_SHAPE;
  if (tokens == 0) return WKV7_OK;
  if (!io->q || !io->k || !io->v || !io->y || !io->log_decay) return WKV7_ERR_ARG;
  const int64_t qk = int64_t(io->Hq) * io->K, hv = int64_t(io->H) * io->V;
  if (io->ldq < qk || io->ldk < qk || io->ldv < hv || (io->ld_decay && io->ld_decay < io->H))
    return WKV7_ERR_SHAPE;
  if (io->ldq % 8 || io->ldk % 8 || io->ldv % 8 || !aligned16(io->q) || !aligned16(io->k) ||
      !aligned16(io->v) || !aligned16(io->y) || (reinterpret_cast<uintptr_t>(io->log_decay) & 3u))
    return WKV7_ERR_SHAPE;
  // (a chunk's rows are addressed by 32-bit offsets)
  if (io->ldk > kLinearMaxLd || io->ldv > kLinearMaxLd) return WKV7_ERR_SHAPE;
  return WKV7_OK;
}

int device_cus(int* cus) {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess ||
      hipDeviceGetAttribute(cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess)
    return launch_status();
  return WKV7_OK;
}

// Value columns of a workgroup of the outputs' kernel. Of 128 keys its LDS holds 32; of 64 keys it takes
// 64, or 32 where that leaves half of the units without one (512 tokens x 32 heads 18.6 and 15.0 us).
int value_tile(int32_t nseq, const wkv7_linear_io& io, int cus) {
  return io.K == 128 || 2 * int64_t(nseq) * io.H * (io.V / 64) <= cus ? 32 : 64;
}

// Tokens of a piece (a multiple of 64), or 0: no sequence is cut. A unit holds one workgroup of the
// outputs' kernel: as many pieces as leave none of them a second one, sequences of equal lengths
// assumed.
int64_t piece_tokens(int32_t nseq, int64_t tokens, const wkv7_linear_io& io, int cus) {
  const int64_t groups = int64_t(io.H) * (io.V / (io.K == 128 ? 32 : 64)) * nseq;
  const int64_t cuts = int64_t(cus) / groups;  // pieces of a sequence
  if (cuts < 2) return 0;
  // In chunks: a sequence in one piece takes about 6 us and 1.2 for each; in pieces 15 to 18 us and 3 for
  // each chunk of a piece (12 heads: 2,048 tokens in 8 pieces 25.7 us, 16,384 in 20 of 13 chunks 59).
  const int64_t chunks = (tokens + int64_t(nseq) * kChunk - 1) / (int64_t(nseq) * kChunk);
  const int64_t piece = std::max<int64_t>(kMinPiece / kChunk, (chunks + cuts - 1) / cuts);
  return chunks > 10 + 2 * piece ? piece * kChunk : 0;
}

// Numbers of pieces, as first_piece gives them out.
int64_t piece_slots(int32_t nseq, int64_t tokens, int64_t piece) {
  return piece ? tokens / piece + nseq : nseq;
}

size_t workspace_bytes_of(int64_t slots, const wkv7_linear_io& io) {
  return size_t(slots) * size_t(io.H) * (size_t(io.K) * size_t(io.V) * sizeof(float) +
                                         sizeof(double));
}

// Chunks of the outputs' ring: one asked for ahead. (More are no faster: 8 x 4,096 tokens x 32 heads 135.4
// us with five and with six, 512 tokens x 32 heads 15.0 and 15.1.)
constexpr int kRing = 5;

template <int KD, int VT, bool kF32>
int launch_prefill(const LinearSeqs& sq, const wkv7_linear_io& io, float* ws, int cus,
                   hipStream_t s) {
  LinearSeqs a = sq;
  auto grid = [&](int tile) {
    const int64_t items = a.slots * io.H * (io.V / tile);
    const int own = io.H / io.Hq * (io.V / tile);  // (as find_item deals them)
    const int64_t deal = int64_t(own) * ((3 + own) / own) * kLinearXcds;
    return (items + deal - 1) / deal * deal;
  };
  a.pieces = ws;
  a.sums = ws ? reinterpret_cast<double*>(ws + sq.slots * io.H * int64_t(io.K) * io.V) : nullptr;
  if (grid(32) > int64_t(0x7fffffff)) return WKV7_ERR_ARG;
  // Where a unit takes one workgroup after the other the long sequences go first (19 of up to 2,062
  // tokens, 16 heads of 128 x 128: 104.8 us, 109.9 as they come). Finding them costs a workgroup some 0.7
  // us, too much for short ones.
  a.longest_first = !a.piece && !a.order && a.nseq > 1 && a.nseq < 64 &&
                    a.tokens >= int64_t(256) * a.nseq && a.slots * io.H * (io.V / VT) > cus;
  if (a.piece) {
    linear_states_kernel<KD, 64, 4><<<unsigned(grid(64)), 320, 0, s>>>(a, io);
    int rc = launch_status();
    if (rc != WKV7_OK) return rc;
    const int64_t blocks = int64_t(a.nseq) * io.H * (KD * io.V / kChainElems);
    if (blocks > int64_t(0x7fffffff)) return WKV7_ERR_ARG;
    linear_chain_kernel<KD><<<unsigned(blocks), kChainThreads, 0, s>>>(a, io);
    rc = launch_status();
    if (rc != WKV7_OK) return rc;
  }
  linear_prefill_kernel<KD, VT, kF32, kRing><<<unsigned(grid(VT)), 768, 0, s>>>(a, io);
  return launch_status();
}

}  // namespace
}  // namespace wkv7

extern "C" int wkv7_linear_decode(float* state, int64_t num_rows, const int32_t* slot_ids,
                                  const int32_t* row_order, int32_t B, const wkv7_linear_io* io,
                                  void* stream) {
  const int rc = validate(state, num_rows, B, io);
  if (rc != WKV7_OK) return rc;
  if (B == 0) return WKV7_OK;
  if (!slot_ids) return WKV7_ERR_ARG;
  const int64_t blocks = int64_t(B) * io->H * (io->V / 64);
  if (blocks > int64_t(0x7fffffff)) return WKV7_ERR_ARG;
  auto launch = [&](auto kernel) {
    kernel<<<unsigned(blocks), 64 * kDecodeWaves, 0, as_stream(stream)>>>(
        state, num_rows, slot_ids, row_order, B, *io);
    return launch_status();
  };
  const bool f32 = io->y_dtype == WKV7_Y_F32;
  if (io->K == 64)
    return f32 ? launch(linear_decode_kernel<64, true>) : launch(linear_decode_kernel<64, false>);
  return f32 ? launch(linear_decode_kernel<128, true>) : launch(linear_decode_kernel<128, false>);
}

extern "C" size_t wkv7_linear_prefill_workspace_bytes(int32_t nseq, int64_t total_tokens,
                                                      const wkv7_linear_io* io) {
  if (!io || nseq < 1 || total_tokens < 1 || io->H < 1 || io->V < 64) return 0;
  int cus = 0;
  if (device_cus(&cus) != WKV7_OK) return 0;
  const int64_t piece = piece_tokens(nseq, total_tokens, *io, cus);
  return piece ? workspace_bytes_of(piece_slots(nseq, total_tokens, piece), *io) : 0;
}

extern "C" int wkv7_linear_prefill(float* state, int64_t num_rows, const int32_t* slot_ids,
                                   const int32_t* cu_seqlens, const int32_t* seq_order,
                                   int32_t nseq, int64_t total_tokens, const wkv7_linear_io* io,
                                   int32_t zero_init, void* workspace, size_t workspace_bytes,
                                   void* stream) {
  if (nseq < 0 || total_tokens > int64_t(0x7fffffff)) return WKV7_ERR_ARG;
  const int rc = validate(state, num_rows, total_tokens, io);
  if (rc != WKV7_OK) return rc;
  if (nseq == 0) return WKV7_OK;
  if (!slot_ids || !cu_seqlens) return WKV7_ERR_ARG;
  int cus = 0;
  const int drc = device_cus(&cus);
  if (drc != WKV7_OK) return drc;
  int64_t piece = piece_tokens(nseq, total_tokens, *io, cus);
  if (piece && (!workspace || !aligned16(workspace) ||
                workspace_bytes < workspace_bytes_of(piece_slots(nseq, total_tokens, piece), *io)))
    piece = 0;
  LinearSeqs sq{};
  sq.state = state;
  sq.rows = num_rows;
  sq.slot_ids = slot_ids;
  sq.cu = cu_seqlens;
  sq.order = seq_order;
  sq.nseq = nseq;
  sq.tokens = total_tokens;
  sq.zero_init = zero_init != 0;
  sq.piece = piece;
  sq.slots = piece_slots(nseq, total_tokens, piece);
  float* ws = piece ? static_cast<float*>(workspace) : nullptr;
  hipStream_t s = as_stream(stream);
  const bool f32 = io->y_dtype == WKV7_Y_F32;
  if (io->K == 128)
    return f32 ? launch_prefill<128, 32, true>(sq, *io, ws, cus, s)
               : launch_prefill<128, 32, false>(sq, *io, ws, cus, s);
  if (!piece && value_tile(nseq, *io, cus) == 32)
    return f32 ? launch_prefill<64, 32, true>(sq, *io, ws, cus, s)
               : launch_prefill<64, 32, false>(sq, *io, ws, cus, s);
  return f32 ? launch_prefill<64, 64, true>(sq, *io, ws, cus, s)
             : launch_prefill<64, 64, false>(sq, *io, ws, cus, s);
}
