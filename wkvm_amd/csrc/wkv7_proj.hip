// Grouped projection GEMMs for few rows (RWKV-7 time-mix decode batches):
//   y_g = act_g(x_g w_g^T + bias_g),  x_g [m, k] bf16, w_g [n, k] bf16 ([out, in]).
//
// At a few hundred rows each product of the block (r, k, v, o: 2048 x 2048;
// the LoRA stages: 2048 -> 64..256 -> 2048) is a thin GEMM whose weights
// take about 1 us to stream from HBM, while a separate library launch per
// product costs 4-13 us. One launch here covers up to 8 independent products:
// the workgroups of all groups form one grid, each computing a BM x BN output
// tile over the whole k.
//
// Workgroup: GM x GN waves (4, 8 or 16), each a (BM/GM) x (BN/GN) block of
// 16 x 16 accumulator tiles on v_mfma_f32_16x16x32_bf16. Operand layout of
// that instruction (lane l, li = l % 16, lg = l / 16): A lane holds
// A[li][8lg .. 8lg+7] of a 32-wide k block, B lane holds B[8lg .. 8lg+7][li],
// the accumulator holds D[4lg .. 4lg+3][li]. With x rows and w rows both
// k-contiguous, every operand register is one 16-byte chunk of one row.
// k advances BK (64 or 128) per stage through a ring of S LDS stages whose
// rows hold KC = BK / 8 chunks of 16 bytes, chunk c of row r at slot
// c ^ (r & (KC - 1)), so the 16 rows a fragment read touches spread over the
// banks. Stages are filled by direct global -> LDS loads (no register
// staging) issued S - 1 stages ahead and spread between the MFMAs of the
// stage being multiplied. One barrier per stage. Rows past m and columns past
// n load a clamped (valid) row and are not stored. Tiles are dealt to the
// XCDs in contiguous runs so that each XCD's L2 keeps the x rows it
// re-reads. With few tiles and long k, k can be split over several
// workgroups per tile (fp32 partials in a caller-provided workspace, summed
// in part order by proj_reduce_kernel). Up to 16 rows have a kernel of their own
// (proj_thin_kernel) where it is the faster one.
#include <mutex>

#include "wkv7_proj_plan.h"

using namespace wkv7;

namespace wkv7 {
namespace {

// Split-k partials of wkv7_proj_grouped_noalloc: a library-owned device array,
// one per GPU (each device holds its own copy until the process ends). Host
// code never passes the array's name to a kernel (on the host it is only a
// stand-in symbol); it passes the device address hipGetSymbolAddress returns
// for the current device, looked up once per device and kept below.
static __device__ __align__(256) float scratch[WKV7_PROJ_STATIC_SCRATCH_BYTES / sizeof(float)];

constexpr int kMaxDevices = 64;
std::mutex g_scratch_mutex;
void* g_scratch_ptr[kMaxDevices] = {};

// The current device's address of `scratch` (looked up on the first call made
// with that device current).
int scratch_address(float** out) {
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return static_cast<int>(e);
  if (dev < 0 || dev >= kMaxDevices) return WKV7_ERR_ARG;
  std::lock_guard<std::mutex> lock(g_scratch_mutex);
  if (!g_scratch_ptr[dev]) {
    void* p = nullptr;
    e = hipGetSymbolAddress(&p, HIP_SYMBOL(scratch));
    if (e != hipSuccess) return static_cast<int>(e);
    if (!p) return WKV7_ERR_WORKSPACE;
    g_scratch_ptr[dev] = p;
  }
  *out = static_cast<float*>(g_scratch_ptr[dev]);
  return WKV7_OK;
}

}  // namespace
}  // namespace wkv7

extern "C" size_t wkv7_proj_workspace_bytes(int64_t m, const wkv7_proj_group* groups,
                                            int32_t ngroups) {
  if (validate(m, groups, ngroups) != WKV7_OK || m == 0) return 0;
  int cus = 0;
  if (device_cus(&cus) != WKV7_OK) return 0;
  return make_plan(m, groups, ngroups, cus).ws_bytes;
}

extern "C" int wkv7_proj_grouped(int64_t m, const wkv7_proj_group* groups, int32_t ngroups,
                                 void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = validate(m, groups, ngroups);
  if (rc != WKV7_OK) return rc;
  if (m == 0) return WKV7_OK;
  int cus = 0;
  const int drc = device_cus(&cus);
  if (drc != WKV7_OK) return drc;
  const int waves = thin_waves(m, groups, ngroups, cus);
  if (waves == 4) return launch_thin<4>(m, groups, ngroups, NoAdapters{}, as_stream(stream));
  if (waves == 8) return launch_thin<8>(m, groups, ngroups, NoAdapters{}, as_stream(stream));
  Plan p = make_plan(m, groups, ngroups, cus);
  // without (enough) workspace every tile's workgroup covers all of k
  if (p.parts > 1 && (!workspace || workspace_bytes < p.ws_bytes || !aligned16(workspace)))
    p.parts = 1;
  float* ws = static_cast<float*>(workspace);
  return launch_plan(m, groups, ngroups, p, ws, NoAdapters{}, as_stream(stream));
}

extern "C" int wkv7_proj_grouped_noalloc(int64_t m, const wkv7_proj_group* groups,
                                         int32_t ngroups, void* stream) {
  const int rc = validate(m, groups, ngroups);
  if (rc != WKV7_OK) return rc;
  if (m == 0) return WKV7_OK;
  int cus = 0;
  const int drc = device_cus(&cus);
  if (drc != WKV7_OK) return drc;
  const int waves = thin_waves(m, groups, ngroups, cus);
  if (waves == 4) return launch_thin<4>(m, groups, ngroups, NoAdapters{}, as_stream(stream));
  if (waves == 8) return launch_thin<8>(m, groups, ngroups, NoAdapters{}, as_stream(stream));
  const Plan p = make_plan(m, groups, ngroups, cus);
  float* ws = nullptr;
  if (p.parts > 1) {
    // the split needs more partials than the static buffer holds
    if (p.ws_bytes > WKV7_PROJ_STATIC_SCRATCH_BYTES) return WKV7_ERR_WORKSPACE;
    const int src = scratch_address(&ws);
    if (src != WKV7_OK) return src;
  }
  return launch_plan(m, groups, ngroups, p, ws, NoAdapters{}, as_stream(stream));
}
