// pa_host.h — host-side planning helpers shared by the C-ABI entry points
// (pa_api.cu) and the allocation-free entry point (pa_noalloc.cu).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <atomic>
#include <cmath>
#include <mutex>

namespace xpa {
namespace host {

int ceil_div(long long a, long long b);

// SM count of device `dev` (cached; 148 when the query fails).
int sm_count_of(int dev);

// Bound on every pipeline wait of kernels launched by this host thread
// (nxt_paged_attention_set_wait_budget_ns; 1 s by default).
unsigned long long wait_budget_ns();

// Split-context partials of one call, in one workspace: part_o
// [rows][slots][D] fp32 from byte 0, then part_ml [rows][slots][2] fp32 from
// the next kPartAlign-byte boundary (rows = B * Hq). The merge reads (m, l)
// as 8-byte pairs, which an odd rows * slots * D would otherwise misalign,
// and part_o rows as 16-byte vectors, so the workspace itself must start on a
// 16-byte boundary.
constexpr size_t kPartAlign = 256;
inline size_t part_ml_offset_bytes(long long row_slots, int D) {
  const size_t o = (size_t)row_slots * (size_t)D * sizeof(float);
  return (o + kPartAlign - 1) / kPartAlign * kPartAlign;
}
inline size_t partial_bytes(long long row_slots, int D) {
  return part_ml_offset_bytes(row_slots, D) + (size_t)row_slots * 2 * sizeof(float);
}
inline bool workspace_aligned(const void* ws) {
  return (reinterpret_cast<size_t>(ws) & 15u) == 0;
}

// Context partitioning of one call and the split-context partial bytes it needs.
struct Plan {
  int part_pages = 32;
  int max_parts = 1;
  size_t ws_bytes = 0;
};
// kv_es: bytes per K / V element (1 for fp8 pools, whose partitions keep
// shrinking until the grid holds 24 CTAs per SM instead of 12).
// min_items: items per SM instead of the default floor (0); min_pages: the
// shortest partition, in pages.
Plan make_plan(int B, int Hq, int D, int Hkv, int max_blocks, int nsm, int kv_es = 2,
               int min_items = 0, int min_pages = 4);

// Params::ml_unit of the same kernels: they handle scores as q . k times this,
// with the scale's sign in Q (a scale of 0 is a Q of 0).
inline float score_unit(float scale_log2) {
  return scale_log2 == 0.f ? 1.f : std::fabs(scale_log2);
}

// Plan of the kernels that take an item in 16-token tiles (4-bit, fp16 pages).
Plan tile_plan(int B, int Hq, int D, int Hkv, int max_blocks, int bs, int nsm);

// nxt_paged_attention_ex with these floors; `ws` holds at least
// make_plan(...).ws_bytes of the same floors.
int attention_planned(void* out, const void* q, const void* k, const void* v, const int* bt,
                      const int* sl, int B, int Hq, int D, int Hkv, float scale, int max_blocks,
                      int bs, int ds, long long kbs, long long khs, long long num_blocks, void* ws,
                      size_t ws_bytes, int* dev_status, cudaStream_t st, int min_items,
                      int min_pages);

// Tensor map of one pool for the TMA path; false when it cannot be encoded.
// es: bytes per K / V element (2 = fp16, 1 = fp8).
bool encode_pool(CUtensorMap* m, const void* base, int D, int Hkv, long long num_blocks,
                 long long kbs, long long khs, int es = 2);

// Pool alignment and stride order the TMA path needs.
bool fast_layout_ok(const void* k, const void* v, int D, int Hkv, long long kbs, long long khs,
                    int es = 2);

// What every call on 4-bit pools needs of them: NXT_PA_OK or NXT_PA_EINVAL.
int check_q4_pools(const void* k, const void* v, int Hkv, int D, int bs, float k_scale,
                   float v_scale, int64_t kbs, int64_t khs);
// The 4-bit kernels address tiles by 32 bits of the largest unit that divides a
// page and a tile. False: pools that are known (num_blocks > 0) to be larger.
bool q4_addresses_ok(int D, int bs, int64_t kbs, int64_t num_blocks);

// NXT_PA_OK or NXT_PA_EINVAL for the argument set of one call.
int check_args(const void* out, const void* q, const void* k, const void* v, const int* bt,
               const int* sl, int B, int Hq, int D, int Hkv, int max_blocks, int bs, int ds,
               long long kbs, long long khs);

// Raises a kernel's dynamic shared memory limit once per device (`done` is the
// kernel's own set of devices), with all of the L1 / shared storage as shared
// memory when `carve`.
template <typename Kernel>
cudaError_t smem_limit(Kernel kern, size_t bytes, bool carve, std::atomic<unsigned long long>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const unsigned long long bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == cudaSuccess && carve)
    e = cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout,
                             (int)cudaSharedmemCarveoutMaxShared);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

// The library status word of device `dev` (the current device).
int status_word(int dev, int** out);

// Library-owned scratch of the 4-bit and sparse entry points: one buffer per
// (device, stream) for calls that run at once, and one per stream capture for
// captured calls, which the graph owns, so that graphs may be replayed at the
// same time as each other and as eager calls. `lk` holds the stream's lock on
// return: keep it until the call's kernels are enqueued, so that no other
// thread on the same stream can hand out the buffer in between. A buffer that
// has to grow is replaced, and the old one kept until release_scratch(). No
// thread's capture is disturbed.
// EINVAL / ECUDA / ENOMEM / OK.
int acquire_scratch(int dev, cudaStream_t st, size_t bytes, void** out,
                    std::unique_lock<std::mutex>& lk);
int release_scratch();

}  // namespace host
}  // namespace xpa
