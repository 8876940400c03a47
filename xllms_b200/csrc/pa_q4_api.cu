// pa_q4_api.cu — C ABI of the 4-bit KV cache (include/operator_api.h): argument
// checks, launch planning and workspaces.
#include <algorithm>
#include <climits>
#include <cmath>
#include <cstring>
#include <numeric>

#include "operator_api.h"
#include "pa_host.h"
#include "pa_launch.h"
#include "pa_q4.h"

using namespace xpa::host;

namespace xpa {
namespace host {

// Partitions of a call, in 16-token tiles rounded to whole pages: at most
// XPA_Q4_PART_TILES, halved while the grid would hold fewer than
// XPA_Q4_ITEMS_PER_SM items per SM (8 sequences of 2048 tokens, 8 KV heads: 3
// 11.5 us, 4 14.4; 512 rows of 64 tiles with their selection 56 and 59), but not
// below 8, nor below sqrt(tiles / 2): with few rows, a shorter partition saves
// its own time and costs as much in the merge of the longer list of partials
// (2 rows of 3254 tiles, D = 256: 8 tiles 55 us, 64 tiles 26).
// Short rows stay whole, without a merge. That costs the tiles that a warp then
// takes one after the other, by head size up to 128 (the few bytes of smaller ones
// than 64 and the longer steps of larger ones are no part of it), and saves
// the merge, whose time grows with the rows: XPA_Q4_WHOLE_TILES at D = 128, and
// XPA_Q4_WHOLE_TILES_MANY at any from half as many rows as SMs on. Whole / split:
//   rows   D = 64: 24, 32, 48, 64 tiles        D = 128: 16, 24, 32, 48
//      8   4.8/6.2 5.5/5.6 6.8/6.6 8.0/6.2     5.4/6.6 6.1/7.0 7.2/6.4 9.0/7.2
//     48   5.0/6.8 5.6/6.4 7.0/7.2 8.2/7.6     5.8/6.8 6.4/7.6 7.6/7.2 9.5/8.6
//    128   5.1/7.8 5.8/7.4 7.0/10.9 8.3/8.9    5.8/7.8 6.6/9.1 7.8/8.8 9.7/12.6
// and D = 256: 16, 24, 32 tiles  8 rows 9.3/11.1 10.5/12.1 12.3/10.9, 128 rows
// 10.5/12.7 11.5/19.8 13.6/19.7 us. Finer steps (3/4, 2/3) gain where
// lengths differ and lose as much where they do not (16 sequences, 8 KV heads, a
// tenth less than now: 4-8K tokens 38 -> 32 us, 8K each 39 -> 45).
#ifndef XPA_Q4_PART_TILES
#define XPA_Q4_PART_TILES 128
#endif
#ifndef XPA_Q4_ITEMS_PER_SM
#define XPA_Q4_ITEMS_PER_SM 3
#endif
#ifndef XPA_Q4_WHOLE_TILES
#define XPA_Q4_WHOLE_TILES 24
#endif
#ifndef XPA_Q4_WHOLE_TILES_MANY
#define XPA_Q4_WHOLE_TILES_MANY 48
#endif
#ifndef XPA_Q4_MIN_TILES
#define XPA_Q4_MIN_TILES 8
#endif
Plan tile_plan(int B, int Hq, int D, int Hkv, int max_blocks, int bs, int nsm) {
  const int spp = bs / 16;
  const long long tiles = std::max(1LL, (long long)max_blocks * spp);
  const long long rows = (long long)B * Hkv, want = (long long)XPA_Q4_ITEMS_PER_SM * nsm;
  long long pt = XPA_Q4_PART_TILES;
  const bool whole = tiles * std::clamp(D, 64, 128) <= XPA_Q4_WHOLE_TILES * 128 ||
                     (2 * rows >= nsm && tiles <= XPA_Q4_WHOLE_TILES_MANY);
  if (!whole)
    while (pt > XPA_Q4_MIN_TILES && pt * pt > tiles && rows * ceil_div(tiles, pt) < want)
      pt >>= 1;
  while (ceil_div(tiles, pt) > 8192) pt <<= 1;
  Plan pl;
  pl.part_pages = (int)std::max(1LL, pt / spp);
  pl.max_parts = ceil_div(max_blocks > 0 ? max_blocks : 1, pl.part_pages);
  pl.ws_bytes = pl.max_parts > 1 ? partial_bytes((long long)B * Hq * pl.max_parts, D) : 0;
  return pl;
}

}  // namespace host
}  // namespace xpa

namespace {

bool scale_ok(float s) { return s > 0.f && std::isfinite(s); }

bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

}  // namespace

namespace xpa {
namespace host {

// What every call on 4-bit pools needs of them.
int check_q4_pools(const void* k, const void* v, int Hkv, int D, int bs, float ks, float vs,
                   int64_t kbs, int64_t khs) {
  if (!k || !v || !aligned(k, 16) || !aligned(v, 16)) return NXT_PA_EINVAL;
  if (Hkv <= 0 || D <= 0 || D > 256 || D % 16 || bs <= 0 || bs % 16) return NXT_PA_EINVAL;
  if (!scale_ok(ks) || !scale_ok(vs)) return NXT_PA_EINVAL;
  if (kbs < 0 || kbs > INT_MAX || khs < 0 || kbs % 16 || khs % 16) return NXT_PA_EINVAL;
  return NXT_PA_OK;
}

bool q4_addresses_ok(int D, int bs, int64_t kbs, int64_t num_blocks) {
  if (num_blocks <= 0 || kbs <= 0) return true;
  const long long unit = std::gcd((long long)kbs, 9LL * D);
  const long long last = 0xfffffffeLL - (bs / 16) * (9LL * D / unit);
  return last >= 0 && num_blocks - 1 <= last / (kbs / unit);
}

}  // namespace host
}  // namespace xpa

namespace {

int map_cuda(cudaError_t e) { return e == cudaSuccess ? NXT_PA_OK : NXT_PA_ECUDA; }

// 1 / s for the kernel's corrected quotient, which needs a significand that is
// not all ones and room at both ends of the range; 0: divide.
float inverse_of(float s) {
  uint32_t u;
  std::memcpy(&u, &s, sizeof u);
  const bool ones = (u & 0x7fffffu) == 0x7fffffu;
  return ones || s < 0x1p-60f || s > 0x1p60f ? 0.f : 1.f / s;
}

int rows_call(bool write, void* key, void* value, void* kc, void* vc, const int64_t* slots, int T,
              int Hkv, int D, int bs, float ks, float vs, int64_t kbs, int64_t khs,
              int64_t token_stride, int64_t num_blocks, cudaStream_t st) {
  if (T < 0) return NXT_PA_EINVAL;
  if (T == 0) return NXT_PA_OK;
  const int rc = check_q4_pools(kc, vc, Hkv, D, bs, ks, vs, kbs, khs);
  if (rc != NXT_PA_OK) return rc;
  if (!key || !value || !slots || token_stride < (int64_t)Hkv * D) return NXT_PA_EINVAL;
  if (!aligned(key, 2) || !aligned(value, 2)) return NXT_PA_EINVAL;
  if ((long long)T * Hkv > INT_MAX / 2) return NXT_PA_EINVAL;  // warps of one grid
  xpa::Q4RowsParams a{};
  a.key = key;
  a.value = value;
  a.key_cache = kc;
  a.value_cache = vc;
  a.slots = reinterpret_cast<const long long*>(slots);
  a.kv_block_stride = kbs;
  a.kv_head_stride = khs;
  a.token_stride = token_stride;
  a.num_tokens = T;
  a.Hkv = Hkv;
  a.D = D;
  a.block_size = bs;
  a.vec16 = token_stride % 8 == 0 && aligned(key, 16) && aligned(value, 16) ? 1 : 0;
  a.num_slots = num_blocks > 0 ? num_blocks * bs : LLONG_MAX;
  a.k_scale = ks;
  a.v_scale = vs;
  a.k_inverse = inverse_of(ks);
  a.v_inverse = inverse_of(vs);
  a.divide = a.k_inverse == 0.f || a.v_inverse == 0.f;
  a.clamp = !(6.f * 448.f * std::max(ks, vs) <= 65504.f);
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return NXT_PA_ECUDA;
  a.sms = sm_count_of(dev);
  return map_cuda(write ? xpa::launch_q4_write(a, st) : xpa::launch_q4_read(a, st));
}

int attention_call(void* out, const void* q, const void* k, const void* v, const int* bt,
                   const int* sl, int B, int Hq, int D, int Hkv, float scale, int max_blocks,
                   int bs, float ks, float vs, long long kbs, long long khs, long long num_blocks,
                   void* ws, size_t ws_bytes, int* dev_status, cudaStream_t st,
                   bool check_only = false) {
  int rc = check_args(out, q, k, v, bt, sl, B, Hq, D, Hkv, max_blocks, bs, 2, kbs, khs);
  if (rc != NXT_PA_OK || B == 0) return rc;
  rc = check_q4_pools(k, v, Hkv, D, bs, ks, vs, kbs, khs);
  if (rc != NXT_PA_OK) return rc;
  if (!aligned(q, 2) || !aligned(out, 2) || !q4_addresses_ok(D, bs, kbs, num_blocks))
    return NXT_PA_EINVAL;
  if (ws && !workspace_aligned(ws)) return NXT_PA_EINVAL;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return NXT_PA_ECUDA;
  const Plan pl = tile_plan(B, Hq, D, Hkv, max_blocks, bs, sm_count_of(dev));
  // one CTA per partition and 8 query heads (16 of a larger group) at least
  if ((long long)B * Hkv * pl.max_parts > INT_MAX || (long long)B * Hq > INT_MAX)
    return NXT_PA_EINVAL;
  if (check_only) return NXT_PA_OK;
  int* status = dev_status;
  if (!status) {
    rc = status_word(dev, &status);
    if (rc != NXT_PA_OK) return rc;
  }
  void* part = ws;
  std::unique_lock<std::mutex> lk;
  if (pl.ws_bytes > 0) {
    if (ws) {
      if (ws_bytes < pl.ws_bytes) return NXT_PA_EWORKSPACE;
    } else {
      rc = acquire_scratch(dev, st, pl.ws_bytes, &part, lk);
      if (rc != NXT_PA_OK) return rc;
    }
  }
  xpa::Params p{};
  p.out = out;
  p.q = q;
  p.k = k;
  p.v = v;
  p.block_tables = bt;
  p.seq_lens = sl;
  p.part_o = static_cast<float*>(part);
  p.part_ml = part ? reinterpret_cast<float*>(
                         static_cast<char*>(part) +
                         part_ml_offset_bytes((long long)B * Hq * pl.max_parts, D))
                   : nullptr;
  p.status = status;
  p.kv_block_stride = kbs;
  p.kv_head_stride = khs;
  p.num_blocks = num_blocks;
  p.B = B;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.D = D;
  p.GS = Hq / Hkv;
  p.max_blocks = max_blocks;
  p.block_size = bs;
  p.part_pages = pl.part_pages;
  p.max_parts = pl.max_parts;
  p.slots = pl.max_parts;
  p.scale_log2 = scale * ks * 1.4426950408889634f;
  p.ml_unit = score_unit(p.scale_log2);
  p.v_scale = vs;
  p.vec8 = aligned(out, 16) ? 1 : 0;
  cudaError_t e = xpa::launch_q4_attention(p, st);
  if (e == cudaSuccess && pl.max_parts > 1) e = xpa::launch_reduce(p, 2, st);
  return map_cuda(e);
}

}  // namespace

extern "C" {

int nxt_reshape_and_cache_q4(const void* key, const void* value, void* key_cache,
                             void* value_cache, const int64_t* slot_mapping, int num_tokens,
                             int num_kv_heads, int head_size, int block_size, float k_scale,
                             float v_scale, int64_t kv_block_stride, int64_t kv_head_stride,
                             int64_t token_stride, int64_t num_blocks, nxt_stream_t stream) {
  return rows_call(true, const_cast<void*>(key), const_cast<void*>(value), key_cache, value_cache,
                   slot_mapping, num_tokens, num_kv_heads, head_size, block_size, k_scale, v_scale,
                   kv_block_stride, kv_head_stride, token_stride, num_blocks,
                   static_cast<cudaStream_t>(stream));
}

int nxt_read_cache_q4(void* key, void* value, const void* key_cache, const void* value_cache,
                      const int64_t* slot_mapping, int num_tokens, int num_kv_heads, int head_size,
                      int block_size, float k_scale, float v_scale, int64_t kv_block_stride,
                      int64_t kv_head_stride, int64_t token_stride, int64_t num_blocks,
                      nxt_stream_t stream) {
  return rows_call(false, key, value, const_cast<void*>(key_cache),
                   const_cast<void*>(value_cache), slot_mapping, num_tokens, num_kv_heads,
                   head_size, block_size, k_scale, v_scale, kv_block_stride, kv_head_stride,
                   token_stride, num_blocks, static_cast<cudaStream_t>(stream));
}

int nxt_paged_attention_q4_ex(void* out, const void* query, const void* key_cache,
                              const void* value_cache, const int* block_tables,
                              const int* seq_lens, int num_seqs, int num_heads, int head_size,
                              int num_kv_heads, float scale, int max_num_blocks_per_seq,
                              int block_size, float k_scale, float v_scale,
                              int64_t kv_block_stride, int64_t kv_head_stride, int64_t num_blocks,
                              void* workspace, size_t workspace_bytes, int* device_status,
                              nxt_stream_t stream) {
  return attention_call(out, query, key_cache, value_cache, block_tables, seq_lens, num_seqs,
                        num_heads, head_size, num_kv_heads, scale, max_num_blocks_per_seq,
                        block_size, k_scale, v_scale, kv_block_stride, kv_head_stride, num_blocks,
                        workspace, workspace_bytes, device_status,
                        static_cast<cudaStream_t>(stream));
}

size_t nxt_paged_attention_q4_workspace_size(int num_seqs, int num_heads, int head_size,
                                             int num_kv_heads, int max_num_blocks_per_seq,
                                             int block_size) {
  if (num_seqs <= 0 || num_heads <= 0 || num_kv_heads <= 0 || head_size <= 0 || block_size < 16)
    return 0;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) dev = -1;
  return tile_plan(num_seqs, num_heads, head_size, num_kv_heads, max_num_blocks_per_seq, block_size,
                 sm_count_of(dev))
      .ws_bytes;
}

int nxt_paged_attention_q4_append_ex(void* out, const void* query, void* key_cache,
                                     void* value_cache, const int* block_tables,
                                     const int* seq_lens, const void* new_key,
                                     const void* new_value, const int64_t* slot_mapping,
                                     int num_seqs, int num_heads, int head_size, int num_kv_heads,
                                     float scale, int max_num_blocks_per_seq, int block_size,
                                     float k_scale, float v_scale, int64_t kv_block_stride,
                                     int64_t kv_head_stride, int64_t num_blocks,
                                     int* device_status, nxt_stream_t stream) {
  // everything is checked before anything is launched
  int rc = attention_call(out, query, key_cache, value_cache, block_tables, seq_lens, num_seqs,
                          num_heads, head_size, num_kv_heads, scale, max_num_blocks_per_seq,
                          block_size, k_scale, v_scale, kv_block_stride, kv_head_stride,
                          num_blocks, nullptr, 0, device_status,
                          static_cast<cudaStream_t>(stream), true);
  if (rc != NXT_PA_OK || num_seqs == 0) return rc;
  rc = nxt_reshape_and_cache_q4(new_key, new_value, key_cache, value_cache, slot_mapping, num_seqs,
                                num_kv_heads, head_size, block_size, k_scale, v_scale,
                                kv_block_stride, kv_head_stride,
                                (int64_t)num_kv_heads * head_size, num_blocks, stream);
  if (rc != NXT_PA_OK) return rc;
  return attention_call(out, query, key_cache, value_cache, block_tables, seq_lens, num_seqs,
                        num_heads, head_size, num_kv_heads, scale, max_num_blocks_per_seq,
                        block_size, k_scale, v_scale, kv_block_stride, kv_head_stride, num_blocks,
                        nullptr, 0, device_status, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
