// pa_sparse_api.cu — C ABI of page bounds and sparse decode attention
// (include/operator_api.h). Attention over the kept pages is the framework's
// own decode attention on per-head pages: page p of KV head h is page
// p * (kv_block_stride / kv_head_stride) + h of a pool with one KV head.
#include <algorithm>
#include <climits>
#include <cmath>

#include "operator_api.h"
#include "pa_host.h"
#include "pa_launch.h"
#include "pa_sparse.h"

using namespace xpa::host;

namespace {

int map_cuda(cudaError_t e) { return e == cudaSuccess ? NXT_PA_OK : NXT_PA_ECUDA; }

bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

int bounds_call(void* bounds, const void* key_cache, const int* bt, const int* sl, int B, int Hkv,
                int D, int max_blocks, int bs, int kind, float k_scale, int64_t kbs, int64_t khs,
                int64_t num_blocks, int num_new, int* dev_status, cudaStream_t st) {
  const bool q4 = kind == xpa::kBoundsQ4;
  if (B < 0 || num_new < 0) return NXT_PA_EINVAL;
  if (B == 0) return NXT_PA_OK;
  if (!bounds || !key_cache || !bt || !sl) return NXT_PA_EINVAL;
  if (Hkv <= 0 || D <= 0 || D > 256 || bs <= 0 || max_blocks < 0 || kbs < 0 || khs < 0)
    return NXT_PA_EINVAL;
  const unsigned es = kind == xpa::kBoundsF32 ? 4 : 2;
  if (!aligned(bounds, es)) return NXT_PA_EINVAL;
  if (q4) {
    if (D % 16 || bs % 16 || kbs % 16 || khs % 16 || !aligned(key_cache, 16) ||
        !(k_scale > 0.f) || !std::isfinite(k_scale))
      return NXT_PA_EINVAL;
  } else if (!aligned(key_cache, es)) {
    return NXT_PA_EINVAL;
  }
  if (max_blocks == 0) return NXT_PA_OK;
  xpa::BoundsParams p{};
  p.bounds = bounds;
  p.key_cache = key_cache;
  p.block_tables = bt;
  p.seq_lens = sl;
  p.kv_block_stride = kbs;
  p.kv_head_stride = khs;
  p.num_blocks = num_blocks;
  p.B = B;
  p.Hkv = Hkv;
  p.D = D;
  p.max_blocks = max_blocks;
  p.block_size = bs;
  p.num_new = num_new;
  // the last num_new tokens lie in at most this many pages
  p.pages_per_seq = max_blocks;
  if (num_new > 0)
    p.pages_per_seq = (int)std::min<long long>(max_blocks, (num_new - 1LL) / bs + 2);
  p.kind = kind;
  p.k_scale = k_scale;
  if (!q4) {
    p.vec = aligned(key_cache, 16) && aligned(bounds, 16) && (D * es) % 16 == 0 &&
            (kbs * es) % 16 == 0 && (khs * es) % 16 == 0;
  }
  if ((long long)B * p.pages_per_seq > INT_MAX)
    return NXT_PA_EINVAL;
  p.status = dev_status;
  if (!p.status) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return NXT_PA_ECUDA;
    const int rc = status_word(dev, &p.status);
    if (rc != NXT_PA_OK) return rc;
  }
  return map_cuda(xpa::launch_bounds(p, st));
}

// One sparse call. Exactly one of the attention forms is asked for, or none
// (selection alone, into the caller's arrays).
struct SparseCall {
  // selection
  const void *q, *bounds;
  const int *bt, *sl;
  int* sel_pages;
  int B, Hq, D, Hkv;
  float scale;
  int max_blocks, bs, ds;
  int64_t kbs, khs, num_blocks;
  int keep, sink, recent;
  // attention
  void* out = nullptr;
  const void *k = nullptr, *v = nullptr;
  bool q4 = false;
  float k_scale = 1.f, v_scale = 1.f;
};

// Items per SM below which the attention over the kept pages splits its rows
// further. A row holds few pages here, so the partials of a finer split cost
// more than an idle SM (64 rows of 256 pages, whole sparse call: 8 items took 5
// us more than 3).
#ifndef XPA_SPARSE_ITEMS_PER_SM
#define XPA_SPARSE_ITEMS_PER_SM 3
#endif

bool tma_shape(int D, int bs, int ds) {
  return ds == 2 && bs == 16 && (D == 64 || D == 128 || D == 256);
}

// Heads of a group that the TMA kernel reads a page for.
int tma_heads(int D) { return D == 256 ? 8 : 16; }

// What attends to a row's kept pages.
enum Path { kPathDecode, kPathPages, kPathQ4 };

// Parts that a KV head's group of query heads is taken in. The tensor-core
// decode kernel of fp16 pools reads a page for up to 16 heads (8 at head size
// 256), and re-reading it from L2 for the next part costs less than the
// CUDA-core kernel (whole sparse call, 8 sequences: 192 heads over 8 KV heads,
// D = 128, 64 pages: 302 -> 53 us; 48 over 3, D = 256, 18 pages: 116 -> 39).
// The CUDA-core kernel goes over a page once per `most` heads, so CTAs of that
// many side by side read no more.
int head_parts(int GS, int D, int bs, int ds) {
  const int tma = tma_shape(D, bs, ds) ? tma_heads(D) : 0;
  const int most = D <= 64 ? 16 : D <= 128 ? 8 : 4;
  int parts = 1;
  for (int s = 1; s <= 8; ++s) {
    if (GS % s) continue;
    if (tma && GS / s <= tma) return s;
    if (GS / parts > most) parts = s;
  }
  return parts;
}

// fp16 shapes of the pages kernel: those that the decode kernel, with a page in
// `sub` pieces, takes to its CUDA-core form. At the TMA kernel's shapes it is the
// slower one from a few dozen pages a row on (64 rows of 256 pages, whole sparse
// call: 98 against 85 us).
bool pages_shape(int GS, int D, int bs, int ds, int sub) {
  if (ds != 2 || D % 16 || bs % 16) return false;
  return !(tma_shape(D, bs / sub, ds) &&
           GS / head_parts(GS, D, bs / sub, ds) <= tma_heads(D));
}

// Shortest partition of the attention, in pages: 64 tokens.
int min_pages(int bs) { return bs >= 64 ? 1 : 64 / bs; }

// Workspace: scores and near pages of the selection, the kept pages' tables,
// the attention's partials, each from a 256-byte boundary.
struct Layout {
  size_t keys, magnitude, near_page, near_key, order, tables, lens, part, total;
  size_t part_bytes;
  int parts;  // of a group's heads, see head_parts
  int width;  // entries of a row's tables: no more than a sequence has pages
};

// sub: the attention takes a page as this many of bs / sub tokens.
Layout layout_of(long long rows, int GS, int D, int max_blocks, int bs, int ds, int keep,
                 Path path, bool attention, int sms, int sub) {
  Layout l{};
  l.parts = 1;
  l.width = attention ? std::max(1, std::min(keep, max_blocks)) : keep;
  size_t at = 0;
  auto take = [&at](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  const size_t scored = max_blocks > keep ? (size_t)rows * max_blocks : 0;
  l.keys = take(scored * sizeof(unsigned));
  l.magnitude = take(scored ? (size_t)rows * ceil_div(max_blocks, xpa::kScoreChunkLeast) * sizeof(float) : 0);
  l.near_page = take(scored * sizeof(unsigned));
  l.near_key = take(scored * sizeof(unsigned long long));
  l.order = take(sub > 1 ? (size_t)rows * l.width * sizeof(int) : 0);
  if (attention) {
    if (path == kPathDecode) l.parts = head_parts(GS, D, bs / sub, ds);
    const long long n = rows * l.parts;
    l.tables = take((size_t)n * l.width * sub * sizeof(int));
    l.lens = take((size_t)n * sizeof(int));
    l.part_bytes = path != kPathDecode
                       ? tile_plan((int)n, GS, D, 1, l.width, bs, sms).ws_bytes
                       : make_plan((int)n, GS / l.parts, D, 1, l.width * sub, sms, ds,
                                   XPA_SPARSE_ITEMS_PER_SM, min_pages(bs / sub))
                             .ws_bytes;
    l.part = take(l.part_bytes);
  }
  l.total = at;
  return l;
}

int sparse_call(const SparseCall& c, int* sel_tables, int* sel_lens, void* ws, size_t ws_bytes,
                int* dev_status, cudaStream_t st) {
  const bool attention = c.out || c.k;
  int rc;
  if (attention) {
    rc = check_args(c.out, c.q, c.k, c.v, c.bt, c.sl, c.B, c.Hq, c.D, c.Hkv, c.max_blocks, c.bs,
                    c.ds, c.kbs, c.khs);
  } else {
    rc = check_args(c.q, c.q, c.q, c.q, c.bt, c.sl, c.B, c.Hq, c.D, c.Hkv, c.max_blocks, c.bs,
                    c.ds, c.kbs, c.khs);
    if (rc == NXT_PA_OK && c.B > 0 && (!sel_tables || !sel_lens)) rc = NXT_PA_EINVAL;
  }
  if (rc != NXT_PA_OK || c.B == 0) return rc;
  if (!c.bounds || !aligned(c.bounds, c.ds) || !aligned(c.q, c.ds)) return NXT_PA_EINVAL;
  if (c.sink < 0 || c.recent < 1 || c.keep < 1 || (long long)c.sink + c.recent > c.keep ||
      (long long)c.keep * c.bs > INT_MAX)
    return NXT_PA_EINVAL;
  if (std::isnan(c.scale)) return NXT_PA_EINVAL;
  if (c.Hkv > 1 && (c.khs <= 0 || c.kbs % c.khs || c.kbs / c.khs < c.Hkv)) return NXT_PA_EINVAL;
  if (ws && !workspace_aligned(ws)) return NXT_PA_EINVAL;
  const long long rows = (long long)c.B * c.Hkv;
  const int GS = c.Hq / c.Hkv;
  if (rows * ceil_div(c.max_blocks, xpa::kScoreTile) > INT_MAX || rows * GS > INT_MAX ||
      rows * c.keep * std::max(1, c.bs / 16) > INT_MAX / 8)
    return NXT_PA_EINVAL;
  const long long head_pages = c.Hkv > 1 ? c.kbs / c.khs : 1;
  const int64_t page_stride = c.Hkv > 1 ? c.khs : c.kbs;
  // pages of the pool with one KV head, -1: unknown; ids are ints
  int64_t nb = c.num_blocks > 0 ? c.num_blocks : -1;
  if (nb > 0) nb = nb > INT_MAX / head_pages ? INT_MAX : nb * head_pages;
  // all that the attention would refuse, before the selection is launched
  if (c.q4) {
    rc = check_q4_pools(c.k, c.v, 1, c.D, c.bs, c.k_scale, c.v_scale, page_stride, c.khs);
    if (rc != NXT_PA_OK) return rc;
    if (!aligned(c.q, 2) || !aligned(c.out, 2) || !q4_addresses_ok(c.D, c.bs, page_stride, nb))
      return NXT_PA_EINVAL;
  }
  // Longer pages go to the tensor-core kernel as pages of 16 tokens, where ids
  // of those fit
  int sub = 1;
  long long sub_ids = 1;
  const int64_t piece = 16LL * c.D;
  if (attention && !c.q4 && c.bs > 16 && c.bs % 16 == 0 && tma_shape(c.D, 16, c.ds) &&
      page_stride % piece == 0 && page_stride / piece >= c.bs / 16 && c.num_blocks > 0 &&
      c.num_blocks <= INT_MAX / head_pages / (page_stride / piece)) {
    sub = c.bs / 16;
    sub_ids = page_stride / piece;
  }
  // What the TMA kernel's boxes and heads do not fit goes to the kernel of plain
  // copies where rows start on 16-byte boundaries, else to the CUDA-core kernel.
  Path path = c.q4 ? kPathQ4 : kPathDecode;
  if (attention && !c.q4 && pages_shape(GS, c.D, c.bs, c.ds, sub) && aligned(c.k, 16) &&
      aligned(c.v, 16) && page_stride % 8 == 0 && aligned(c.q, 4)) {
    path = kPathPages;
    sub = 1;
    sub_ids = 1;
  }

  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return NXT_PA_ECUDA;
  int* status = dev_status;
  if (!status) {
    rc = status_word(dev, &status);
    if (rc != NXT_PA_OK) return rc;
  }
  const Layout l =
      layout_of(rows, GS, c.D, c.max_blocks, c.bs, c.ds, c.keep, path, attention,
                sm_count_of(dev), sub);
  std::unique_lock<std::mutex> lk;
  if (ws) {
    if (ws_bytes < l.total) return NXT_PA_EWORKSPACE;
  } else if (l.total > 0) {
    rc = acquire_scratch(dev, st, l.total, &ws, lk);
    if (rc != NXT_PA_OK) return rc;
  }
  char* base = static_cast<char*>(ws);
  xpa::SelectParams p{};
  p.q = c.q;
  p.bounds = c.bounds;
  p.block_tables = c.bt;
  p.seq_lens = c.sl;
  p.status = status;
  p.sel_tables = attention ? reinterpret_cast<int*>(base + l.tables) : sel_tables;
  p.sel_lens = attention ? reinterpret_cast<int*>(base + l.lens) : sel_lens;
  p.sel_pages = c.sel_pages;
  p.order = sub > 1 ? reinterpret_cast<int*>(base + l.order) : nullptr;
  p.width = l.width;
  p.sub = sub;
  p.sub_ids = (int)sub_ids;
  p.keys = reinterpret_cast<unsigned*>(base + l.keys);
  p.magnitude = reinterpret_cast<float*>(base + l.magnitude);
  p.near_page = reinterpret_cast<unsigned*>(base + l.near_page);
  p.near_key = reinterpret_cast<unsigned long long*>(base + l.near_key);
  p.num_blocks = c.num_blocks;
  p.head_pages = head_pages;
  p.B = c.B;
  p.Hq = c.Hq;
  p.Hkv = c.Hkv;
  p.D = c.D;
  p.GS = GS;
  p.max_blocks = c.max_blocks;
  p.block_size = c.bs;
  p.keep = c.keep;
  p.sink = c.sink;
  p.recent = c.recent;
  p.copies = l.parts;
  p.sign = c.scale > 0.f ? 1.f : c.scale < 0.f ? -1.f : 0.f;
  p.vec = c.ds == 2 && c.D % 8 == 0 && aligned(c.q, 16) && aligned(c.bounds, 16);
  p.chunk_pages = p.vec ? xpa::score_chunk(c.B, c.Hkv, c.max_blocks, sm_count_of(dev))
                        : xpa::score_chunk_scalar(rows, c.max_blocks, sm_count_of(dev));
  p.tile_pages = p.vec ? xpa::kScoreTile : p.chunk_pages;
  p.chunks = ceil_div(c.max_blocks, p.chunk_pages);
  p.tiles = ceil_div(c.max_blocks, p.tile_pages);
  const cudaError_t e = xpa::launch_select(p, c.ds, st);
  if (e != cudaSuccess) return map_cuda(e);
  if (!attention) return NXT_PA_OK;

  void* part = l.part_bytes ? base + l.part : nullptr;
  if (c.q4)
    return nxt_paged_attention_q4_ex(c.out, c.q, c.k, c.v, p.sel_tables, p.sel_lens, (int)rows,
                                     GS, c.D, 1, c.scale, l.width, c.bs, c.k_scale,
                                     c.v_scale, page_stride, c.khs, nb, part, l.part_bytes, status,
                                     st);
  if (path == kPathPages) {
    const Plan pl = tile_plan((int)rows, GS, c.D, 1, l.width, c.bs, sm_count_of(dev));
    xpa::Params a{};
    a.out = c.out;
    a.q = c.q;
    a.k = c.k;
    a.v = c.v;
    a.block_tables = p.sel_tables;
    a.seq_lens = p.sel_lens;
    a.part_o = static_cast<float*>(part);
    a.part_ml = part ? reinterpret_cast<float*>(
                           static_cast<char*>(part) +
                           part_ml_offset_bytes(rows * GS * pl.max_parts, c.D))
                     : nullptr;
    a.status = status;
    a.kv_block_stride = page_stride;
    a.num_blocks = nb;
    a.B = (int)rows;
    a.Hq = a.GS = GS;
    a.Hkv = 1;
    a.D = c.D;
    a.max_blocks = l.width;
    a.block_size = c.bs;
    a.part_pages = pl.part_pages;
    a.max_parts = a.slots = pl.max_parts;
    a.scale_log2 = c.scale * 1.4426950408889634f;
    a.ml_unit = score_unit(a.scale_log2);
    a.v_scale = 1.f;
    a.vec8 = aligned(c.out, 16) ? 1 : 0;
    cudaError_t err = xpa::launch_pages(a, st);
    if (err == cudaSuccess && pl.max_parts > 1) err = xpa::launch_reduce(a, 2, st);
    return map_cuda(err);
  }
  if (sub > 1) nb = c.num_blocks * head_pages * sub_ids;
  return attention_planned(c.out, c.q, c.k, c.v, p.sel_tables, p.sel_lens, (int)rows * l.parts,
                           GS / l.parts, c.D, 1, c.scale, l.width * sub, c.bs / sub, c.ds,
                           sub > 1 ? piece : page_stride, sub > 1 ? piece : c.khs, nb, part,
                           l.part_bytes, status, st, XPA_SPARSE_ITEMS_PER_SM,
                           min_pages(c.bs / sub));
}

}  // namespace

extern "C" {

int nxt_page_bounds(void* bounds, const void* key_cache, const int* block_tables,
                    const int* seq_lens, int num_seqs, int num_kv_heads, int head_size,
                    int max_num_blocks_per_seq, int block_size, int dtype_size,
                    int64_t kv_block_stride, int64_t kv_head_stride, int64_t num_blocks,
                    int num_new_tokens, int* device_status, nxt_stream_t stream) {
  if (dtype_size != 2 && dtype_size != 4) return NXT_PA_EINVAL;
  return bounds_call(bounds, key_cache, block_tables, seq_lens, num_seqs, num_kv_heads, head_size,
                     max_num_blocks_per_seq, block_size,
                     dtype_size == 4 ? xpa::kBoundsF32 : xpa::kBoundsF16, 1.f, kv_block_stride,
                     kv_head_stride, num_blocks, num_new_tokens, device_status,
                     static_cast<cudaStream_t>(stream));
}

int nxt_page_bounds_q4(void* bounds, const void* key_cache, const int* block_tables,
                       const int* seq_lens, int num_seqs, int num_kv_heads, int head_size,
                       int max_num_blocks_per_seq, int block_size, float k_scale,
                       int64_t kv_block_stride, int64_t kv_head_stride, int64_t num_blocks,
                       int num_new_tokens, int* device_status, nxt_stream_t stream) {
  return bounds_call(bounds, key_cache, block_tables, seq_lens, num_seqs, num_kv_heads, head_size,
                     max_num_blocks_per_seq, block_size, xpa::kBoundsQ4, k_scale, kv_block_stride,
                     kv_head_stride, num_blocks, num_new_tokens, device_status,
                     static_cast<cudaStream_t>(stream));
}

int nxt_select_pages(int* sel_tables, int* sel_lens, int* sel_pages, const void* query,
                     const void* bounds, const int* block_tables, const int* seq_lens,
                     int num_seqs, int num_heads, int head_size, int num_kv_heads, float scale,
                     int max_num_blocks_per_seq, int block_size, int dtype_size,
                     int64_t kv_block_stride, int64_t kv_head_stride, int64_t num_blocks,
                     int max_pages, int sink_pages, int recent_pages, void* workspace,
                     size_t workspace_bytes, int* device_status, nxt_stream_t stream) {
  SparseCall c{query, bounds, block_tables, seq_lens, sel_pages, num_seqs, num_heads, head_size,
               num_kv_heads, scale, max_num_blocks_per_seq, block_size, dtype_size,
               kv_block_stride, kv_head_stride, num_blocks, max_pages, sink_pages, recent_pages};
  return sparse_call(c, sel_tables, sel_lens, workspace, workspace_bytes, device_status,
                     static_cast<cudaStream_t>(stream));
}

int nxt_paged_attention_sparse_ex(void* out, const void* query, const void* key_cache,
                                  const void* value_cache, const void* bounds,
                                  const int* block_tables, const int* seq_lens, int* sel_pages,
                                  int num_seqs, int num_heads, int head_size, int num_kv_heads,
                                  float scale, int max_num_blocks_per_seq, int block_size,
                                  int dtype_size, int64_t kv_block_stride, int64_t kv_head_stride,
                                  int64_t num_blocks, int max_pages, int sink_pages,
                                  int recent_pages, void* workspace, size_t workspace_bytes,
                                  int* device_status, nxt_stream_t stream) {
  SparseCall c{query, bounds, block_tables, seq_lens, sel_pages, num_seqs, num_heads, head_size,
               num_kv_heads, scale, max_num_blocks_per_seq, block_size, dtype_size,
               kv_block_stride, kv_head_stride, num_blocks, max_pages, sink_pages, recent_pages,
               out, key_cache, value_cache};
  if (num_seqs > 0 && (!out || !key_cache || !value_cache)) return NXT_PA_EINVAL;
  return sparse_call(c, nullptr, nullptr, workspace, workspace_bytes, device_status,
                     static_cast<cudaStream_t>(stream));
}

int nxt_paged_attention_q4_sparse_ex(void* out, const void* query, const void* key_cache,
                                     const void* value_cache, const void* bounds,
                                     const int* block_tables, const int* seq_lens, int* sel_pages,
                                     int num_seqs, int num_heads, int head_size, int num_kv_heads,
                                     float scale, int max_num_blocks_per_seq, int block_size,
                                     float k_scale, float v_scale, int64_t kv_block_stride,
                                     int64_t kv_head_stride, int64_t num_blocks, int max_pages,
                                     int sink_pages, int recent_pages, void* workspace,
                                     size_t workspace_bytes, int* device_status,
                                     nxt_stream_t stream) {
  SparseCall c{query, bounds, block_tables, seq_lens, sel_pages, num_seqs, num_heads, head_size,
               num_kv_heads, scale, max_num_blocks_per_seq, block_size, 2, kv_block_stride,
               kv_head_stride, num_blocks, max_pages, sink_pages, recent_pages, out, key_cache,
               value_cache, true, k_scale, v_scale};
  if (num_seqs > 0 && (!out || !key_cache || !value_cache)) return NXT_PA_EINVAL;
  return sparse_call(c, nullptr, nullptr, workspace, workspace_bytes, device_status,
                     static_cast<cudaStream_t>(stream));
}

size_t nxt_paged_attention_sparse_workspace_size(int num_seqs, int num_heads, int head_size,
                                                 int num_kv_heads, int max_num_blocks_per_seq,
                                                 int block_size, int dtype_size, int max_pages) {
  if (num_seqs <= 0 || num_heads <= 0 || num_kv_heads <= 0 || head_size <= 0 || block_size <= 0 ||
      max_pages <= 0 || max_num_blocks_per_seq < 0)
    return 0;
  const long long rows = (long long)num_seqs * num_kv_heads;
  if (rows > INT_MAX / 8 || max_pages > INT_MAX / block_size) return 0;
  const int GS = num_heads / num_kv_heads;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) dev = -1;
  const int sms = sm_count_of(dev);
  // the largest of what a call may take: 4-bit pools, pages whole or in pieces
  size_t most = 0;
  auto add = [&](Path path, int sub) {
    most = std::max(most, layout_of(rows, GS, head_size, max_num_blocks_per_seq, block_size,
                                    dtype_size, max_pages, path, true, sms, sub)
                              .total);
  };
  add(kPathDecode, 1);
  if (block_size % 16 == 0) {
    add(kPathQ4, 1);  // and kPathPages
    add(kPathDecode, block_size / 16);
  }
  return most;
}

}  // extern "C"
