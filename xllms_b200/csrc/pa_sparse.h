// pa_sparse.h — host-side launchers of the page bounds and page selection
// kernels (pa_sparse.cu).
#pragma once

#include <cuda_runtime.h>

#include "pa_device.cuh"

namespace xpa {

// Element type of the cache the bounds are taken from.
constexpr int kBoundsF16 = 0;
constexpr int kBoundsF32 = 1;
constexpr int kBoundsQ4 = 2;  // 4-bit keys; the bounds are fp16

struct BoundsParams {
  void* bounds;  // [num_blocks][Hkv][2][D]: lowest, then highest key per channel
  const void* key_cache;
  const int* block_tables;
  const int* seq_lens;
  int* status;
  long long kv_block_stride, kv_head_stride;  // elements (4-bit: bytes)
  long long num_blocks;
  int B, Hkv, D, max_blocks, block_size;
  int num_new;        // > 0: only pages that hold one of the last num_new tokens
  int pages_per_seq;  // pages of a sequence that may be due
  int kind;
  int vec;            // every key row and bounds row starts on a 16-byte boundary
  float k_scale;      // 4-bit
};

cudaError_t launch_bounds(const BoundsParams& p, cudaStream_t st);

struct SelectParams {
  const void* q;       // [B][Hq][D]
  const void* bounds;  // [num_blocks][Hkv][2][D]
  const int* block_tables;
  const int* seq_lens;
  int* status;
  int* sel_tables;  // [B * Hkv][copies][width][sub] page * head_pages + kv head, see sub
  int* sel_lens;    // [B * Hkv][copies] tokens kept
  int* sel_pages;   // [B * Hkv][keep] page index within the sequence, -1 past the last; or null
  // workspace
  int* order;             // [B * Hkv][width] kept pages' indices on the way; null: in sel_tables
  unsigned* keys;         // [B * Hkv][max_blocks] ordered scores, 0: page not eligible
  float* magnitude;       // [B * Hkv][tiles] per tile_pages pages, the largest sum of the
                          // magnitudes of a score's terms
  unsigned* near_page;    // [B * Hkv][max_blocks] pages too near the border for fp32
  unsigned long long* near_key;  // [B * Hkv][max_blocks] their scores in 64 bits
  long long num_blocks;
  long long head_pages;  // kv_block_stride / kv_head_stride
  int B, Hq, Hkv, D, GS, max_blocks, block_size;
  int keep, sink, recent;
  int width;   // kept pages that a row's tables have room for
  int copies;  // of every row's tables, for attention that takes its heads in parts
  int sub;     // entries per kept page: page id * sub_ids + 0 .. sub - 1, for attention
  int sub_ids; // that takes a page in pieces of 16 tokens (sub > 1 needs order)
  int chunks, chunk_pages;  // score CTAs per row (or kScoreWarps rows), pages of each
  int tiles, tile_pages;    // entries of a row's magnitude, pages of each
  float sign;  // of the score scale: -1, 0 or 1
  int vec;     // fp16, D % 8 == 0, q and bounds on 16-byte boundaries
};

// Pages of one magnitude entry and of one score CTA. The tensor-core kernel
// takes tiles of 16, 128 pages a CTA (8 sequences of 32-128K tokens: 64 pages
// 80 us with the selection, 128 74, 32 91), fewer while that leaves the GPU
// without three CTAs per SM; the scalar one, whose warps take a page at a time,
// 32 to 4 in the same way (whole sparse call, 60 rows of up to
// 49 pages: 24 us with 32, 20 with 4).
constexpr int kScoreTile = 16, kScoreChunkScalar = 32, kScoreChunkLeast = 4, kScoreWarps = 4;
inline int score_chunk_scalar(long long rows, int max_blocks, int sms) {
  int chunk = kScoreChunkScalar;
  while (chunk > kScoreChunkLeast && rows * ((max_blocks + chunk - 1) / chunk) < 3LL * sms)
    chunk >>= 1;
  return chunk;
}
inline int score_chunk(int B, int Hkv, int max_blocks, int sms) {
  const long long cols = (long long)B * ((Hkv + kScoreWarps - 1) / kScoreWarps);
  int chunk = 128;
  while (chunk > kScoreTile && cols * ((max_blocks + chunk - 1) / chunk) < 3LL * sms) chunk >>= 1;
  return chunk;
}

cudaError_t launch_select(const SelectParams& p, int dtype_size, cudaStream_t st);

// Decode attention over fp16 pages (pa_pages.cu): D and block_size multiples of
// 16, rows on 16-byte boundaries, the query on 4-byte ones. Params as for the
// other attention kernels; part_pages / max_parts / slots as tile_plan has them,
// ml_unit as score_unit does.
cudaError_t launch_pages(const Params& p, cudaStream_t st);

}  // namespace xpa
