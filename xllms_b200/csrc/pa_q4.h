// pa_q4.h — host-side launchers of the 4-bit KV cache kernels (pa_q4.cu).
#pragma once

#include <cuda_runtime.h>

#include "pa_device.cuh"

namespace xpa {

// Rows into (write) or out of (read) 4-bit pools by slot. Pool strides in
// bytes, the rows' token_stride in elements.
struct Q4RowsParams {
  void* key;    // fp16 rows; read by the write, written by the read
  void* value;
  void* key_cache;
  void* value_cache;
  const long long* slots;
  long long kv_block_stride, kv_head_stride, token_stride;
  long long num_slots;  // slots >= this are skipped like negative ones
  int num_tokens, Hkv, D, block_size;
  int vec16;  // every row starts on a 16-byte boundary
  float k_scale, v_scale;
  float k_inverse, v_inverse;  // 1 / scale rounded to nearest
  int divide;                  // 1: divide by the scales instead
  int clamp;                   // 1: a value read back may pass the fp16 range
  int sms;
  int warps_per_token;  // set by the launchers
};

cudaError_t launch_q4_write(const Q4RowsParams& a, cudaStream_t st);
cudaError_t launch_q4_read(const Q4RowsParams& a, cudaStream_t st);

// Decode attention over 4-bit pools; Params as for the other attention
// kernels, with the pool strides in bytes. p.part_pages / max_parts / slots
// as planned by host::tile_plan, p.ml_unit from host::score_unit.
cudaError_t launch_q4_attention(const Params& p, cudaStream_t st);

}  // namespace xpa
