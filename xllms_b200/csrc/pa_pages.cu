// pa_pages.cu — decode attention over fp16 pages of any 16 n tokens and head
// sizes of 16 n channels, for the kept pages of sparse attention that the TMA
// kernel's fixed boxes do not fit (other head sizes, groups it cannot split).
//
// CTA = (item, 8 query heads of its group); its warps take the item's 16-token
// tiles in turn, each through a two-stage ring of its own that its lanes fill
// with cp.async, as the 4-bit kernel's do. Rows are padded by 16 bytes to an odd
// number of 16-byte units, so ldmatrix reads eight of them without a bank
// conflict. Per tile, with mma.sync m16n8k16 (fp16 in, fp32 sums):
//   S^T(16 tokens x 8 heads) = K . Q^T,  O^T(D x 8 heads) += V^T . P^T
// The weights go in as two fp16 terms (22 bits). The reference point of the
// softmax moves when a score passes it by more than 8 in the exp2 domain, and
// exponents are formed from the distance to it, as in the 4-bit kernel. Rows past
// the end, or of pages that are not there, are filled with zeros.
// Bound by the latency of short items: 4 D bytes a token against 4 D flop per
// head and token leave HBM the limit, and the kept pages of a row are few.
// 43 sequences, 20 heads over 5 of 112, 28 pages each (43 MB): 17 us, where the
// CUDA-core kernel took 110.
#include <algorithm>
#include <utility>

#include "pa_host.h"
#include "pa_q4.cuh"
#include "pa_sparse.h"

namespace xpa {

namespace {

constexpr int kWarps = 4, kPagesHeads = 8;
constexpr float kRaiseBy = 8.f;  // log2 units a score may exceed the reference point by
constexpr float kShiftBy = 7.f;  // weights are 2^(x - m + kShiftBy) <= 2^15

__host__ __device__ constexpr int pages_pitch(int D) { return 2 * D + 16; }  // bytes per row

inline size_t pages_smem(int D, int row) {
  const size_t ring = (size_t)kWarps * 2 * 2 * 16 * pages_pitch(D);
  const size_t merge = (size_t)kWarps * kPagesHeads * (row + 2) * sizeof(float);
  return std::max(ring, merge);
}

// 16 bytes to shared memory, or as many zeros.
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(in ? 16 : 0)
               : "memory");
}

// NGM: 16-channel groups, D <= 16 NGM.
template <int NGM>
__global__ void __launch_bounds__(kWarps * 32) pa_pages_kernel(const Params p, int head_chunks) {
  constexpr int NW = kWarps, HEADS = kPagesHeads, ROW = 16 * NGM + 4;
  extern __shared__ __align__(128) uint8_t smem[];
  pdl_wait_primary();
  pdl_launch_dependents();
  Item it;
  const int col = blockIdx.y + blockIdx.z * kGridY;
  if (col >= p.B * p.Hkv * head_chunks) return;
  const int row = col / head_chunks;
  const ItemKind kind = part_item(p, row, it);
  if (kind == kItemNone) return;
  const int D = p.D, ng = D / 16, bs = p.block_size;
  const int h0 = (col - row * head_chunks) * HEADS;
  const int nh = min(p.GS - h0, HEADS);
  const long long row0 = (long long)it.b * p.Hq + (long long)it.kvh * p.GS + h0;
  if (kind == kItemZero) {
    for (int i = threadIdx.x; i < nh * D; i += NW * 32)
      store_out<__half>(p, row0 + i / D, i % D, 0.f);
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;

  // scores are q . k times sl; see score_unit
  const float sl = p.ml_unit;
  const float sign = p.scale_log2 > 0.f ? 1.f : p.scale_log2 < 0.f ? -1.f : 0.f;
  const float slack = fminf(kRaiseBy / sl, 1e30f);
  // head g: channels 16 s + 2 t, + 1 and + 8, + 9
  uint32_t qf[NGM][2];
  {
    const __half2 sg = __float2half2_rn(sign);
    const __half* q = static_cast<const __half*>(p.q) + (row0 + g) * D + 2 * t;
#pragma unroll
    for (int s = 0; s < NGM; ++s)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        __half2 x = __float2half2_rn(0.f);
        if (g < nh && s < ng) x = __ldg(reinterpret_cast<const __half2*>(q + 16 * s + 8 * k));
        if (sign <= 0.f) x = __hmul2(x, sg);
        qf[s][k] = *reinterpret_cast<const uint32_t*>(&x);
      }
  }

  const long long tok_end = min((long long)it.L, (long long)it.page_end * bs);
  const long long tok_begin = (long long)it.page_begin * bs;
  const int tokens = (int)(tok_end - tok_begin);
  const int tiles = (tokens + 15) >> 4, spp = bs >> 4;
  const int pitch = pages_pitch(D), tile_bytes = 16 * pitch;
  const uint32_t ring = smem_u32(smem) + warp * 4 * tile_bytes;  // [stage][K, V]
  const long long head_off = (long long)it.kvh * p.kv_head_stride;
  const __half* kp = static_cast<const __half*>(p.k) + head_off;
  const __half* vp = static_cast<const __half*>(p.v) + head_off;
  const int* table = p.block_tables + (long long)it.b * p.max_blocks + it.page_begin;

  // This warp's tiles are warp, warp + NW, ...; the table entry of a tile is
  // read a step before its copies, those a step before their use.
  auto entry = [&](int i) { return i < tiles ? __ldg(table + i / spp) : -1; };
  const int cpr = D / 8;  // 16-byte chunks per row
  const int r_first = lane / cpr, c_first = lane - r_first * cpr;
  // Copies tile i, whose entry is e; returns its valid tokens.
  auto issue = [&](int i, int e, uint32_t stage) {
    if (i >= tiles) return 0;
    const bool ok = e >= 0 && (p.num_blocks <= 0 || e < p.num_blocks);
    if (!ok) raise_status(p, kDevBadPage);
    const int here = ok ? min(16, tokens - 16 * i) : 0;
    const long long at = (long long)(ok ? e : 0) * p.kv_block_stride + (long long)(i % spp) * 16 * D;
    int r = r_first, c = c_first;
    for (int n = 0; n < ng; ++n) {  // 16 rows of 2 ng chunks
      const bool in = r < here;
      const long long off = in ? at + r * D + c * 8 : 0;
      const uint32_t dst = ring + stage + r * pitch + c * 16;
      cp_async16_or_zero(dst, kp + off, in);
      cp_async16_or_zero(dst + tile_bytes, vp + off, in);
      for (c += 32; c >= cpr; c -= cpr) ++r;
    }
    return here;
  };

  float o[NGM][4] = {};
  // heads 2 t, 2 t + 1: reference point in units of q . k, and the weights' sum
  float m[2] = {kNoScore, kNoScore}, l[2] = {0.f, 0.f};
  // rows 0-7, 8-15, then the next 8 values; transposed: tokens 0-7, then 8-15
  const uint32_t kfrag = (lane & 15) * pitch + (lane >> 4) * 16;
  const uint32_t vfrag =
      tile_bytes + ((lane & 7) + 8 * (lane >> 4)) * pitch + ((lane >> 3) & 1) * 16;

  uint32_t st = 0;
  int here = issue(warp, entry(warp), st);
  cp_async_commit();
  int e = entry(warp + NW);
#pragma unroll 1
  for (int i = warp; i < tiles; i += NW) {
    const int next = issue(i + NW, e, st ^ (uint32_t)(2 * tile_bytes));
    cp_async_commit();
    e = entry(i + 2 * NW);
    cp_async_wait<1>();
    __syncwarp();
    const uint32_t at = ring + st;
    float x[4] = {}, y[4] = {};  // two chains
#pragma unroll
    for (int s = 0; s < NGM; ++s) {
      if (s >= ng) break;
      uint32_t a[4];
      ldsm_x4(at + kfrag + s * 32, a[0], a[1], a[2], a[3]);
      mma_f16_16816(s & 1 ? y : x, a[0], a[1], a[2], a[3], qf[s][0], qf[s][1]);
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      x[c] += y[c];
      if (g + 8 * (c >> 1) >= here) x[c] = -INFINITY;
    }
    const bool raise = fmaxf(x[0], x[2]) - m[0] > slack || fmaxf(x[1], x[3]) - m[1] > slack;
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float mx = fmaxf(x[c], x[c + 2]);
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
        mx = fmaxf(mx, m[c]);
        const float f = ex2((m[c] - mx) * sl);
        m[c] = mx;
        l[c] *= f;
#pragma unroll
        for (int s = 0; s < NGM; ++s) {
          o[s][c] *= f;
          o[s][c + 2] *= f;
        }
      }
    }
    float w[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) w[c] = ex2(fmaf(x[c] - m[c & 1], sl, kShiftBy));
    l[0] += w[0] + w[2];
    l[1] += w[1] + w[3];
    uint32_t hi[2], lo[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const uint32_t h = pack_half2(w[2 * r], w[2 * r + 1]);
      const float2 f = unpack_half2(h);
      hi[r] = movmatrix_trans(h);
      lo[r] = movmatrix_trans(pack_half2(w[2 * r] - f.x, w[2 * r + 1] - f.y));
    }
#pragma unroll
    for (int s = 0; s < NGM; ++s) {
      if (s >= ng) break;
      uint32_t a[4];
      ldsm_x4_trans(at + vfrag + s * 32, a[0], a[1], a[2], a[3]);
      mma_f16_16816(o[s], a[0], a[1], a[2], a[3], hi[0], hi[1]);
      mma_f16_16816(o[s], a[0], a[1], a[2], a[3], lo[0], lo[1]);
    }
    __syncwarp();  // the stage may be filled again
    st ^= (uint32_t)(2 * tile_bytes);
    here = next;
  }
  cp_async_wait<0>();
  __syncthreads();  // the rings become merge space

  float* so = reinterpret_cast<float*>(smem);   // [NW][heads][ROW]
  float* sml = so + (size_t)NW * HEADS * ROW;   // [NW][heads][2]
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int head = 2 * t + c;
    float* dst = so + (size_t)(warp * HEADS + head) * ROW;
#pragma unroll
    for (int s = 0; s < NGM; ++s) {
      dst[16 * s + g] = o[s][c];
      dst[16 * s + g + 8] = o[s][c + 2];
    }
    float sum = l[c];
#pragma unroll
    for (int off = 4; off < 32; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    if (g == 0) {
      sml[(warp * HEADS + head) * 2] = m[c] == kNoScore ? -INFINITY : m[c];
      sml[(warp * HEADS + head) * 2 + 1] = sum;
    }
  }
  __syncthreads();
  merge_warps<NW, HEADS, ROW>(p, it, so, sml, row0, nh, D);
}

template <int NGM>
cudaError_t launch_pages_t(const Params& p, cudaStream_t st) {
  auto kern = pa_pages_kernel<NGM>;
  constexpr int ROW = 16 * NGM + 4;
  static std::atomic<unsigned long long> done{0};
  cudaError_t e = host::smem_limit(kern, pages_smem(16 * NGM, ROW), true, done);
  if (e != cudaSuccess) return e;
  const int chunks = (p.GS + kPagesHeads - 1) / kPagesHeads;
  const long long cols = (long long)p.B * p.Hkv * chunks;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)p.max_parts, (unsigned)std::min<long long>(cols, kGridY),
                     (unsigned)((cols + kGridY - 1) / kGridY));
  cfg.blockDim = dim3(kWarps * 32);
  cfg.dynamicSmemBytes = pages_smem(p.D, ROW);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, p, chunks);
}

}  // namespace

cudaError_t launch_pages(const Params& p, cudaStream_t st) {
  if (p.D <= 64) return launch_pages_t<4>(p, st);
  if (p.D <= 128) return launch_pages_t<8>(p, st);
  return launch_pages_t<16>(p, st);
}

}  // namespace xpa
