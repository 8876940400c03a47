// pa_sparse.cu — page bounds, and the selection of the pages that sparse
// decode attention reads.
//
// A page's bounds are, per KV head and channel, the lowest and the highest of
// its keys. For a query head q the page's score is
//   sum_d max(q_d lo_d, q_d hi_d) = sum_d (q_d^+ hi_d + q_d^- lo_d),
// no less than any q . k of the page; the score of a KV head is the largest
// over its query heads. The best pages are kept, in the exact order of the
// scores, ties to the earlier page.
#include <cfloat>
#include <climits>
#include <utility>

#include "pa_q4.cuh"
#include "pa_sparse.h"

namespace xpa {

namespace {

__device__ __forceinline__ int clamped_len(const int* lens, int b, int max_blocks, int bs,
                                           int* status, bool tell) {
  const int L = __ldg(lens + b);
  const long long cap = (long long)max_blocks * bs;
  if (L < 0 || L > cap) {
    if (tell && status) atomicOr(status, kDevSeqClamped);
    return L < 0 ? 0 : (int)cap;
  }
  return L;
}

// Keys and queries as the bounds and scores see them: finite, NaN as 0.
__device__ __forceinline__ float tame(float x, float big) {
  return isnan(x) ? 0.f : fminf(fmaxf(x, -big), big);
}

// ════════════════════════════════════════════════════════════════════════
// Page bounds: one CTA per (sequence, due page), a warp per KV head. HBM-bound:
// a page's keys are read once with 16-byte loads (a lane takes E channels of
// every R-th token, R = 32 / vectors per row), the bounds written once. Two
// heads' loads are in flight together, which with a page's table entry read
// once per CTA took 8 prompts of 2-32K tokens from 117 to 66 us (359 MB).
// Minima and maxima are taken in the cache's type with a NaN passed on; a warp
// that ends with a NaN or an infinity goes over its page again, element by
// element. Pages shared by several sequences are full in each and get the same
// bytes from all.
// ════════════════════════════════════════════════════════════════════════
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// A 32-bit word of a row: two fp16 channels or one fp32 channel.
template <typename T>
struct BoundsWord;
template <>
struct BoundsWord<__half> {
  static constexpr uint32_t kTop = 0x7bff7bffu;  // 65504, twice
  static constexpr uint32_t kBottom = 0xfbfffbffu;
  static __device__ __forceinline__ __half2 h2(uint32_t w) {
    return *reinterpret_cast<const __half2*>(&w);
  }
  static __device__ __forceinline__ uint32_t bits(__half2 h) {
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ uint32_t lower(uint32_t a, uint32_t b) {
    return bits(__hmin2_nan(h2(a), h2(b)));
  }
  static __device__ __forceinline__ uint32_t upper(uint32_t a, uint32_t b) {
    return bits(__hmax2_nan(h2(a), h2(b)));
  }
  // whether either channel is an infinity or a NaN
  static __device__ __forceinline__ bool odd(uint32_t a) {
    return (a & 0x7c00u) == 0x7c00u || (a & 0x7c000000u) == 0x7c000000u;
  }
};
template <>
struct BoundsWord<float> {
  static constexpr uint32_t kTop = 0x7f7fffffu;  // FLT_MAX
  static constexpr uint32_t kBottom = 0xff7fffffu;
  static __device__ __forceinline__ uint32_t lower(uint32_t a, uint32_t b) {
    return __float_as_uint(min_nan(__uint_as_float(a), __uint_as_float(b)));
  }
  static __device__ __forceinline__ uint32_t upper(uint32_t a, uint32_t b) {
    return __float_as_uint(max_nan(__uint_as_float(a), __uint_as_float(b)));
  }
  static __device__ __forceinline__ bool odd(uint32_t a) {
    return (a & 0x7f800000u) == 0x7f800000u;
  }
};

struct DuePage {
  long long page;
  int live;  // valid tokens of the page
};

// The i-th due page of sequence b; `tell`: this thread reports what is wrong.
__device__ __forceinline__ bool due_page(const BoundsParams& p, int b, int i, bool tell,
                                         DuePage& out) {
  const int L =
      clamped_len(p.seq_lens, b, p.max_blocks, p.block_size, p.status, tell && i == 0);
  const int npages = (int)(((long long)L + p.block_size - 1) / p.block_size);
  const int first = p.num_new > 0 ? max(0, L - p.num_new) / p.block_size : 0;
  const int at = first + i;
  if (at >= npages) return false;
  const int e = __ldg(p.block_tables + (long long)b * p.max_blocks + at);
  if (e < 0 || (p.num_blocks > 0 && e >= p.num_blocks)) {
    if (tell && p.status) atomicOr(p.status, kDevBadPage);
    return false;
  }
  out.page = e;
  out.live = min(p.block_size, L - at * p.block_size);
  return true;
}

// One page of one head, element by element.
template <typename T>
__device__ __noinline__ void bounds_by_element(const T* key, T* dst, int D, int live, int lane) {
  constexpr float big = sizeof(T) == 2 ? 65504.f : FLT_MAX;
  for (int d = lane; d < D; d += 32) {
    float lo = big, hi = -big;
    for (int s = 0; s < live; ++s) {
      const float x = tame(to_float<T>(key[(long long)s * D + d]), big);
      lo = fminf(lo, x);
      hi = fmaxf(hi, x);
    }
    dst[d] = from_float<T>(lo);
    dst[D + d] = from_float<T>(hi);
  }
}

template <typename T>
__global__ void __launch_bounds__(128) pa_bounds_kernel(const BoundsParams p) {
  constexpr int E = 16 / sizeof(T);
  using Word = BoundsWord<T>;
  pdl_wait_primary();
  const int b = blockIdx.x / p.pages_per_seq, i = blockIdx.x - b * p.pages_per_seq;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  DuePage dp;
  if (!due_page(p, b, i, threadIdx.x == 0, dp)) return;
  const T* page = static_cast<const T*>(p.key_cache) + dp.page * p.kv_block_stride;
  T* bounds = static_cast<T*>(p.bounds) + dp.page * p.Hkv * 2 * p.D;
  if (!p.vec) {
    for (int h = warp; h < p.Hkv; h += 4)
      bounds_by_element(page + h * p.kv_head_stride, bounds + (long long)h * 2 * p.D, p.D, dp.live,
                        lane);
    return;
  }
  const int nv = p.D / E;  // vectors per row
  for (int h0 = warp; h0 < p.Hkv; h0 += 8) {
    bool odd[2] = {false, false};
    const bool two = h0 + 4 < p.Hkv;
    for (int v0 = 0; v0 < nv; v0 += 32) {
      const int cols = min(nv - v0, 32), R = 32 / cols;
      const int row = lane / cols, v = v0 + lane - row * cols;
      uint32_t lo[2][4], hi[2][4];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          lo[u][k] = Word::kTop;
          hi[u][k] = Word::kBottom;
        }
      const T* k0 = page + h0 * p.kv_head_stride + v * E;
      const T* k1 = k0 + (two ? 4 * p.kv_head_stride : 0);
      if (row < R) {
#pragma unroll 4
        for (int s = row; s < dp.live; s += R) {
          const uint4 a = __ldg(reinterpret_cast<const uint4*>(k0 + (long long)s * p.D));
          const uint4 c = __ldg(reinterpret_cast<const uint4*>(k1 + (long long)s * p.D));
          const uint32_t x[2][4] = {{a.x, a.y, a.z, a.w}, {c.x, c.y, c.z, c.w}};
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              lo[u][k] = Word::lower(lo[u][k], x[u][k]);
              hi[u][k] = Word::upper(hi[u][k], x[u][k]);
            }
        }
      }
      // lanes v, v + cols, ... hold the same channels; the first row's gather them
      for (int r = 1; r < R; ++r)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t l = __shfl_sync(0xffffffffu, lo[u][k], (lane + r * cols) & 31);
            const uint32_t m = __shfl_sync(0xffffffffu, hi[u][k], (lane + r * cols) & 31);
            if (row == 0) {
              lo[u][k] = Word::lower(lo[u][k], l);
              hi[u][k] = Word::upper(hi[u][k], m);
            }
          }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (row == 0 && (u == 0 || two)) {
          T* dst = bounds + (long long)(h0 + 4 * u) * 2 * p.D + v * E;
          *reinterpret_cast<uint4*>(dst) = make_uint4(lo[u][0], lo[u][1], lo[u][2], lo[u][3]);
          *reinterpret_cast<uint4*>(dst + p.D) = make_uint4(hi[u][0], hi[u][1], hi[u][2], hi[u][3]);
#pragma unroll
          for (int k = 0; k < 4; ++k) odd[u] |= Word::odd(lo[u][k]) || Word::odd(hi[u][k]);
        }
      }
    }
    __syncwarp();  // what follows may store the same bounds from other lanes
#pragma unroll
    for (int u = 0; u < 2; ++u)
      if (__any_sync(0xffffffffu, odd[u]))
        bounds_by_element(page + (h0 + 4 * u) * p.kv_head_stride,
                          bounds + (long long)(h0 + 4 * u) * 2 * p.D, p.D, dp.live, lane);
  }
}

// Bounds of 4-bit keys: of the values that nxt_read_cache_q4 returns, fp16.
__global__ void __launch_bounds__(128) pa_bounds_q4_kernel(const BoundsParams p) {
  pdl_wait_primary();
  const int b = blockIdx.x / p.pages_per_seq, i = blockIdx.x - b * p.pages_per_seq;
  const int warp = threadIdx.x >> 5;
  DuePage dp;
  if (!due_page(p, b, i, threadIdx.x == 0, dp)) return;
  const int v = threadIdx.x & 31;  // channels 8 v .. 8 v + 7; D <= 256
  if (v >= p.D / 8) return;
  for (int h = warp; h < p.Hkv; h += 4) {
    const uint8_t* tile0 = static_cast<const uint8_t*>(p.key_cache) + dp.page * p.kv_block_stride +
                           h * p.kv_head_stride;
    __half* dst = static_cast<__half*>(p.bounds) + (dp.page * p.Hkv + h) * 2 * p.D;
    float lo[8], hi[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      lo[k] = 65504.f;
      hi[k] = -65504.f;
    }
#pragma unroll 4
    for (int s = 0; s < dp.live; ++s) {
      const uint8_t* tile = tile0 + (long long)(s >> 4) * (9 * p.D);
      const int tok = s & 15;
      const uint8_t* at = tile + q4_k_off(p.D, tok, v);
      const uint32_t code = *reinterpret_cast<const uint16_t*>(at) |
                            ((uint32_t) * reinterpret_cast<const uint16_t*>(at + p.D / 8) << 16);
      const float sc = fp8_to_float<kKvE4M3>(tile[q4_k_scale_off(p.D, tok, v >> 1)]);
      uint32_t h[4];
      q4x8_to_h2(code, h);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 f = unpack_half2(h[k]);
        const float a = tame(f.x * sc * p.k_scale, 65504.f), b = tame(f.y * sc * p.k_scale, 65504.f);
        lo[2 * k] = fminf(lo[2 * k], a);
        hi[2 * k] = fmaxf(hi[2 * k], a);
        lo[2 * k + 1] = fminf(lo[2 * k + 1], b);
        hi[2 * k + 1] = fmaxf(hi[2 * k + 1], b);
      }
    }
    // rounding to fp16 is monotone: it may follow the minimum
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      dst[8 * v + k] = __float2half_rn(lo[k]);
      dst[p.D + 8 * v + k] = __float2half_rn(hi[k]);
    }
  }
}

// ════════════════════════════════════════════════════════════════════════
// Selection, first kernel: fp32 scores of chunk_pages pages of one (sequence,
// KV head) row per CTA, as keys whose unsigned order is the scores' (0: the
// table names no page). Rows that keep every page are skipped.
// ════════════════════════════════════════════════════════════════════════
__device__ __forceinline__ unsigned key_of(float s) {
  if (isnan(s)) return 1u;  // from bounds that no call wrote
  const unsigned u = __float_as_uint(s);
  return (u >> 31) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float score_of(unsigned k) {
  return __uint_as_float((k >> 31) ? (k & 0x7fffffffu) : ~k);
}
__device__ __forceinline__ unsigned long long key_of(double s) {
  if (isnan(s)) return 1ull;
  const unsigned long long u = (unsigned long long)__double_as_longlong(s);
  return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}

// The entry of page `at` of sequence b, or -1 (with the status bit) when it
// names no page or one whose per-head index would not fit.
__device__ __forceinline__ int table_entry(const SelectParams& p, int b, int at) {
  const int e = __ldg(p.block_tables + (long long)b * p.max_blocks + at);
  if (e < 0 || (p.num_blocks > 0 && e >= p.num_blocks) ||
      (long long)e * p.head_pages + p.Hkv - 1 > INT_MAX) {
    if (p.status) atomicOr(p.status, kDevBadPage);
    return -1;
  }
  return e;
}

// fp16 with 16-byte rows: 16 pages x 8 heads per warp step on mma.sync. The
// work per page is 2 D bytes x 2 against 4 D flop per head, far below the
// tensor ridge: bound by HBM. k index 2 t, 2 t + 1, 2 t + 8, 2 t + 9 of the
// two steps over channels 32 c .. + 31 are channels 32 c + 8 t .. + 7, so a
// lane's share of a bounds row is one 16-byte load.
// C: 32-channel blocks, ceil(D / 32) rounded up.
template <int C>
__global__ void __launch_bounds__(128) pa_score_mma_kernel(const SelectParams p) {
  __shared__ float s_max[4];
  pdl_wait_primary();
  const int row = blockIdx.x / p.chunks, chunk = blockIdx.x - row * p.chunks;
  const int b = row / p.Hkv, h = row - b * p.Hkv;
  const int L = clamped_len(p.seq_lens, b, p.max_blocks, p.block_size, nullptr, false);
  const int npages = (int)(((long long)L + p.block_size - 1) / p.block_size);
  const int page_end = min(npages, (chunk + 1) * p.chunk_pages);
  if (npages <= p.keep || chunk * p.chunk_pages >= npages) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const __half* bounds = static_cast<const __half*>(p.bounds) + (long long)h * 2 * p.D;
  const long long page_stride = (long long)p.Hkv * 2 * p.D;
  unsigned* keys = p.keys + (long long)row * p.max_blocks;
  float big = 0.f;
  for (int h0 = 0; h0 < p.GS; h0 += 8) {
    // q^- and q^+ of head h0 + g, finite, times the sign of the score scale
    uint32_t qn[C][4], qp[C][4];
    {
      const __half* q = static_cast<const __half*>(p.q) +
                        ((long long)b * p.Hq + (long long)h * p.GS + h0 + g) * p.D + 8 * t;
      const __half2 zero = __float2half2_rn(0.f), top = __float2half2_rn(65504.f);
      const __half2 sg = __float2half2_rn(p.sign);
#pragma unroll
      for (int c = 0; c < C; ++c) {
        uint4 u = make_uint4(0u, 0u, 0u, 0u);
        if (h0 + g < p.GS && 32 * c + 8 * t < p.D)
          u = __ldg(reinterpret_cast<const uint4*>(q + 32 * c));
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          // max and min drop a NaN operand, so a NaN becomes 0 in both halves
          const __half2 x = *reinterpret_cast<const __half2*>(&w[k]);
          __half2 pos = __hmin2(__hmax2(x, zero), top);
          __half2 neg = __hmax2(__hmin2(x, zero), __hneg2(top));
          if (p.sign <= 0.f) {
            const __half2 a = __hmul2(neg, sg), z = __hmul2(pos, sg);
            pos = a;
            neg = z;
          }
          qp[c][k] = *reinterpret_cast<const uint32_t*>(&pos);
          qn[c][k] = *reinterpret_cast<const uint32_t*>(&neg);
        }
      }
    }
    // entries of this warp's next tile, read one tile ahead
    int p0 = chunk * p.chunk_pages + warp * 16;
    int next = lane < 16 && p0 + lane < page_end ? table_entry(p, b, p0 + lane) : -1;
    for (; p0 < page_end; p0 += 64) {
      const int e0 = __shfl_sync(0xffffffffu, next, g), e1 = __shfl_sync(0xffffffffu, next, g + 8);
      next = lane < 16 && p0 + 64 + lane < page_end ? table_entry(p, b, p0 + 64 + lane) : -1;
      const uint4 none = make_uint4(0u, 0u, 0u, 0u);
      uint4 a[2][2][C];  // [lo, hi][row g, row g + 8][block]
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const bool in = 32 * c + 8 * t < p.D;
#pragma unroll
        for (int side = 0; side < 2; ++side) {
          const long long off = (long long)side * p.D + 32 * c + 8 * t;
          a[side][0][c] = in && e0 >= 0 ? __ldg(reinterpret_cast<const uint4*>(
                                              bounds + e0 * page_stride + off))
                                        : none;
          a[side][1][c] = in && e1 >= 0 ? __ldg(reinterpret_cast<const uint4*>(
                                              bounds + e1 * page_stride + off))
                                        : none;
        }
      }
      float x[4] = {};
      __half2 mx = __float2half2_rn(0.f);
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int side = 0; side < 2; ++side) {
          const uint4 u = a[side][0][c], v = a[side][1][c];
          const uint32_t* qq = side ? qp[c] : qn[c];
          mma_f16_16816(x, u.x, v.x, u.y, v.y, qq[0], qq[1]);
          mma_f16_16816(x, u.z, v.z, u.w, v.w, qq[2], qq[3]);
          if (h0 == 0) {
            const uint32_t all[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
            for (int k = 0; k < 8; ++k)
              mx = __hmax2(mx, __habs2(*reinterpret_cast<const __half2*>(&all[k])));
          }
        }
      big = fmaxf(big, fmaxf(__low2float(mx), __high2float(mx)));
      // heads h0 + 2 t, + 1 of pages g and g + 8: the largest over the group
      const bool c0 = h0 + 2 * t < p.GS, c1 = h0 + 2 * t + 1 < p.GS;
      float r0 = fmaxf(c0 ? x[0] : -INFINITY, c1 ? x[1] : -INFINITY);
      float r1 = fmaxf(c0 ? x[2] : -INFINITY, c1 ? x[3] : -INFINITY);
      r0 = fmaxf(r0, __shfl_xor_sync(0xffffffffu, r0, 1));
      r1 = fmaxf(r1, __shfl_xor_sync(0xffffffffu, r1, 1));
      r0 = fmaxf(r0, __shfl_xor_sync(0xffffffffu, r0, 2));
      r1 = fmaxf(r1, __shfl_xor_sync(0xffffffffu, r1, 2));
      if (t == 0) {
        if (p0 + g < page_end) {
          unsigned k = e0 < 0 ? 0u : key_of(r0);
          if (h0 > 0) k = max(k, keys[p0 + g]);
          keys[p0 + g] = k;
        }
        if (p0 + g + 8 < page_end) {
          unsigned k = e1 < 0 ? 0u : key_of(r1);
          if (h0 > 0) k = max(k, keys[p0 + g + 8]);
          keys[p0 + g + 8] = k;
        }
      }
    }
  }
  big = warp_max(big);
  if (lane == 0) s_max[warp] = big;
  __syncthreads();
  if (threadIdx.x == 0)
    p.absmax[(long long)row * p.chunks + chunk] =
        fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
}

// Every other type and size: one warp per page, lanes across the channels.
template <typename T>
__global__ void __launch_bounds__(128) pa_score_kernel(const SelectParams p) {
  __shared__ float s_max[4];
  constexpr float top = sizeof(T) == 2 ? 65504.f : FLT_MAX;
  pdl_wait_primary();
  const int row = blockIdx.x / p.chunks, chunk = blockIdx.x - row * p.chunks;
  const int b = row / p.Hkv, h = row - b * p.Hkv;
  const int L = clamped_len(p.seq_lens, b, p.max_blocks, p.block_size, nullptr, false);
  const int npages = (int)(((long long)L + p.block_size - 1) / p.block_size);
  const int page_end = min(npages, (chunk + 1) * p.chunk_pages);
  if (npages <= p.keep || chunk * p.chunk_pages >= npages) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T* q = static_cast<const T*>(p.q) + ((long long)b * p.Hq + (long long)h * p.GS) * p.D;
  float big = 0.f;
  for (int at = chunk * p.chunk_pages + warp; at < page_end; at += 4) {
    const int e = table_entry(p, b, at);
    unsigned key = 0;
    if (e >= 0) {
      const T* lo = static_cast<const T*>(p.bounds) + ((long long)e * p.Hkv + h) * 2 * p.D;
      float best = -INFINITY;
      for (int x = 0; x < p.GS; ++x) {
        float s = 0.f;
        for (int d = lane; d < p.D; d += 32) {
          const float qd = p.sign * tame(to_float<T>(q[(long long)x * p.D + d]), top);
          const float l = to_float<T>(lo[d]), u = to_float<T>(lo[p.D + d]);
          s = fmaf(fmaxf(qd, 0.f), u, s);
          s = fmaf(fminf(qd, 0.f), l, s);
          if (x == 0) big = fmaxf(big, fmaxf(fabsf(l), fabsf(u)));
        }
        best = fmaxf(best, warp_sum(s));
      }
      key = key_of(best);
    }
    if (lane == 0) p.keys[(long long)row * p.max_blocks + at] = key;
  }
  big = warp_max(big);
  if (lane == 0) s_max[warp] = big;
  __syncthreads();
  if (threadIdx.x == 0)
    p.absmax[(long long)row * p.chunks + chunk] =
        fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
}

// ════════════════════════════════════════════════════════════════════════
// Selection, second kernel: one CTA per row.
//   1. T = the r-th largest fp32 score, by bisection on the ordered keys
//      (each step one count over the row and one barrier).
//   2. A score is off by at most E, so T is within E of the true r-th
//      largest: scores above T + 2 E are in, those below T - 2 E out. When
//      more lie between than places are left, those few are scored again in
//      64 bits (products of the operands are exact there) and the best taken,
//      the earlier page on a tie.
//   3. The kept pages go out in order, as per-head page ids.
// E: a tensor-core step of 16 products and its accumulator is taken to be off
// by at most 2^-18 of the sum of their magnitudes, a scalar sum by less; with
// up to 16 steps and that sum at most |q|_1 max |bound|, E = 2^-14 of the
// latter covers both.
// ════════════════════════════════════════════════════════════════════════
constexpr int kNearCap = 1024;  // near pages that are ranked in shared memory

template <int NT>
struct BlockCount {
  int buf[2][NT / 32];
};

// Sum of every thread's `mine`, to every thread; `turn` alternates the buffer
// so that one barrier suffices.
template <int NT>
__device__ __forceinline__ int block_sum(BlockCount<NT>& s, int mine, int& turn) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int w = __reduce_add_sync(0xffffffffu, mine);
  if (lane == 0) s.buf[turn][warp] = w;
  __syncthreads();
  const int r = __reduce_add_sync(0xffffffffu, lane < NT / 32 ? s.buf[turn][lane] : 0);
  turn ^= 1;
  return r;
}

// The largest T in [lo, hi] that at least r keys reach; at least r reach lo.
template <int NT, typename K, typename Count>
__device__ __forceinline__ K bisect(BlockCount<NT>& s, int& turn, K lo, K hi, int r, Count reach) {
  while (lo < hi) {
    const K mid = lo + (hi - lo) / 2 + ((hi - lo) & 1);
    if (block_sum<NT>(s, reach(mid), turn) >= r)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

// NT threads hold the first NT * KPT keys of the row in registers (thread t
// the pages t, t + NT, ...); a longer row's others are read again each time.
template <typename T, int NT, int KPT>
__global__ void __launch_bounds__(NT, 1) pa_select_kernel(const SelectParams p) {
  constexpr int NWARP = NT / 32;
  __shared__ BlockCount<NT> s_cnt;
  __shared__ float s_red[2][NWARP];
  __shared__ unsigned s_ends[2];
  __shared__ int s_near;
  __shared__ unsigned s_near_page[kNearCap];
  __shared__ unsigned long long s_near_key[kNearCap];
  __shared__ int s_count[KPT * NWARP];
  constexpr float top = sizeof(T) == 2 ? 65504.f : FLT_MAX;
  pdl_wait_primary();
  const int row = blockIdx.x;
  const int b = row / p.Hkv, h = row - b * p.Hkv;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int L = clamped_len(p.seq_lens, b, p.max_blocks, p.block_size, p.status,
                            h == 0 && tid == 0);
  const int n = (int)(((long long)L + p.block_size - 1) / p.block_size);
  const bool scored = n > p.keep;
  unsigned* keys = p.keys + (long long)row * p.max_blocks;
  const int first = p.sink, last = n - p.recent;  // [first, last): pages that compete
  unsigned take = 1u;  // a competing page with a key of at least this is kept
  unsigned kr[KPT];    // 0: the table names no page there
#pragma unroll
  for (int i = 0; i < KPT; ++i) {
    const int at = tid + i * NT;
    kr[i] = 0u;
    if (at < n) kr[i] = scored ? keys[at] : table_entry(p, b, at) >= 0;
  }
  if (scored) {
    const int r = p.keep - p.sink - p.recent;
    int turn = 0;
    int mine = 0;
    unsigned kmin = 0xffffffffu, kmax = 0u;
    // f(page, key) for the competing pages with a key
    auto each = [&](auto f) {
#pragma unroll
      for (int i = 0; i < KPT; ++i) {
        const int at = tid + i * NT;
        if (at >= first && at < last && kr[i]) f(at, kr[i]);
      }
      for (int at = tid + KPT * NT; at < last; at += NT)
        if (at >= first && keys[at]) f(at, keys[at]);
    };
    each([&](int, unsigned k) {
      ++mine;
      kmin = min(kmin, k);
      kmax = max(kmax, k);
    });
    if (tid == 0) {
      s_ends[0] = 0xffffffffu;
      s_ends[1] = 0u;
      s_near = 0;
    }
    const int eligible = block_sum<NT>(s_cnt, mine, turn);
    if (r <= 0) {
      take = 0xffffffffu;  // no competing page fits; no key is this large
    } else if (eligible > r) {
      kmin = __reduce_min_sync(0xffffffffu, kmin);
      kmax = __reduce_max_sync(0xffffffffu, kmax);
      if (lane == 0) {
        atomicMin(&s_ends[0], kmin);
        atomicMax(&s_ends[1], kmax);
      }
      // max |bound| of the row and max over heads of |q|_1
      float big = 0.f, l1 = 0.f;
      const int chunks = (n + p.chunk_pages - 1) / p.chunk_pages;
      for (int i = tid; i < chunks; i += NT)
        big = fmaxf(big, p.absmax[(long long)row * p.chunks + i]);
      const T* q = static_cast<const T*>(p.q) + ((long long)b * p.Hq + (long long)h * p.GS) * p.D;
      for (int x = warp; x < p.GS; x += NWARP) {
        float s = 0.f;
        for (int d = lane; d < p.D; d += 32)
          s += fabsf(tame(to_float<T>(q[(long long)x * p.D + d]), top));
        l1 = fmaxf(l1, warp_sum(s));
      }
      big = warp_max(big);
      if (lane == 0) {
        s_red[0][warp] = big;
        s_red[1][warp] = l1;
      }
      __syncthreads();
      big = warp_max(lane < NWARP ? s_red[0][lane] : 0.f);
      l1 = warp_max(lane < NWARP ? s_red[1][lane] : 0.f);
      const unsigned T32 =
          bisect<NT, unsigned>(s_cnt, turn, s_ends[0], s_ends[1], r, [&](unsigned t) {
            int c = 0;
            each([&](int, unsigned k) { c += k >= t; });
            return c;
          });
      const float E = big * l1 * 0x1p-14f + 0x1p-118f;
      const float tf = score_of(T32);
      unsigned near_lo = 1u, near_hi = 0xfffffffeu;
      if (fabsf(E) < 0x1p126f && fabsf(tf) < 0x1p126f) {
        near_lo = max(1u, key_of(tf - 2.001f * E));
        near_hi = key_of(tf + 2.001f * E);
      }
      int above = 0, near = 0;
      each([&](int, unsigned k) {
        above += k > near_hi;
        near += k >= near_lo && k <= near_hi;
      });
      above = block_sum<NT>(s_cnt, above, turn);
      near = block_sum<NT>(s_cnt, near, turn);
      const int need = r - above;
      take = near_lo;
      if (near > need) {
        const bool few = near <= kNearCap;
        unsigned* lp = few ? s_near_page : p.near_page + (long long)row * p.max_blocks;
        unsigned long long* lk = few ? s_near_key : p.near_key + (long long)row * p.max_blocks;
        each([&](int at, unsigned k) {
          if (k >= near_lo && k <= near_hi) lp[atomicAdd(&s_near, 1)] = (unsigned)at;
        });
        __syncthreads();
        for (int i = warp; i < near; i += NWARP) {
          const int e = table_entry(p, b, (int)lp[i]);
          double best = -INFINITY;
          const T* lo = static_cast<const T*>(p.bounds) +
                        ((long long)(e < 0 ? 0 : e) * p.Hkv + h) * 2 * p.D;
          for (int x = 0; x < p.GS && e >= 0; ++x) {
            double s = 0.0;
            for (int d = lane; d < p.D; d += 32) {
              const double qd =
                  (double)(p.sign * tame(to_float<T>(q[(long long)x * p.D + d]), top));
              s = fma(fmax(qd, 0.0), (double)to_float<T>(lo[p.D + d]), s);
              s = fma(fmin(qd, 0.0), (double)to_float<T>(lo[d]), s);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
            best = fmax(best, s);
          }
          if (lane == 0) lk[i] = key_of(best);
        }
        __syncthreads();
        // kept near pages get the key near_hi, the others 0
        if (few) {
          for (int i = tid; i < near; i += NT) {
            const unsigned long long k = lk[i];
            const unsigned at = lp[i];
            int rank = 0;
            for (int o = 0; o < near; ++o) rank += lk[o] > k || (lk[o] == k && lp[o] < at);
            keys[at] = rank < need ? near_hi : 0u;
          }
        } else {
          const unsigned long long T64 = bisect<NT, unsigned long long>(
              s_cnt, turn, 0ull, ~0ull, need, [&](unsigned long long t) {
                int c = 0;
                for (int i = tid; i < near; i += NT) c += lk[i] >= t;
                return c;
              });
          int more = 0;
          for (int i = tid; i < near; i += NT) more += lk[i] > T64;
          more = block_sum<NT>(s_cnt, more, turn);
          // of the pages that tie at T64, the first need - more: those up to `cut`
          const unsigned cut = ~bisect<NT, unsigned>(
              s_cnt, turn, ~(unsigned)(p.max_blocks), ~0u, need - more, [&](unsigned t) {
                int c = 0;
                for (int i = tid; i < near; i += NT) c += lk[i] == T64 && ~lp[i] >= t;
                return c;
              });
          for (int i = tid; i < near; i += NT) {
            const bool in = lk[i] > T64 || (lk[i] == T64 && lp[i] <= cut);
            keys[lp[i]] = in ? near_hi : 0u;
          }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < KPT; ++i) {
          const int at = tid + i * NT;
          if (at >= first && at < last && kr[i] >= near_lo && kr[i] <= near_hi) kr[i] = keys[at];
        }
      }
    }
  }
  // ── the kept pages, in order: NT * KPT pages a round ────────────────────
  int* tab = p.sel_tables + (long long)row * p.keep;
  int* pages = p.sel_pages ? p.sel_pages + (long long)row * p.keep : nullptr;
  int done = 0;
  bool tail = false;  // the sequence's last page is kept
  for (int base = 0; base < n; base += NT * KPT) {
    unsigned in = 0;  // bit i: page base + tid + i * NT is kept
    unsigned before[KPT];
#pragma unroll
    for (int i = 0; i < KPT; ++i) {
      const int at = base + tid + i * NT;
      unsigned k = kr[i];
      if (base > 0) {
        k = 0u;
        if (at < n) k = scored ? keys[at] : table_entry(p, b, at) >= 0;
      }
      const bool kept = k && (!scored || at < first || at >= last || k >= take);
      const unsigned m = __ballot_sync(0xffffffffu, kept);
      if (kept) in |= 1u << i;
      before[i] = __popc(m & ((1u << lane) - 1u));
      if (lane == 0) s_count[i * NWARP + warp] = __popc(m);
    }
    __syncthreads();
    // exclusive sums of s_count, by the first warp
    constexpr int PER = (KPT * NWARP + 31) / 32;
    if (warp == 0) {
      int c[PER], sum = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int x = lane * PER + i;
        c[i] = x < KPT * NWARP ? s_count[x] : 0;
        sum += c[i];
      }
      int pre = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, pre, o);
        if (lane >= o) pre += y;
      }
      if (lane == 31) s_near = pre;
      pre -= sum;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int x = lane * PER + i;
        if (x < KPT * NWARP) s_count[x] = pre;
        pre += c[i];
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < KPT; ++i)
      if (in >> i & 1u) {
        const int at = base + tid + i * NT;
        const int to = done + s_count[i * NWARP + warp] + (int)before[i];
        const int e = __ldg(p.block_tables + (long long)b * p.max_blocks + at);
        tab[to] = (int)((long long)e * p.head_pages + h);
        if (pages) pages[to] = at;
        if (at == n - 1) tail = true;
      }
    done += s_near;
    __syncthreads();
  }
  tail = __syncthreads_or(tail);
  for (int i = done + tid; i < p.keep; i += NT) {
    tab[i] = -1;
    if (pages) pages[i] = -1;
  }
  if (tid == 0)
    p.sel_lens[row] = done * p.block_size - (tail ? n * p.block_size - L : 0);
}

template <typename... KArgs, typename... Args>
cudaError_t launch_pdl(void (*kern)(KArgs...), long long grid, unsigned block, cudaStream_t st,
                       Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(block);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...);
}

template <typename T>
cudaError_t launch_select_t(const SelectParams& p, cudaStream_t st) {
  const long long rows = (long long)p.B * p.Hkv;
  // no sequence can hold more pages than are kept: nothing is scored
  if (p.max_blocks > p.keep) {
    cudaError_t e;
    if (!p.vec)
      e = launch_pdl(pa_score_kernel<T>, rows * p.chunks, 128, st, p);
    else if (p.D <= 64)
      e = launch_pdl(pa_score_mma_kernel<2>, rows * p.chunks, 128, st, p);
    else if (p.D <= 128)
      e = launch_pdl(pa_score_mma_kernel<4>, rows * p.chunks, 128, st, p);
    else
      e = launch_pdl(pa_score_mma_kernel<8>, rows * p.chunks, 128, st, p);
    if (e != cudaSuccess) return e;
  }
  // enough threads that each holds few keys, few enough that a barrier is short
  if (p.max_blocks <= 1024)
    return launch_pdl(pa_select_kernel<T, 128, 8>, rows, 128, st, p);
  return launch_pdl(pa_select_kernel<T, 512, 16>, rows, 512, st, p);
}

}  // namespace

cudaError_t launch_bounds(const BoundsParams& p, cudaStream_t st) {
  const long long grid = (long long)p.B * p.pages_per_seq;
  if (p.kind == kBoundsQ4) return launch_pdl(pa_bounds_q4_kernel, grid, 128, st, p);
  if (p.kind == kBoundsF32) return launch_pdl(pa_bounds_kernel<float>, grid, 128, st, p);
  return launch_pdl(pa_bounds_kernel<__half>, grid, 128, st, p);
}

cudaError_t launch_select(const SelectParams& p, int dtype_size, cudaStream_t st) {
  return dtype_size == 4 ? launch_select_t<float>(p, st) : launch_select_t<__half>(p, st);
}

}  // namespace xpa
