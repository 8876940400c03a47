// pa_sparse.cu — page bounds, and the selection of the pages that sparse
// decode attention reads.
//
// A page's bounds are, per KV head and channel, the lowest and the highest of
// its keys. For a query head q the page's score is
//   sum_d max(q_d lo_d, q_d hi_d) = sum_d (q_d^+ hi_d + q_d^- lo_d),
// no less than any q . k of the page (4-bit keys: of the keys rounded to fp16, as
// their bounds are); the score of a KV head is the largest over its query heads. The best pages are kept, in the exact order of the
// scores, ties to the earlier page.
#include <algorithm>
#include <cfloat>
#include <climits>
#include <utility>

#include "pa_host.h"
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
// once per CTA took 8 prompts of 2-32K tokens (404 MB) from 117 to 69 us, 0.9 of
// the copy rate.
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

// fp16 with 16-byte rows: 16 pages x 8 heads per warp step on mma.sync, the
// bounds [lo | hi] of a page as one row of 2 D values against [q^- | q^+], and
// their magnitudes against each other for the error bound. The work per page
// is 4 D bytes against 8 D flop per head, far below the tensor ridge: bound by
// HBM, so each warp copies whole rows (4 D contiguous bytes) into a ring of two
// tiles of its own with cp.async and scores the tile before meanwhile. Rows are
// padded by 16 bytes to an odd number of 16-byte units, so ldmatrix reads eight
// of them without a bank conflict. CTA = (sequence, W KV heads, chunk of pages):
// its warps read the same pages side by side (all heads of a page are one run
// of memory), each with its own KV head, and with a second set of tiles where
// there are few heads.
// S: steps of 16 values, 2 D <= 16 S; FULL: 2 D = 16 S.
// W = kScoreWarps: three CTAs per SM at D = 128, whose starts overlap.
inline size_t score_smem_bytes(int D) {
  return (size_t)kScoreWarps * 2 * kScoreTile * (4 * D + 16);
}

template <int S, bool FULL>
__global__ void __launch_bounds__(kScoreWarps * 32) pa_score_mma_kernel(const SelectParams p) {
  extern __shared__ __align__(128) uint8_t smem[];
  pdl_wait_primary();
  pdl_launch_dependents();  // the selection may be scheduled; it waits for this grid
  const int D = FULL ? 8 * S : p.D;
  constexpr int NW = kScoreWarps;
  const int groups = (p.Hkv + NW - 1) / NW;
  const int chunk = blockIdx.x % p.chunks, col = blockIdx.x / p.chunks;
  const int b = col / groups, first_head = (col - b * groups) * NW;
  const int L = clamped_len(p.seq_lens, b, p.max_blocks, p.block_size, nullptr, false);
  const int npages = (int)(((long long)L + p.block_size - 1) / p.block_size);
  const int page_end = min(npages, (chunk + 1) * p.chunk_pages);
  if (npages <= p.keep || chunk * p.chunk_pages >= npages) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int heads = min(p.Hkv - first_head, NW), sets = NW / heads;
  const int set = warp / heads, h = first_head + warp - set * heads;
  if (set >= sets) return;
  const int row = b * p.Hkv + h;
  const int row_bytes = 4 * D + 16, stage_bytes = kScoreTile * row_bytes;
  const uint32_t ring = smem_u32(smem) + warp * 2 * stage_bytes;
  const uint8_t* bounds = static_cast<const uint8_t*>(p.bounds) + (long long)h * 4 * D;
  const unsigned page_bytes = (unsigned)p.Hkv * 4u * (unsigned)D;
  unsigned* keys = p.keys + (long long)row * p.max_blocks;
  float* magnitude = p.magnitude + (long long)row * p.tiles;
  // lanes 0..15: the entries of the tile at `at`, -1 past the end
  auto entries = [&](int at) {
    return lane < kScoreTile && at + lane < page_end ? table_entry(p, b, at + lane) : -1;
  };
  // Copies a tile's rows; a page that is not there reads the first page's row
  // and is dropped at the end.
  auto issue = [&](int e, uint32_t st) {
    if constexpr (FULL && S == 8) {  // 256-byte rows, two at a time
      const uint8_t* src = bounds + (lane & 15) * 16;
      const uint32_t dst = st + (lane >> 4) * row_bytes + (lane & 15) * 16;
#pragma unroll
      for (int r = 0; r < kScoreTile; r += 2) {
        const int er = max(__shfl_sync(0xffffffffu, e, r + (lane >> 4)), 0);
        cp_async16(dst + r * row_bytes, src + (unsigned long long)(unsigned)er * page_bytes);
      }
    } else if constexpr (FULL) {  // rows of one or more times 512 bytes
      const uint8_t* src = bounds + lane * 16;
      const uint32_t dst = st + lane * 16;
#pragma unroll
      for (int r = 0; r < kScoreTile; ++r) {
        const int er = max(__shfl_sync(0xffffffffu, e, r), 0);
        const uint8_t* from = src + (unsigned long long)(unsigned)er * page_bytes;
#pragma unroll
        for (int c = 0; c < S / 16; ++c)
          cp_async16(dst + r * row_bytes + c * 512, from + c * 512);
      }
    } else {
      const int cpr = D / 4;  // 16-byte chunks per row, fewer than 64
      int r = lane >= cpr ? lane / cpr : 0, c = lane - r * cpr;
#pragma unroll 4
      for (int i = 0; i < kScoreTile * cpr; i += 32) {
        const int er = max(__shfl_sync(0xffffffffu, e, r), 0);
        if (r < kScoreTile)
          cp_async16(st + r * row_bytes + c * 16,
                     bounds + (unsigned long long)(unsigned)er * page_bytes + c * 16);
        for (c += 32; c >= cpr; c -= cpr) ++r;
      }
    }
  };
  // this lane's row and half in ldmatrix.x4: rows 0-7, 8-15, then the next 8 values
  const uint32_t frag = (lane & 15) * row_bytes + (lane >> 4) * 16;
  const int begin = chunk * p.chunk_pages + set * kScoreTile, stride = sets * kScoreTile;
#pragma unroll 1
  for (int h0 = 0; h0 < p.GS; h0 += 8) {
    int e = entries(begin);
    if (begin < page_end) issue(e, ring);
    cp_async_commit();
    // head h0 + g: values 16 s + 2 t, + 1, + 8, + 9 of [q^- | q^+], finite,
    // times the sign of the score scale
    uint32_t qf[S][2];
    {
      const __half* q = static_cast<const __half*>(p.q) +
                        ((long long)b * p.Hq + (long long)h * p.GS + h0 + g) * D + 2 * t;
      const __half2 zero = __float2half2_rn(0.f), top = __float2half2_rn(65504.f);
      const __half2 sg = __float2half2_rn(p.sign);
      const bool head = h0 + g < p.GS;
#pragma unroll
      for (int s = 0; s < S; ++s)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int at = 16 * s + 8 * k;
          const bool upper = at >= D;
          __half2 x = zero;
          if (head && (FULL || at < 2 * D))
            x = __ldg(reinterpret_cast<const __half2*>(q + at - (upper ? D : 0)));
          x = __hmul2(x, sg);
          // max and min drop a NaN operand, so a NaN becomes 0 in both halves
          x = upper ? __hmin2(__hmax2(x, zero), top) : __hmax2(__hmin2(x, zero), __hneg2(top));
          qf[s][k] = *reinterpret_cast<const uint32_t*>(&x);
        }
    }
    uint32_t st = 0;
#pragma unroll 1
    for (int p0 = begin; p0 < page_end; p0 += stride) {
      const int next = entries(p0 + stride);
      if (p0 + stride < page_end) issue(next, ring + (st ^ stage_bytes));
      cp_async_commit();
      cp_async_wait<1>();
      __syncwarp();
      float x[2][4] = {}, y[2][4] = {};  // sums and sums of magnitudes, two chains each
#pragma unroll
      for (int s = 0; s < S; ++s) {
        if (!FULL && 8 * s >= D) break;
        uint32_t a[4], m[4];
        ldsm_x4(ring + st + frag + s * 32, a[0], a[1], a[2], a[3]);
#pragma unroll
        for (int k = 0; k < 4; ++k) m[k] = a[k] & 0x7fff7fffu;
        mma_f16_16816(x[s & 1], a[0], a[1], a[2], a[3], qf[s][0], qf[s][1]);
        mma_f16_16816(y[s & 1], m[0], m[1], m[2], m[3], qf[s][0] & 0x7fff7fffu,
                      qf[s][1] & 0x7fff7fffu);
      }
      __syncwarp();  // the stage may be filled again
      st ^= stage_bytes;
      // heads h0 + 2 t, + 1 of pages g and g + 8: the largest over the group.
      // Rows of pages that are not there hold another page's bounds, and those
      // widen no error bound.
      const int e0 = __shfl_sync(0xffffffffu, e, g), e1 = __shfl_sync(0xffffffffu, e, g + 8);
      float most = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        x[0][k] += x[1][k];
        most = fmaxf(most, (k < 2 ? e0 : e1) < 0 ? 0.f : y[0][k] + y[1][k]);
      }
      const bool c0 = h0 + 2 * t < p.GS, c1 = h0 + 2 * t + 1 < p.GS;
      float s0 = fmaxf(c0 ? x[0][0] : -INFINITY, c1 ? x[0][1] : -INFINITY);
      float s1 = fmaxf(c0 ? x[0][2] : -INFINITY, c1 ? x[0][3] : -INFINITY);
      s0 = fmaxf(s0, __shfl_xor_sync(0xffffffffu, s0, 1));
      s1 = fmaxf(s1, __shfl_xor_sync(0xffffffffu, s1, 1));
      s0 = fmaxf(s0, __shfl_xor_sync(0xffffffffu, s0, 2));
      s1 = fmaxf(s1, __shfl_xor_sync(0xffffffffu, s1, 2));
      most = warp_max(most);
      e = next;
      // lane 0 of a quad stores page g, lane 1 page g + 8
      if (t < 2 && p0 + g + 8 * t < page_end) {
        unsigned k = (t ? e1 : e0) < 0 ? 0u : key_of(t ? s1 : s0);
        unsigned* dst = keys + p0 + g + 8 * t;
        if (h0 > 0) k = max(k, *dst);
        *dst = k;
      }
      if (lane == 0) {
        float* dst = magnitude + p0 / kScoreTile;
        *dst = h0 > 0 ? fmaxf(*dst, most) : most;
      }
    }
    cp_async_wait<0>();
    __syncwarp();
  }
}

// Every other type and size: one warp per page, lanes across the channels.
template <typename T>
__global__ void __launch_bounds__(128) pa_score_kernel(const SelectParams p) {
  __shared__ float s_max[4];
  constexpr float top = sizeof(T) == 2 ? 65504.f : FLT_MAX;
  pdl_wait_primary();
  pdl_launch_dependents();
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
        float s = 0.f, m = 0.f;
#pragma unroll 4
        for (int d = lane; d < p.D; d += 32) {
          const float qd = p.sign * tame(to_float<T>(q[(long long)x * p.D + d]), top);
          const float l = to_float<T>(lo[d]), u = to_float<T>(lo[p.D + d]);
          s = fmaf(fmaxf(qd, 0.f), u, s);
          s = fmaf(fminf(qd, 0.f), l, s);
          m = fmaf(fabsf(qd), qd > 0.f ? fabsf(u) : fabsf(l), m);
        }
        best = fmaxf(best, warp_sum(s));
        big = fmaxf(big, warp_sum(m));
      }
      key = key_of(best);
    }
    if (lane == 0) p.keys[(long long)row * p.max_blocks + at] = key;
  }
  if (lane == 0) s_max[warp] = big;
  __syncthreads();
  if (threadIdx.x == 0)
    p.magnitude[(long long)row * p.tiles + chunk] =
        fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
}

// ════════════════════════════════════════════════════════════════════════
// Selection, second kernel: one CTA per row.
//   1. A histogram of the fp32 scores' ordered keys over their range finds the
//      bin that holds the r-th largest.
//   2. A score is off by at most E, so scores above the bin's end + 2 E are in
//      and those below its start - 2 E are out. When more lie between than
//      places are left, those few are scored again in 64 bits (products of the
//      operands are exact there) and the best taken, the earlier page on a tie.
//   3. The kept pages go out in order, as per-head page ids.
// E: a tensor-core step of 16 products and its accumulator is taken to be off
// by at most 2^-18 of the sum of their magnitudes (17 terms cut at 2^-23 of the
// largest), a scalar sum by less; over the at most 16 steps of a chain that is
// 2^-14 of the sum of a score's terms' magnitudes, whose largest of the row the
// score kernel has left.
// A row is read once and the code runs through once: what counts is the latency
// of its barriers, of its few dependent reads and of fetching the code, so loops
// stay loops and reads are issued together (6144 pages a row, 512 threads: 16.6
// us; rows of 64-512 pages, 128 threads: 11.5 us).
// ════════════════════════════════════════════════════════════════════════
constexpr int kBins = 2048;
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

// The score of page e for KV head h of sequence b in 64 bits, over a warp (its
// lanes all get it). K32: 32 K32 >= D; all loads of four heads before their use.
template <typename T, int K32>
__device__ __forceinline__ double score64(const SelectParams& p, int b, int h, int e, int lane) {
  constexpr float top = sizeof(T) == 2 ? 65504.f : FLT_MAX;
  const T* q = static_cast<const T*>(p.q) + ((long long)b * p.Hq + (long long)h * p.GS) * p.D;
  const T* lo = static_cast<const T*>(p.bounds) + ((long long)e * p.Hkv + h) * 2 * p.D;
  T l[K32], u[K32];
#pragma unroll
  for (int k = 0; k < K32; ++k) {
    const int d = lane + 32 * k;
    l[k] = d < p.D ? lo[d] : from_float<T>(0.f);
    u[k] = d < p.D ? lo[p.D + d] : from_float<T>(0.f);
  }
  double best = -INFINITY;
#pragma unroll 1
  for (int x0 = 0; x0 < p.GS; x0 += 4) {  // four heads' sums side by side
    T qx[K32][4];
#pragma unroll
    for (int k = 0; k < K32; ++k)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int d = lane + 32 * k;
        qx[k][x] = d < p.D ? q[(long long)min(x0 + x, p.GS - 1) * p.D + d] : from_float<T>(0.f);
      }
    double s[4] = {};
#pragma unroll
    for (int k = 0; k < K32; ++k)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float qd = p.sign * tame(to_float<T>(qx[k][x]), top);
        s[x] = fma((double)qd, (double)to_float<T>(qd > 0.f ? u[k] : l[k]), s[x]);
      }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
      for (int x = 0; x < 4; ++x) s[x] += __shfl_xor_sync(0xffffffffu, s[x], o);
    best = fmax(best, fmax(fmax(s[0], s[1]), fmax(s[2], s[3])));
  }
  return best;
}

// The row's keys stay in shared memory up to kSmemKeys pages (`smem_keys`),
// longer rows are read again from the workspace.
constexpr int kSmemKeys = 32768;

template <typename T, int NT>
__global__ void __launch_bounds__(NT, 512 / NT) pa_select_kernel(const SelectParams p, int smem_keys) {
  constexpr int NWARP = NT / 32;
  extern __shared__ unsigned s_keys[];
  __shared__ BlockCount<NT> s_cnt;
  __shared__ float s_red[NWARP];
  __shared__ unsigned s_low[NWARP], s_high[NWARP];
  __shared__ int s_near, s_bin;
  __shared__ unsigned s_near_page[kNearCap];
  __shared__ unsigned long long s_near_key[kNearCap];
  __shared__ int s_count[NWARP], s_total[NWARP];
  __shared__ __align__(16) int s_bins[kBins];
  pdl_wait_primary();
  // No early trigger here: the merge behind the attention reads sel_lens
  // before it waits for anything, so nothing may start until they are written.
  const int row = blockIdx.x;
  const int b = row / p.Hkv, h = row - b * p.Hkv;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int L = clamped_len(p.seq_lens, b, p.max_blocks, p.block_size, p.status,
                            h == 0 && tid == 0);
  const int n = (int)(((long long)L + p.block_size - 1) / p.block_size);
  const bool scored = n > p.keep;
  // keys of the row's pages, 0: the table names no page there
  unsigned* K = p.keys + (long long)row * p.max_blocks;
  const int first = p.sink, last = n - p.recent;  // [first, last): pages that compete
  unsigned take = 1u;  // a competing page with a key of at least this is kept
  if (scored) {
    const int r = p.keep - p.sink - p.recent;
    int turn = 0;
    int mine = 0;
    unsigned kmin = 0xffffffffu, kmax = 0u;
    // the largest sum of magnitudes of the row
    float most = 0.f;
    const int tiles = (n + p.tile_pages - 1) / p.tile_pages;
    for (int i = tid; i < tiles; i += NT)
      most = fmaxf(most, p.magnitude[(long long)row * p.tiles + i]);
#pragma unroll 1
    for (int at0 = tid; at0 < n; at0 += 8 * NT) {
      unsigned k[8];  // all eight on the way together, the row's end included
#pragma unroll
      for (int j = 0; j < 8; ++j) k[j] = at0 + j * NT < n ? K[at0 + j * NT] : 0u;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int at = at0 + j * NT;
        if (at < n && n <= smem_keys) s_keys[at] = k[j];
        if (k[j] && at >= first && at < last) {
          ++mine;
          kmin = min(kmin, k[j]);
          kmax = max(kmax, k[j]);
        }
      }
    }
    if (n <= smem_keys) K = s_keys;  // each thread goes on with the keys it copied
    if (tid == 0) s_near = 0;
    for (int i = tid; i < kBins; i += NT) s_bins[i] = 0;
    mine = __reduce_add_sync(0xffffffffu, mine);
    kmin = __reduce_min_sync(0xffffffffu, kmin);
    kmax = __reduce_max_sync(0xffffffffu, kmax);
    most = warp_max(most);
    if (lane == 0) {
      s_count[warp] = mine;
      s_low[warp] = kmin;
      s_high[warp] = kmax;
      s_red[warp] = most;
    }
    __syncthreads();
    const int eligible = __reduce_add_sync(0xffffffffu, lane < NWARP ? s_count[lane] : 0);
    if (r <= 0) {
      take = 0xffffffffu;  // no competing page fits; no key is this large
    } else if (eligible > r) {
      kmin = __reduce_min_sync(0xffffffffu, lane < NWARP ? s_low[lane] : 0xffffffffu);
      kmax = __reduce_max_sync(0xffffffffu, lane < NWARP ? s_high[lane] : 0u);
      most = warp_max(lane < NWARP ? s_red[lane] : 0.f);
      // histogram of the keys over [kmin, kmax], each bin 2^shift keys wide
      const int shift = max(0, 32 - __clz(kmax - kmin) - 11);
#pragma unroll 4
      for (int at = tid; at < last; at += NT) {
        const unsigned k = at >= first ? K[at] : 0u;
        if (k) atomicAdd(&s_bins[(k - kmin) >> shift], 1);
      }
      __syncthreads();
      // the bin of the r-th largest: a thread's bins, from the top, then the scan
      constexpr int BPT = kBins / NT;
      int in_bins = 0;
#pragma unroll
      for (int i = 0; i < BPT / 4; ++i) {
        const int4 v = reinterpret_cast<const int4*>(s_bins)[(kBins - (tid + 1) * BPT) / 4 + i];
        in_bins += v.x + v.y + v.z + v.w;
      }
      int upto = in_bins;  // keys in this warp's bins down to this thread's
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
      }
      if (lane == 31) s_count[warp] = upto;
      __syncthreads();
      // keys in the bins of the warps before, and before this thread's
      int over = __reduce_add_sync(0xffffffffu, lane < warp ? s_count[lane] : 0) + upto - in_bins;
      if (over < r && over + in_bins >= r) {
#pragma unroll 1
        for (int i = 0; over < r; ++i) {
          s_bin = kBins - 1 - (tid * BPT + i);
          over += s_bins[s_bin];
        }
      }
      __syncthreads();
      const unsigned start = kmin + ((unsigned)s_bin << shift);
      const unsigned end = min(kmax, start + ((1u << shift) - 1u));
      const float E = most * 0x1p-14f + 0x1p-118f;
      const float flo = score_of(start), fhi = score_of(end);
      unsigned near_lo = 1u, near_hi = 0xfffffffeu;
      if (fabsf(E) < 0x1p126f && fabsf(flo) < 0x1p126f && fabsf(fhi) < 0x1p126f) {
        near_lo = max(1u, key_of(flo - 2.001f * E));
        near_hi = key_of(fhi + 2.001f * E);
      }
      // pages above, and the list of the near ones: its first kNearCap entries
      // in shared memory too
      unsigned* far_page = p.near_page + (long long)row * p.max_blocks;
      int above = 0;
#pragma unroll 4
      for (int at = tid; at < last; at += NT) {
        const unsigned k = at >= first ? K[at] : 0u;
        above += k > near_hi;
        if (k >= near_lo && k <= near_hi) {
          const int to = atomicAdd(&s_near, 1);
          far_page[to] = (unsigned)at;
          if (to < kNearCap) s_near_page[to] = (unsigned)at;
        }
      }
      const int need = r - block_sum<NT>(s_cnt, above, turn);
      const int near = s_near;
      take = near_lo;
      if (near > need) {
        const bool few = near <= kNearCap;
        const unsigned* lp = few ? s_near_page : far_page;
        unsigned long long* lk = few ? s_near_key : p.near_key + (long long)row * p.max_blocks;
#pragma unroll 1
        for (int i = warp; i < near; i += NWARP) {
          const int e = __ldg(p.block_tables + (long long)b * p.max_blocks + lp[i]);
          const double best = p.D <= 128 ? score64<T, 4>(p, b, h, e, lane)
                                         : score64<T, 8>(p, b, h, e, lane);
          if (lane == 0) lk[i] = key_of(best);
        }
        __syncthreads();
        // kept near pages get the key near_hi, the others 0
        if (few) {
          for (int i = tid; i < near; i += NT) {
            const unsigned long long k = lk[i];
            const unsigned at = lp[i];
            int rank = 0;
#pragma unroll 4
            for (int o = 0; o < near; ++o) rank += lk[o] > k || (lk[o] == k && lp[o] < at);
            K[at] = rank < need ? near_hi : 0u;
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
          for (int i = tid; i < near; i += NT)
            K[lp[i]] = lk[i] > T64 || (lk[i] == T64 && lp[i] <= cut) ? near_hi : 0u;
        }
      }
    }
    __syncthreads();  // every key is in its final place
  }
  // ── the kept pages, in order: a warp's run of pages, then the scan ──────
  const int run = ((n + NT - 1) / NT) * 32, begin = min(n, warp * run), stop = min(n, begin + run);
  auto kept = [&](int at) {
    if (at >= stop) return false;
    if (!scored) return table_entry(p, b, at) >= 0;
    const unsigned k = K[at];
    return at < first || at >= last ? k != 0u : k >= take;
  };
  // lane l: which of the pages at + 32 l .. + 31 are kept
  auto mask_at = [&](int at) {
    unsigned own = 0u;
    const int words = min(32, (stop - at + 31) >> 5);
#pragma unroll 4
    for (int j = 0; j < words; ++j) {
      const unsigned m = __ballot_sync(0xffffffffu, kept(at + 32 * j + lane));
      if (lane == j) own = m;
    }
    return own;
  };
  unsigned own = 0u;
  int count = 0;
#pragma unroll 1
  for (int at = begin; at < stop; at += 1024) {
    own = mask_at(at);
    count += __reduce_add_sync(0xffffffffu, __popc(own));
  }
  if (lane == 0) s_total[warp] = count;
  __syncthreads();
  int to = __reduce_add_sync(0xffffffffu, lane < warp ? s_total[lane] : 0);
  const int done = __reduce_add_sync(0xffffffffu, lane < NWARP ? s_total[lane] : 0);
  int* tab = p.sel_tables + (long long)row * p.copies * p.width * p.sub;
  int* order = p.order ? p.order + (long long)row * p.width : tab;
  int* pages = p.sel_pages ? p.sel_pages + (long long)row * p.keep : nullptr;
#pragma unroll 1
  for (int at = begin; at < stop; at += 1024) {
    unsigned m = run <= 1024 ? own : mask_at(at);
    int upto = __popc(m);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += y;
    }
    int mine = to + upto - __popc(m);
    to += __shfl_sync(0xffffffffu, upto, 31);
    for (; m; m &= m - 1u) order[mine++] = at + 32 * lane + __ffs(m) - 1;
  }
  __syncthreads();
  // page indices -> per-head page ids, all table reads at once
  bool tail = false;  // the sequence's last page is kept
  for (int i = tid; i < done; i += NT) {
    const int at = order[i];
    const int e = __ldg(p.block_tables + (long long)b * p.max_blocks + at);
    if (pages) pages[i] = at;
    tail |= at == n - 1;
    const int id = (int)(((long long)e * p.head_pages + h) * p.sub_ids);
    for (int c = 0; c < p.copies; ++c)
      for (int k = 0; k < p.sub; ++k)
        tab[((long long)c * p.width + i) * p.sub + k] = id + k;
  }
  for (int i = done + tid; i < p.width; i += NT)
    for (int c = 0; c < p.copies; ++c)
      for (int k = 0; k < p.sub; ++k) tab[((long long)c * p.width + i) * p.sub + k] = -1;
  if (pages)
    for (int i = done + tid; i < p.keep; i += NT) pages[i] = -1;
  tail = __syncthreads_or(tail);
  if (tid < p.copies)
    p.sel_lens[(long long)row * p.copies + tid] =
        done * p.block_size - (tail ? (int)((long long)n * p.block_size - L) : 0);
}

template <typename... KArgs, typename... Args>
cudaError_t launch_pdl(void (*kern)(KArgs...), long long grid, unsigned block, size_t smem,
                       cudaStream_t st, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...);
}

template <int S, bool FULL>
cudaError_t launch_score_mma(const SelectParams& p, cudaStream_t st) {
  constexpr int NW = kScoreWarps;
  const long long ctas = (long long)p.B * ((p.Hkv + NW - 1) / NW) * p.chunks;
  auto kern = pa_score_mma_kernel<S, FULL>;
  static std::atomic<unsigned long long> done{0};
  const cudaError_t e = host::smem_limit(kern, score_smem_bytes(8 * S), false, done);
  if (e != cudaSuccess) return e;
  return launch_pdl(kern, ctas, NW * 32, score_smem_bytes(p.D), st, p);
}

template <typename T, int NT>
cudaError_t launch_select_nt(const SelectParams& p, long long rows, int keys, cudaStream_t st) {
  auto kern = pa_select_kernel<T, NT>;
  static std::atomic<unsigned long long> done{0};
  const cudaError_t e = host::smem_limit(kern, kSmemKeys * sizeof(unsigned), false, done);
  if (e != cudaSuccess) return e;
  return launch_pdl(kern, rows, NT, keys * sizeof(unsigned), st, p, keys);
}

template <typename T>
cudaError_t launch_select_t(const SelectParams& p, cudaStream_t st) {
  const long long rows = (long long)p.B * p.Hkv;
  // no sequence can hold more pages than are kept: nothing is scored
  if (p.max_blocks > p.keep) {
    cudaError_t e;
    if (!p.vec)
      e = launch_pdl(pa_score_kernel<T>, rows * p.chunks, 128, 0, st, p);
    else if (p.D == 64)
      e = launch_score_mma<8, true>(p, st);
    else if (p.D == 128)
      e = launch_score_mma<16, true>(p, st);
    else if (p.D == 256)
      e = launch_score_mma<32, true>(p, st);
    else if (p.D < 128)
      e = launch_score_mma<16, false>(p, st);
    else
      e = launch_score_mma<32, false>(p, st);
    if (e != cudaSuccess) return e;
  }
  const int keys = p.max_blocks > p.keep ? std::min(p.max_blocks, kSmemKeys) : 0;
  // few threads for short rows, whose barriers are then shorter
  if (p.max_blocks <= 1024) return launch_select_nt<T, 128>(p, rows, keys, st);
  return launch_select_nt<T, 512>(p, rows, keys, st);
}

}  // namespace

cudaError_t launch_bounds(const BoundsParams& p, cudaStream_t st) {
  const long long grid = (long long)p.B * p.pages_per_seq;
  if (p.kind == kBoundsQ4) return launch_pdl(pa_bounds_q4_kernel, grid, 128, 0, st, p);
  if (p.kind == kBoundsF32) return launch_pdl(pa_bounds_kernel<float>, grid, 128, 0, st, p);
  return launch_pdl(pa_bounds_kernel<__half>, grid, 128, 0, st, p);
}

cudaError_t launch_select(const SelectParams& p, int dtype_size, cudaStream_t st) {
  return dtype_size == 4 ? launch_select_t<float>(p, st) : launch_select_t<__half>(p, st);
}

}  // namespace xpa
