// pa_q4.cu — 4-bit KV cache: rows written and read back by slot, and paged
// decode attention over it. Format and tile layout: pa_q4.cuh.
#include <algorithm>
#include <utility>

#include "pa_q4.cuh"
#include "pa_q4.h"

namespace xpa {

namespace {

// ════════════════════════════════════════════════════════════════════════
// Rows <-> tiles. One warp per (token, KV head); a lane holds 8 channels of
// the K row (lanes below D / 8) or of the V row (the lanes after), so at
// D = 128 a warp is full and a group's maximum is one shuffle away.
// ════════════════════════════════════════════════════════════════════════
struct RowAt {
  int t, h;           // token, KV head
  long long tile;     // byte offset of the 16-token tile in its pool
  int tok;            // token's row in the tile
};

__device__ __forceinline__ bool q4_row_at(const Q4RowsParams& a, long long w, RowAt& r) {
  r.t = (int)(w / a.Hkv);
  r.h = (int)(w - (long long)r.t * a.Hkv);
  const long long slot = a.slots[r.t];
  if (slot < 0 || slot >= a.num_slots) return false;
  const long long page = slot / a.block_size;
  const int s = (int)(slot - page * a.block_size);
  r.tile = page * a.kv_block_stride + (long long)r.h * a.kv_head_stride +
           (long long)(s >> 4) * (9 * a.D);
  r.tok = s & 15;
  return true;
}

__global__ void __launch_bounds__(128) pa_q4_write_kernel(const Q4RowsParams a) {
  const long long w = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (w >= (long long)a.num_tokens * a.Hkv) return;
  RowAt r;
  if (!q4_row_at(a, w, r)) return;
  const int NV = a.D / 8;  // 8-channel pieces of a row, an even number
  const long long src = (long long)r.t * a.token_stride + (long long)r.h * a.D;
  for (int i0 = 0; i0 < 2 * NV; i0 += 32) {
    const int i = i0 + lane;
    const bool act = i < 2 * NV, is_v = i >= NV;
    const int v = is_v ? i - NV : i;
    const __half* row = static_cast<const __half*>(is_v ? a.value : a.key) + src + v * 8;
    const float ps = is_v ? a.v_scale : a.k_scale;
    float x[8];
    float amax = 0.f;
    if (act) {
      if (a.vec16) {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(row));
        const uint32_t q[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 f = unpack_half2(q[k]);
          x[2 * k] = f.x;
          x[2 * k + 1] = f.y;
        }
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = __half2float(row[k]);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        x[k] = isnan(x[k]) ? 0.f : __fdiv_rn(x[k], ps);
        amax = fmaxf(amax, fabsf(x[k]));
      }
    }
    // a 16-channel group is two neighbouring lanes (pieces 2 g, 2 g + 1)
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    if (!act) continue;
    const uint32_t sb = q4_scale(amax);
    const float s = fp8_to_float<kKvE4M3>((uint8_t)sb);
    uint32_t code = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float p = s > 0.f ? __fdiv_rn(x[2 * k], s) : 0.f;
      const float q = s > 0.f ? __fdiv_rn(x[2 * k + 1], s) : 0.f;
      code |= q4_pair(p, q) << (8 * k);
    }
    uint8_t* tile = static_cast<uint8_t*>(is_v ? a.value_cache : a.key_cache) + r.tile;
    if (is_v) {
      *reinterpret_cast<uint32_t*>(tile + q4_v_off(a.D, r.tok, v)) = code;
      if ((v & 1) == 0) tile[q4_v_scale_off(a.D, r.tok, v >> 1)] = (uint8_t)sb;
    } else {
      uint8_t* dst = tile + q4_k_off(a.D, r.tok, v);
      *reinterpret_cast<uint16_t*>(dst) = (uint16_t)code;
      *reinterpret_cast<uint16_t*>(dst + a.D / 8) = (uint16_t)(code >> 16);
      if ((v & 1) == 0) tile[q4_k_scale_off(a.D, r.tok, v >> 1)] = (uint8_t)sb;
    }
  }
}

// c * s * ps, rounded to fp16 once and kept finite: a group's largest element
// may have been rounded up past the fp16 range.
__device__ __forceinline__ float q4_value(float cs, float ps) {
  return fminf(fmaxf(cs * ps, -65504.f), 65504.f);
}

__global__ void __launch_bounds__(128) pa_q4_read_kernel(const Q4RowsParams a) {
  const long long w = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (w >= (long long)a.num_tokens * a.Hkv) return;
  RowAt r;
  const bool live = q4_row_at(a, w, r);
  const int NV = a.D / 8;
  const long long dst0 = (long long)r.t * a.token_stride + (long long)r.h * a.D;
  for (int i = lane; i < 2 * NV; i += 32) {
    const bool is_v = i >= NV;
    const int v = is_v ? i - NV : i;
    uint4 u = make_uint4(0u, 0u, 0u, 0u);
    if (live) {
      const uint8_t* tile = static_cast<const uint8_t*>(is_v ? a.value_cache : a.key_cache) + r.tile;
      uint32_t code, sb;
      if (is_v) {
        code = *reinterpret_cast<const uint32_t*>(tile + q4_v_off(a.D, r.tok, v));
        sb = tile[q4_v_scale_off(a.D, r.tok, v >> 1)];
      } else {
        const uint8_t* at = tile + q4_k_off(a.D, r.tok, v);
        code = *reinterpret_cast<const uint16_t*>(at) |
               ((uint32_t) * reinterpret_cast<const uint16_t*>(at + a.D / 8) << 16);
        sb = tile[q4_k_scale_off(a.D, r.tok, v >> 1)];
      }
      const float s = fp8_to_float<kKvE4M3>((uint8_t)sb);
      const float ps = is_v ? a.v_scale : a.k_scale;
      uint32_t h[4], o[4];
      q4x8_to_h2(code, h);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 f = unpack_half2(h[k]);
        o[k] = pack_half2(q4_value(f.x * s, ps), q4_value(f.y * s, ps));
      }
      u = make_uint4(o[0], o[1], o[2], o[3]);
    }
    __half* dst = static_cast<__half*>(is_v ? a.value : a.key) + dst0 + v * 8;
    if (a.vec16) {
      *reinterpret_cast<uint4*>(dst) = u;
    } else {
      const uint32_t o[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int k = 0; k < 8; ++k)
        dst[k] = __ushort_as_half((unsigned short)(o[k >> 1] >> (16 * (k & 1))));
    }
  }
}

// ════════════════════════════════════════════════════════════════════════
// Decode attention. CTA = (item, chunk of 8 NT query heads of its group);
// its NW warps take the item's 16-token tiles in turn, each through a ring
// of its own that its lanes fill with cp.async and only they read, so the
// loop has no barrier beyond the warp.
//
// Per tile, with mma.sync m16n8k16 (fp16 in, fp32 sums):
//   S^T(16 tokens x 8 heads)  = K . Q^T      K as A, D / 16 steps
//   O^T(D x 8 heads)         += V^T . P^T    V as A, D / 16 row tiles, P = hi + lo
// Token order: row r of S^T (and k index r of P^T) is token sigma(r) with
// sigma(2 t) = 4 t, sigma(2 t + 1) = 4 t + 1, sigma(8 + 2 t) = 4 t + 2,
// sigma(9 + 2 t) = 4 t + 3, so a lane's four V tokens are 4 t .. 4 t + 3 and
// their scales one word. Channel order: K step j's k index 2 t, 2 t + 1,
// 2 t + 8, 2 t + 9 are channels 16 j + 4 t .. + 3 (Q's fragments follow); V
// row tile 4 w + i holds channels 8 (g W + w) + 2 i (row g) and + 1 (row g + 8).
//
// Softmax: scores live in the exp2 domain. The reference point m of a head
// moves only when a score exceeds it by more than 8, so most tiles need one
// vote and no shuffles; p <= 2^15 with the shift of 7 that keeps small
// weights above fp16's subnormals. P = hi + lo in fp16 keeps 22 bits.
// ════════════════════════════════════════════════════════════════════════
constexpr float kRaise = 8.f;  // log2 units a score may exceed m by
constexpr float kShift = 7.f;  // p = 2^(x - m + kShift) <= 2^15

template <int W, int NT, bool EXACT, int NW, int STAGES>
struct Q4Cfg {
  static constexpr int kDMax = 64 * W;
  static constexpr int kHeads = 8 * NT;
  static constexpr int kStageBytes = 18 * kDMax;  // one K and one V tile
  static constexpr int kRow = kDMax + 4;          // merge rows, floats
  static constexpr size_t kMergeBytes =
      (size_t)NW * kHeads * kRow * sizeof(float) + (size_t)NW * kHeads * 2 * sizeof(float);
  static constexpr size_t kRingBytes = (size_t)NW * STAGES * kStageBytes;
  static constexpr size_t kSmem = kRingBytes > kMergeBytes ? kRingBytes : kMergeBytes;
};

__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t r;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(r) : "r"(a));
  return r;
}
__device__ __forceinline__ uint32_t lds16(uint32_t a) {
  uint16_t r;
  asm volatile("ld.shared.b16 %0, [%1];" : "=h"(r) : "r"(a));
  return r;
}
__device__ __forceinline__ uint32_t lds8(uint32_t a) {
  uint32_t r;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(r) : "r"(a));
  return r;
}
template <int N>
__device__ __forceinline__ void lds_words(uint32_t a, uint32_t* r) {
  if constexpr (N == 1) {
    r[0] = lds32(a);
  } else if constexpr (N == 2) {
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(a));
  } else {
    static_assert(N == 4, "1, 2 or 4 words");
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a));
  }
}

// Where a tile's pieces sit in a ring stage, and one lane's reads of them.
// EXACT (D = 64 W, W = 1, 2, 4): rows are placed and chunks swizzled so that
// every read below is conflict-free; K row r's place is its S^T row, V row
// 4 t + k's place is 4 k + t. Otherwise a tile is copied as it is.
template <int W, bool EXACT>
struct Q4Stage {
  int D;            // head size
  int lane, g, t;
  uint32_t kd[W], vd[W];  // EXACT: this lane's copy destinations in a stage

  __device__ __forceinline__ Q4Stage(int D_, int lane_) : D(D_), lane(lane_) {
    g = lane >> 2;
    t = lane & 3;
    if constexpr (EXACT) {
      constexpr int CPR = 2 * W;  // 16-byte chunks per row
#pragma unroll
      for (int k = 0; k < W; ++k) {
        const int x = lane + 32 * k, r = x / CPR, c = x % CPR;
        const int kp = 2 * (r >> 2) + (r & 1) + 8 * ((r >> 1) & 1);
        const int vp = 4 * (r & 3) + (r >> 2);
        int ck = c, cv = c;
        if (W == 4) ck = c ^ (kp & 1);
        if (W == 2) cv = c ^ (2 * ((vp >> 1) & 1));
        if (W == 4) cv = c ^ (2 * (vp & 3));
        kd[k] = (uint32_t)(kp * 32 * W + ck * 16);
        vd[k] = (uint32_t)(8 * 64 * W + vp * 32 * W + cv * 16);
      }
    }
  }

  // Issues the copies of one K and one V tile into the stage at `st`.
  __device__ __forceinline__ void copy(uint32_t st, const uint8_t* k, const uint8_t* v) const {
    if constexpr (EXACT) {
      constexpr int DD = 64 * W;
#pragma unroll
      for (int i = 0; i < W; ++i) cp_async16(st + kd[i], k + (lane + 32 * i) * 16);
#pragma unroll
      for (int i = 0; i < W; ++i) cp_async16(st + vd[i], v + (lane + 32 * i) * 16);
      // both tiles' scales: D / 16 chunks each, lanes 0.. and 16..
      const int c = lane & 15;
      if (c < 4 * W)
        cp_async16(st + 16 * DD + (lane >> 4) * DD + c * 16,
                   (lane < 16 ? k : v) + 8 * DD + c * 16);
    } else {
      const int n = 9 * D / 16;
      for (int x = lane; x < n; x += 32) {
        cp_async16(st + x * 16, k + x * 16);
        cp_async16(st + 9 * D + x * 16, v + x * 16);
      }
    }
  }

  // K codes and scales of S^T rows g (r = 0) and g + 8 (r = 1): word i of kw
  // is groups 2 i, 2 i + 1; byte j of ks is group j's scale.
  __device__ __forceinline__ void load_k(uint32_t st, uint32_t (&kw)[2][2 * W],
                                         uint32_t (&ks)[2][W]) const {
    const int tok = 4 * (g >> 1) + (g & 1);  // sigma(g); sigma(g + 8) is + 2
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      if constexpr (EXACT) {
        const uint32_t row = st + (g + 8 * r) * 32 * W;
        if constexpr (W == 1) lds_words<2>(row + t * 8, kw[r]);
        if constexpr (W == 2) lds_words<4>(row + t * 16, kw[r]);
        if constexpr (W == 4) {
          lds_words<4>(row + (((2 * t) ^ (g & 1)) << 4), kw[r]);
          lds_words<4>(row + (((2 * t + 1) ^ (g & 1)) << 4), kw[r] + 4);
        }
        lds_words<W>(st + 16 * 64 * W + (tok + 2 * r) * 4 * W, ks[r]);
      } else {
        const int NG = D / 16;
        const uint32_t row = st + (tok + 2 * r) * (D / 2) + t * (2 * NG);
        const uint32_t sc = st + 8 * D + (tok + 2 * r) * NG;
#pragma unroll
        for (int i = 0; i < 2 * W; ++i) {
          uint32_t lo = 0, hi = 0;
          if (2 * i < NG) lo = lds16(row + 4 * i);
          if (2 * i + 1 < NG) hi = lds16(row + 4 * i + 2);
          kw[r][i] = lo | (hi << 16);
        }
#pragma unroll
        for (int i = 0; i < W; ++i) {
          uint32_t s = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (4 * i + j < NG) s |= lds8(sc + 4 * i + j) << (8 * j);
          ks[r][i] = s;
        }
      }
    }
  }

  // V codes of tokens 4 t + k: word w is channels 8 (g W + w) .. + 7; vs[w]
  // holds the four tokens' scales of those channels.
  __device__ __forceinline__ void load_v(uint32_t st, uint32_t (&vw)[4][W],
                                         uint32_t (&vs)[W]) const {
    if constexpr (EXACT) {
      const uint32_t base = st + 8 * 64 * W;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t row = base + (4 * k + t) * 32 * W;
        if constexpr (W == 1) lds_words<1>(row + 4 * g, vw[k]);
        if constexpr (W == 2)
          lds_words<2>(row + (((g >> 1) ^ (t & 2)) << 4) + (g & 1) * 8, vw[k]);
        if constexpr (W == 4) lds_words<4>(row + ((g ^ (2 * t)) << 4), vw[k]);
      }
      const uint32_t sc = st + 17 * 64 * W + 4 * t;
      if constexpr (W == 1) vs[0] = lds32(sc + (g >> 1) * 16);
      if constexpr (W == 2) vs[0] = vs[1] = lds32(sc + g * 16);
      if constexpr (W == 4) {
        vs[0] = vs[1] = lds32(sc + 2 * g * 16);
        vs[2] = vs[3] = lds32(sc + (2 * g + 1) * 16);
      }
    } else {
      const uint32_t base = st + 9 * D;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const int at = g * W + w;
        const bool in = at < D / 8;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          vw[k][w] = in ? lds32(base + (4 * t + k) * (D / 2) + at * 4) : 0u;
        vs[w] = in ? lds32(base + 8 * D + (at >> 1) * 16 + 4 * t) : 0u;
      }
    }
  }
};

template <int W, int NT, bool EXACT, int NW, int STAGES, int MINB>
__global__ void __launch_bounds__(NW * 32, MINB) pa_q4_kernel(const Params p) {
  using C = Q4Cfg<W, NT, EXACT, NW, STAGES>;
  extern __shared__ __align__(128) uint8_t smem[];
  // Every CTA waits for the kernel before this one (which may be this call's
  // append); the merge may be scheduled from here on and waits for this grid.
  pdl_wait_primary();
  pdl_launch_dependents();
  const int D = EXACT ? C::kDMax : p.D;
  const int NG = D / 16;
  Item it;
  const ItemKind kind = decode_item(p, blockIdx.x, it);
  if (kind == kItemNone) return;
  const int h0 = blockIdx.y * C::kHeads;
  const int nh = min(p.GS - h0, C::kHeads);
  const long long row0 = (long long)it.b * p.Hq + (long long)it.kvh * p.GS + h0;
  if (kind == kItemZero) {
    for (int i = threadIdx.x; i < nh * D; i += NW * 32)
      store_out<__half>(p, row0 + i / D, i % D, 0.f);
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const Q4Stage<W, EXACT> sg(D, lane);

  // ── Q fragments: head g of tile nt, channels 16 j + 4 t .. + 3 ──────────
  uint32_t qf[4 * W][NT][2];
  {
    const __half* q = static_cast<const __half*>(p.q);
    const bool al = (reinterpret_cast<uintptr_t>(q) & 7u) == 0;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const bool head = nt * 8 + g < nh;
      const __half* row = q + (row0 + nt * 8 + g) * D + 4 * t;
#pragma unroll
      for (int j = 0; j < 4 * W; ++j) {
        uint2 u = make_uint2(0u, 0u);
        if (head && j < NG) {
          if (al) {
            u = __ldg(reinterpret_cast<const uint2*>(row + 16 * j));
          } else {
            const unsigned short* s = reinterpret_cast<const unsigned short*>(row + 16 * j);
            u.x = s[0] | ((uint32_t)s[1] << 16);
            u.y = s[2] | ((uint32_t)s[3] << 16);
          }
        }
        qf[j][nt][0] = u.x;
        qf[j][nt][1] = u.y;
      }
    }
  }

  // ── this warp's tiles: j = warp, warp + NW, ... of the item ─────────────
  const int spp = p.block_size >> 4;  // tiles per page
  const long long tok_end = min((long long)it.L, (long long)it.page_end * p.block_size);
  const int tok_begin = it.page_begin * p.block_size;
  const int tiles = (int)((tok_end - tok_begin + 15) >> 4);
  const int n = tiles > warp ? (tiles - warp + NW - 1) / NW : 0;
  const uint8_t* kbase = static_cast<const uint8_t*>(p.k) + (long long)it.kvh * p.kv_head_stride;
  const uint8_t* vbase = static_cast<const uint8_t*>(p.v) + (long long)it.kvh * p.kv_head_stride;
  const int* table = p.block_tables + (long long)it.b * p.max_blocks + it.page_begin;
  const uint32_t ring = smem_u32(smem) + warp * (STAGES * C::kStageBytes);

  long long ent = -1;   // lane l: pool offset of this warp's tile (i & ~31) + l, -1: none
  uint32_t live = 0;    // bit s: stage s holds a tile to compute
  auto issue = [&](int i, int s) {
    if (i < n) {
      if ((i & 31) == 0) {
        ent = -1;
        if (i + lane < n) {
          const int j = warp + (i + lane) * NW;
          const int page = j / spp;
          const int e = __ldg(table + page);
          if (e < 0 || (p.num_blocks > 0 && e >= p.num_blocks))
            raise_status(p, kDevBadPage);
          else
            ent = (long long)e * p.kv_block_stride + (long long)(j - page * spp) * (9 * D);
        }
      }
      const long long off = __shfl_sync(0xffffffffu, ent, i & 31);
      live &= ~(1u << s);
      if (off >= 0) {
        live |= 1u << s;
        sg.copy(ring + s * C::kStageBytes, kbase + off, vbase + off);
      }
    }
    cp_async_commit();
  };

  float o[4 * W][NT][4] = {};
  float m[NT][2], moff[NT][2], l[NT][2];  // heads 2 t, 2 t + 1 of each tile
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      m[nt][c] = -INFINITY;
      moff[nt][c] = 0.f;
      l[nt][c] = 0.f;
    }

#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) issue(s, s);
  int stage = 0;
  for (int i = 0; i < n; ++i) {
    cp_async_wait<STAGES - 2>();
    __syncwarp();  // every lane's copies of this stage are in; the next one is free
    const int prev = stage == 0 ? STAGES - 1 : stage - 1;
    issue(i + STAGES - 1, prev);
    const uint32_t st = ring + stage * C::kStageBytes;
    const bool compute = (live >> stage) & 1u;
    stage = stage + 1 == STAGES ? 0 : stage + 1;
    if (!compute) continue;  // warp-uniform
    // tokens of this tile, sigma(g) and sigma(g + 8) of this lane's S^T rows
    const int left = (int)(tok_end - tok_begin) - (warp + i * NW) * 16;

    // ── S^T = K . Q^T ─────────────────────────────────────────────────────
    float x[NT][4] = {};
    {
      uint32_t kw[2][2 * W], ks[2][W];
      sg.load_k(st, kw, ks);
#pragma unroll
      for (int i2 = 0; i2 < 2 * W; ++i2) {
        if (!EXACT && 2 * i2 >= NG) break;
        uint32_t a[2][4];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint32_t s2 = fp8x2_to_h2<kKvE4M3>(ks[r][i2 >> 1] >> (16 * (i2 & 1)));
          const uint32_t sl = h2_low2(s2), sh = h2_high2(s2);
          q4x8_to_h2(kw[r][i2], a[r]);
          a[r][0] = h2_mul(a[r][0], sl);
          a[r][1] = h2_mul(a[r][1], sl);
          a[r][2] = h2_mul(a[r][2], sh);
          a[r][3] = h2_mul(a[r][3], sh);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          mma_f16_16816(x[nt], a[0][0], a[1][0], a[0][1], a[1][1], qf[2 * i2][nt][0],
                        qf[2 * i2][nt][1]);
          mma_f16_16816(x[nt], a[0][2], a[1][2], a[0][3], a[1][3], qf[2 * i2 + 1][nt][0],
                        qf[2 * i2 + 1][nt][1]);
        }
      }
    }

    // ── softmax step ──────────────────────────────────────────────────────
    const int tok = 4 * (g >> 1) + (g & 1);
    const bool v0 = tok < left, v1 = tok + 2 < left;
    bool raise = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int c = 0; c < 4; ++c)
        x[nt][c] = ((c & 2) ? v1 : v0) ? x[nt][c] * p.scale_log2 : -INFINITY;
      raise |= fmaxf(x[nt][0], x[nt][2]) > m[nt][0] + kRaise;
      raise |= fmaxf(x[nt][1], x[nt][3]) > m[nt][1] + kRaise;
    }
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float mx = fmaxf(x[nt][c], x[nt][c + 2]);
#pragma unroll
          for (int off = 4; off < 32; off <<= 1)
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
          mx = fmaxf(mx, m[nt][c]);
          const float f = m[nt][c] == -INFINITY ? 0.f : ex2(m[nt][c] - mx);
          m[nt][c] = mx;
          moff[nt][c] = mx == -INFINITY ? 0.f : mx - kShift;
          l[nt][c] *= f;
#pragma unroll
          for (int mt = 0; mt < 4 * W; ++mt) {
            o[mt][nt][c] *= f;
            o[mt][nt][c + 2] *= f;
          }
        }
    }
    uint32_t ph[NT][2], pl[NT][2];  // P^T fragments, hi and lo
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float e[4], lo[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        // a masked score is -inf and its weight 2^-inf = 0, whatever moff is
        e[c] = ex2(x[nt][c] - moff[nt][c & 1]);
        lo[c] = e[c];
      }
      l[nt][0] += e[0] + e[2];
      l[nt][1] += e[1] + e[3];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const uint32_t hi = pack_half2(e[2 * r], e[2 * r + 1]);
        const float2 hf = unpack_half2(hi);
        ph[nt][r] = movmatrix_trans(hi);
        pl[nt][r] = movmatrix_trans(pack_half2(lo[2 * r] - hf.x, lo[2 * r + 1] - hf.y));
      }
    }

    // ── O^T += V^T . P^T ──────────────────────────────────────────────────
    {
      uint32_t vw[4][W], vs[W];
      sg.load_v(st, vw, vs);
      uint32_t keep = 0xffffffffu;  // scales of tokens past the end: 0, their V counts as 0
      if (left < 16) {
        const int nv = left - 4 * t;  // valid tokens among this lane's four
        keep = nv >= 4 ? 0xffffffffu : nv <= 0 ? 0u : (1u << (8 * nv)) - 1u;
      }
#pragma unroll
      for (int w = 0; w < W; ++w) {
        if (!EXACT && w * 8 >= D) break;
        const uint32_t sw = vs[w] & keep;
        const uint32_t s01 = fp8x2_to_h2<kKvE4M3>(sw), s23 = fp8x2_to_h2<kKvE4M3>(sw >> 16);
        uint32_t a[4][4];  // [even 01, odd 01, even 23, odd 23][channel pair]
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          // nibbles of two tokens side by side: byte i = channels 2 i / 2 i + 1
          const uint32_t w0 = vw[2 * k][w], w1 = vw[2 * k + 1][w];
          const uint32_t ev = (w0 & 0x0f0f0f0fu) | ((w1 << 4) & 0xf0f0f0f0u);
          const uint32_t od = ((w0 >> 4) & 0x0f0f0f0fu) | (w1 & 0xf0f0f0f0u);
          q4x8_to_h2(ev, a[2 * k]);
          q4x8_to_h2(od, a[2 * k + 1]);
        }
#pragma unroll
        for (int i2 = 0; i2 < 4; ++i2) {
          const uint32_t a0 = h2_mul(a[0][i2], s01), a1 = h2_mul(a[1][i2], s01);
          const uint32_t a2 = h2_mul(a[2][i2], s23), a3 = h2_mul(a[3][i2], s23);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma_f16_16816(o[4 * w + i2][nt], a0, a1, a2, a3, ph[nt][0], ph[nt][1]);
            mma_f16_16816(o[4 * w + i2][nt], a0, a1, a2, a3, pl[nt][0], pl[nt][1]);
          }
        }
      }
    }
  }
  cp_async_wait<0>();
  __syncthreads();  // the rings become merge space

  // ── merge the warps' (m, l, O) and store ────────────────────────────────
  float* so = reinterpret_cast<float*>(smem);                        // [NW][heads][kRow]
  float* sml = so + (size_t)NW * C::kHeads * C::kRow;                // [NW][heads][2]
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int head = nt * 8 + 2 * t + c;
      float* dst = so + (size_t)(warp * C::kHeads + head) * C::kRow;
#pragma unroll
      for (int mt = 0; mt < 4 * W; ++mt) {
        const int d = 8 * (g * W + (mt >> 2)) + 2 * (mt & 3);
        *reinterpret_cast<float2*>(dst + d) = make_float2(o[mt][nt][c], o[mt][nt][c + 2]);
      }
      float s = l[nt][c];
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
      if (g == 0) {
        sml[(warp * C::kHeads + head) * 2] = m[nt][c];
        sml[(warp * C::kHeads + head) * 2 + 1] = s;
      }
    }
  __syncthreads();
  const int nc = D / 8;
  for (int idx = threadIdx.x; idx < nh * nc; idx += NW * 32) {
    const int head = idx / nc, d0 = (idx - head * nc) * 8;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, sml[(w * C::kHeads + head) * 2]);
    float num[8] = {}, den = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float mw = sml[(w * C::kHeads + head) * 2];
      // a warp without a score above -inf holds zeros, or NaN to pass on
      const float wt = mw == M ? 1.f : ex2(mw - M);
      den = fmaf(wt, sml[(w * C::kHeads + head) * 2 + 1], den);
      const float* src = so + (size_t)(w * C::kHeads + head) * C::kRow + d0;
#pragma unroll
      for (int k = 0; k < 8; ++k) num[k] = fmaf(wt, src[k], num[k]);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) num[k] *= p.v_scale;
    if (it.direct) {
#pragma unroll
      for (int k = 0; k < 8; ++k) num[k] = den == 0.f ? 0.f : num[k] / den;
      if (p.vec8) {
        store_out8<__half>(p, row0 + head, d0, num);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) store_out<__half>(p, row0 + head, d0 + k, num[k]);
      }
    } else {
      const long long pr = (row0 + head) * p.slots + it.slot0 + it.part;
      float* dst = p.part_o + pr * D + d0;
#pragma unroll
      for (int k = 0; k < 8; ++k) dst[k] = num[k];
      if (d0 == 0) {
        p.part_ml[2 * pr] = M;
        p.part_ml[2 * pr + 1] = den;
      }
    }
  }
}

// ── launchers ─────────────────────────────────────────────────────────────
template <typename... KArgs, typename... Args>
cudaError_t launch_pdl(void (*kern)(KArgs...), dim3 grid, unsigned block, size_t smem,
                       cudaStream_t st, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
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

#ifndef XPA_Q4_WARPS
#define XPA_Q4_WARPS 4
#endif
#ifndef XPA_Q4_STAGES
#define XPA_Q4_STAGES 4
#endif
#ifndef XPA_Q4_MIN_CTAS
#define XPA_Q4_MIN_CTAS 4
#endif

template <int W, int NT, bool EXACT>
cudaError_t launch_q4_t(const Params& p, cudaStream_t st) {
  constexpr int NW = XPA_Q4_WARPS, STAGES = XPA_Q4_STAGES;
  constexpr int MINB = (EXACT && W <= 2 && NT == 1) ? XPA_Q4_MIN_CTAS : 1;
  using C = Q4Cfg<W, NT, EXACT, NW, STAGES>;
  auto kern = pa_q4_kernel<W, NT, EXACT, NW, STAGES, MINB>;
  cudaError_t e =
      cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::kSmem);
  if (e != cudaSuccess) return e;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout,
                           (int)cudaSharedmemCarveoutMaxShared);
  if (e != cudaSuccess) return e;
  const long long items = (long long)p.B * p.Hkv * p.max_parts;
  const unsigned chunks = (unsigned)((p.GS + C::kHeads - 1) / C::kHeads);
  return launch_pdl(kern, dim3((unsigned)items, chunks), NW * 32, C::kSmem, st, p);
}

}  // namespace

cudaError_t launch_q4_attention(const Params& p, cudaStream_t st) {
  // 16 heads per CTA where the group has more than 8 and the accumulators fit
  const bool two = p.GS > 8;
  switch (p.D) {
    case 64: return two ? launch_q4_t<1, 2, true>(p, st) : launch_q4_t<1, 1, true>(p, st);
    case 128: return two ? launch_q4_t<2, 2, true>(p, st) : launch_q4_t<2, 1, true>(p, st);
    case 256: return launch_q4_t<4, 1, true>(p, st);
    default: break;
  }
  if (p.D < 64) return launch_q4_t<1, 1, false>(p, st);
  if (p.D < 128) return launch_q4_t<2, 1, false>(p, st);
  if (p.D <= 192) return launch_q4_t<3, 1, false>(p, st);
  return launch_q4_t<4, 1, false>(p, st);
}

cudaError_t launch_q4_write(const Q4RowsParams& a, cudaStream_t st) {
  const long long warps = (long long)a.num_tokens * a.Hkv;
  pa_q4_write_kernel<<<(unsigned)((warps + 3) / 4), 128, 0, st>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_q4_read(const Q4RowsParams& a, cudaStream_t st) {
  const long long warps = (long long)a.num_tokens * a.Hkv;
  pa_q4_read_kernel<<<(unsigned)((warps + 3) / 4), 128, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace xpa
