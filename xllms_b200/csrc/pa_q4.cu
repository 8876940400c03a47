// pa_q4.cu — 4-bit KV cache: rows written and read back by slot, and paged
// decode attention over it. Format and tile layout: pa_q4.cuh.
#include <algorithm>
#include <numeric>
#include <type_traits>
#include <utility>

#include "pa_host.h"
#include "pa_q4.cuh"
#include "pa_q4.h"

namespace xpa {

namespace {

// ════════════════════════════════════════════════════════════════════════
// Rows <-> tiles. A token's K and V rows are pieces of 8 channels, head by head,
// K before V; a lane takes a piece, neighbouring lanes a 16-channel group, and
// a warp P times 32 pieces, whose reads are all in flight together: four where
// that still leaves the GPU warps enough, one for the few tokens of a decode
// step, whose time is the chain of one piece. Instruction issue is the bound:
// storing 8192 tokens x 8 heads x 128 and reading them back (43 MB each) takes 32
// us with the rows and pools in L2 (40 from HBM, where the bytes alone take 13),
// 70-75 % of the issue slots used: the corrected quotients, conversions and
// addresses are 31 instructions a channel to write and 18 to read, the addresses of
// two 2-byte codes and a scale byte for only 8 channels a large part of them. A
// quotient by the reciprocal alone would be off by an ulp, and a code by a step
// wherever that crosses a midpoint.
// ════════════════════════════════════════════════════════════════════════

struct RowAt {
  long long tile;  // byte offset of the 16-token tile in its pool, head 0
  int tok;         // token's row in the tile
};

__device__ __forceinline__ bool q4_row_at(const Q4RowsParams& a, int t, RowAt& r) {
  const long long slot = __ldg(a.slots + t);
  if (slot < 0 || slot >= a.num_slots) return false;
  const long long page = slot / a.block_size;
  const int s = (int)(slot - page * a.block_size);
  r.tile = page * a.kv_block_stride + (long long)(s >> 4) * (9 * a.D);
  r.tok = s & 15;
  return true;
}

// Piece j of a token: its head, its K or V row, its 8 channels, and where they
// are in the tile. K and V lanes go the same way: 16 codes each at two places.
struct Piece {
  int h, v;
  bool is_v;
  int code, code2, scale;  // byte offsets of the codes' halves and the scale
};
__device__ __forceinline__ Piece q4_piece(int D, int tok, int j) {
  const int per_head = D / 4;  // pieces of K and V
  Piece c;
  c.h = j / per_head;
  const int i = j - c.h * per_head;
  c.is_v = i >= per_head / 2;
  c.v = c.is_v ? i - per_head / 2 : i;
  c.code = c.is_v ? q4_v_off(D, tok, c.v) : q4_k_off(D, tok, c.v);
  c.code2 = c.code + (c.is_v ? 2 : D / 8);
  c.scale = c.is_v ? q4_v_scale_off(D, tok, c.v >> 1) : q4_k_scale_off(D, tok, c.v >> 1);
  return c;
}

template <int P, int DC>
__global__ void __launch_bounds__(128) pa_q4_write_kernel(const Q4RowsParams a) {
  const int D = DC ? DC : a.D;
  const int w = (int)(((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5);
  const int lane = threadIdx.x & 31;
  const int t = w / a.warps_per_token, first = (w - t * a.warps_per_token) * 32 * P;
  if (t >= a.num_tokens) return;
  const int pieces = a.Hkv * (D / 4);
  RowAt r;
  const bool live = q4_row_at(a, t, r);
  const long long src = (long long)t * a.token_stride;
  const int tok = live ? r.tok : 0;
  uint4 x4[P];
#pragma unroll
  for (int k = 0; k < P; ++k) {
    const int j = first + 32 * k + lane;
    x4[k] = make_uint4(0u, 0u, 0u, 0u);
    if (j >= pieces) continue;
    const Piece c = q4_piece(D, tok, j);
    const __half* row =
        static_cast<const __half*>(c.is_v ? a.value : a.key) + src + c.h * D + c.v * 8;
    if (a.vec16) {
      x4[k] = __ldg(reinterpret_cast<const uint4*>(row));
    } else {
      const unsigned short* u = reinterpret_cast<const unsigned short*>(row);
      x4[k] = make_uint4(u[0] | ((uint32_t)u[1] << 16), u[2] | ((uint32_t)u[3] << 16),
                         u[4] | ((uint32_t)u[5] << 16), u[6] | ((uint32_t)u[7] << 16));
    }
  }
  if (!live) return;  // warp-uniform
#pragma unroll
  for (int k = 0; k < P; ++k) {
    const int j = first + 32 * k + lane;
    if (first + 32 * k >= pieces) break;  // warp-uniform
    const Piece c = q4_piece(D, tok, j);
    const float ps = c.is_v ? a.v_scale : a.k_scale, inv = c.is_v ? a.v_inverse : a.k_inverse;
    const uint32_t u[4] = {x4[k].x, x4[k].y, x4[k].z, x4[k].w};
    float x[8], amax = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack_half2(u[i]);
      x[2 * i] = div_by(f.x, ps, inv);
      x[2 * i + 1] = div_by(f.y, ps, inv);
    }
    if (a.divide) {  // a scale that div_by does not take
#pragma unroll 1
      for (int i = 0; i < 8; ++i) {
        const float y = __half2float(__ushort_as_half(
            (unsigned short)((i < 2 ? x4[k].x : i < 4 ? x4[k].y : i < 6 ? x4[k].z : x4[k].w) >>
                             (16 * (i & 1)))));
        const float q = __fdiv_rn(y, ps);
#pragma unroll
        for (int m = 0; m < 8; ++m) x[m] = m == i ? q : x[m];
      }
    }
    // A quotient that is an infinity or a NaN (an infinity's residual is one)
    // stands for an infinity, here any value whose scale saturates, or a NaN: 0.
    constexpr float kHuge = 1e30f;
    bool odd = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) odd |= !(fabsf(x[i]) < kHuge);
    if (odd) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 f = unpack_half2(u[i >> 1]);
        const float y = i & 1 ? f.y : f.x;
        if (!(fabsf(x[i]) < kHuge)) x[i] = isnan(y) ? 0.f : copysignf(kHuge, y);
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(x[i]));
    // a 16-channel group is two neighbouring lanes (pieces 2 g, 2 g + 1)
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    if (j >= pieces) continue;
    const uint32_t sb = q4_scale(amax);
    const float s = fp8_to_float<kKvE4M3>((uint8_t)sb);
    const float si = s > 0.f ? __frcp_rn(s) : 0.f;
    uint32_t code = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack_half2(u[i]);  // the signs, zeros' too
      code |= q4_pair(copysignf(div_by(x[2 * i], s, si), f.x),
                      copysignf(div_by(x[2 * i + 1], s, si), f.y))
              << (8 * i);
    }
    if (!(s > 0.f)) code = 0;  // no scale
    uint8_t* tile = static_cast<uint8_t*>(c.is_v ? a.value_cache : a.key_cache) + r.tile +
                    c.h * a.kv_head_stride;
    *reinterpret_cast<uint16_t*>(tile + c.code) = (uint16_t)code;
    *reinterpret_cast<uint16_t*>(tile + c.code2) = (uint16_t)(code >> 16);
    if ((c.v & 1) == 0) tile[c.scale] = (uint8_t)sb;
  }
}

template <int P, int DC>
__global__ void __launch_bounds__(128) pa_q4_read_kernel(const Q4RowsParams a) {
  const int D = DC ? DC : a.D;
  const int w = (int)(((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5);
  const int lane = threadIdx.x & 31;
  const int t = w / a.warps_per_token, first = (w - t * a.warps_per_token) * 32 * P;
  if (t >= a.num_tokens) return;
  const int pieces = a.Hkv * (D / 4);
  RowAt r;
  const bool live = q4_row_at(a, t, r);
  uint32_t code[P], sb[P];
#pragma unroll
  for (int k = 0; k < P; ++k) {
    const int j = first + 32 * k + lane;
    code[k] = sb[k] = 0u;  // a row of zeros
    if (!live || j >= pieces) continue;
    const Piece c = q4_piece(D, r.tok, j);
    const uint8_t* tile = static_cast<const uint8_t*>(c.is_v ? a.value_cache : a.key_cache) +
                          r.tile + c.h * a.kv_head_stride;
    code[k] = __ldg(reinterpret_cast<const uint16_t*>(tile + c.code)) |
              ((uint32_t)__ldg(reinterpret_cast<const uint16_t*>(tile + c.code2)) << 16);
    sb[k] = __ldg(tile + c.scale);
  }
#pragma unroll
  for (int k = 0; k < P; ++k) {
    const int j = first + 32 * k + lane;
    if (j >= pieces) break;
    const Piece c = q4_piece(D, 0, j);
    const uint32_t s2 = fp8x2_to_h2<kKvE4M3>(sb[k]);
    const float ps = c.is_v ? a.v_scale : a.k_scale;
    uint32_t h[4], o[4];
    q4x8_to_h2(code[k], h);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // c * s is exact in fp16, times ps in fp32, rounded to fp16 and, where a
      // group's largest element may have been rounded up past the range, kept finite
      const float2 f = unpack_half2(h2_mul_low(h[i], s2));
      float x = f.x * ps, y = f.y * ps;
      if (a.clamp) {
        x = fminf(fmaxf(x, -65504.f), 65504.f);
        y = fminf(fmaxf(y, -65504.f), 65504.f);
      }
      o[i] = pack_half2(x, y);
    }
    __half* dst = static_cast<__half*>(c.is_v ? a.value : a.key) +
                  (long long)t * a.token_stride + c.h * D + c.v * 8;
    if (a.vec16) {
      *reinterpret_cast<uint4*>(dst) = make_uint4(o[0], o[1], o[2], o[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        dst[i] = __ushort_as_half((unsigned short)(o[i >> 1] >> (16 * (i & 1))));
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
//   O^T(D x 8 heads)         += V^T . P^T    V as A, D / 16 row tiles
// Token order: row r of S^T (and k index r of P^T) is token sigma(r) with
// sigma(2 t) = 4 t, sigma(2 t + 1) = 4 t + 1, sigma(8 + 2 t) = 4 t + 2,
// sigma(9 + 2 t) = 4 t + 3, so a lane's four V tokens are 4 t .. 4 t + 3 and
// their scales one word. Channel order: K step j's k index 2 t, 2 t + 1,
// 2 t + 8, 2 t + 9 are channels 16 j + 4 t .. + 3 (Q's fragments follow); V
// row tile 4 w + i holds channels 8 (g W + w) + 2 i (row g) and + 1 (row g + 8).
//
// Softmax: the reference point m of a head moves only when a score exceeds it
// by more than 8 in the exp2 domain, so most steps need one vote and no
// shuffles. Exponents are formed from x - m: the distance is all but exact
// where it matters, while x or m times the scale is rounded by more than a whole
// unit from 2^25 on. The weights p = 2^(x - m + 7) <= 2^15 go into the
// product as two fp16 terms, p rounded and what that leaves: 22 bits, like the
// other decode kernels' (2^-22 of a weight at most, 2^-32 of the largest where
// the second term is subnormal). The rounded weight alone takes a tenth less
// time (64 sequences of 1-8K tokens: 78 us against 86) and adds an error as large
// as the output's own rounding.
//
// Bound and measured, 32 heads over 8 of 128: 12 sequences of 64K tokens (906
// MB) take 198 us, 0.70 of the copy rate, 64 of 1-8K (336 MB) 88 us, 0.58, as
// the items of a ragged batch end apart (shorter items, or the short ones last,
// were no faster); 61 us if nothing is computed, 75 if nothing is copied. At the
// copy rate there are 3.1 issue slots for 32 elements and the kernel uses 2.4,
// half an instruction each of them for conversions and scalings; the long case
// has the issue slots 62 % busy, the conversions' half-rate pipe 49 %, the tensor
// pipe 38 %, and a warp waits for its turn, a fixed latency or a pipe. So the
// shape that counts is the one with the fewest
// instructions per element: K and V go through mma.sync straight from
// registers, where tcgen05 would want the unpacked fp16 operands written to
// shared memory first (3.6 times the bytes that were read) and the few rows of
// heads would fill a sixteenth of its tiles; and two tiles a step give a warp
// two independent chains. A loop over the ring's stages instead of their
// unrolling, a third stage, a fifth CTA per SM and Q kept in shared memory were
// each slower.
// ════════════════════════════════════════════════════════════════════════
constexpr float kRaise = 8.f;  // log2 units a score may exceed m by
constexpr float kShift = 7.f;  // p = 2^(x - m + kShift) <= 2^15

template <int D, int NT, int NW, int STAGES, int U>
struct Q4Cfg {
  static constexpr int kDMax = (D + 63) / 64 * 64;  // whole words of V per lane
  static constexpr int kHeads = 8 * NT;
  static constexpr int kTileBytes = 18 * D;         // one K and one V tile
  static constexpr int kStageBytes = U * kTileBytes;
  static constexpr int kRow = kDMax + 4;          // merge rows, floats
  static constexpr size_t kMergeBytes =
      (size_t)NW * kHeads * kRow * sizeof(float) + (size_t)NW * kHeads * 2 * sizeof(float);
  static constexpr size_t kRingBytes = (size_t)NW * STAGES * kStageBytes;
  static constexpr size_t kSmem = kRingBytes > kMergeBytes ? kRingBytes : kMergeBytes;
};

// Shared-memory reads and copies at compile-time offsets from one register.
template <int OFF>
__device__ __forceinline__ uint32_t lds16(uint32_t a) {
  uint16_t r;
  asm volatile("ld.shared.b16 %0, [%1+%2];" : "=h"(r) : "r"(a), "n"(OFF));
  return r;
}
template <int OFF>
__device__ __forceinline__ uint32_t lds8(uint32_t a) {
  uint32_t r;
  asm volatile("ld.shared.u8 %0, [%1+%2];" : "=r"(r) : "r"(a), "n"(OFF));
  return r;
}
template <int N, int OFF>
__device__ __forceinline__ void lds_words(uint32_t a, uint32_t* r) {
  if constexpr (N == 1) {
    asm volatile("ld.shared.b32 %0, [%1+%2];" : "=r"(r[0]) : "r"(a), "n"(OFF));
  } else if constexpr (N == 2) {
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2+%3];"
                 : "=r"(r[0]), "=r"(r[1])
                 : "r"(a), "n"(OFF));
  } else {
    static_assert(N == 4, "1, 2 or 4 words");
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4+%5];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a), "n"(OFF));
  }
}
template <int DST, int SRC>
__device__ __forceinline__ void cp_async16_at(uint32_t dst, const uint8_t* src) {
  asm volatile("cp.async.cg.shared.global [%0+%2], [%1+%3], 16;" ::"r"(dst), "l"(src), "n"(DST),
               "n"(SRC)
               : "memory");
}

// Where a tile's pieces sit in a ring stage, and one lane's copies and reads
// of them; S0 is the stage's byte offset in the warp's ring.
// EXACT (D = 64 W, W = 1, 2, 4): rows are placed and chunks swizzled so that
// every read below is conflict-free; K row r's place is its S^T row, V row
// 4 t + k's place is 4 k + t. Otherwise a tile is copied as it is.
template <int D>
struct Q4Stage {
  static constexpr int W = (D + 63) / 64;
  static constexpr bool EXACT = D == 64 || D == 128 || D == 256;
  int lane, g, t;
  // sources in page 0; EXACT: this lane's first chunk of each piece
  const uint8_t *ksrc, *vsrc, *ssrc;
  uint32_t ring;               // the warp's ring
  uint32_t kd, sd, vd[W];      // EXACT: copy destinations in stage 0
  uint32_t ka[2], ksa, va, vsa;  // read addresses in stage 0

  __device__ __forceinline__ Q4Stage(int lane_, const uint8_t* k, const uint8_t* v,
                                     uint32_t ring_)
      : lane(lane_), ksrc(k), vsrc(v), ssrc(k), ring(ring_) {
    g = lane >> 2;
    t = lane & 3;
    const int tok = 4 * (g >> 1) + (g & 1);  // sigma(g); sigma(g + 8) is + 2
    if constexpr (EXACT) {
      constexpr int DD = D;
      constexpr int CPR = 2 * W;  // 16-byte chunks per row
      ksrc = k + lane * 16;
      vsrc = v + lane * 16;
      // both tiles' scales: D / 16 chunks each, lanes 0.. and 16..
      const int sc = lane & 15;
      ssrc = (lane < 16 ? k : v) + 8 * DD + sc * 16;
      sd = ring + 16 * DD + (lane >> 4) * DD + sc * 16;
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const int x = lane + 32 * i, r = x / CPR, c = x % CPR;
        const int kp = 2 * (r >> 2) + (r & 1) + 8 * ((r >> 1) & 1);
        const int vp = 4 * (r & 3) + (r >> 2);
        int ck = c, cv = c;
        if (W == 4) ck = c ^ (kp & 1);
        if (W == 2) cv = c ^ (2 * ((vp >> 1) & 1));
        if (W == 4) cv = c ^ (2 * (vp & 3));
        // 32 chunks further on is a whole number of token groups: the K place
        // moves by a constant
        if (i == 0) kd = ring + (uint32_t)(kp * 32 * W + ck * 16);
        vd[i] = ring + (uint32_t)(8 * DD + vp * 32 * W + cv * 16);
      }
      const uint32_t row = ring + g * 32 * W;
      ka[0] = ka[1] = row + t * 8 * W;
      if (W == 4) {
        ka[0] = row + (((2 * t) ^ (g & 1)) << 4);
        ka[1] = row + (((2 * t + 1) ^ (g & 1)) << 4);
      }
      ksa = ring + 16 * DD + tok * 4 * W;
      va = ring + 8 * DD + t * 32 * W;
      if (W == 1) va += 4 * g;
      if (W == 2) va += (((g >> 1) ^ (t & 2)) << 4) + (g & 1) * 8;
      if (W == 4) va += (g ^ (2 * t)) << 4;
      vsa = ring + 17 * DD + 4 * t + (g * W >> 1) * 16;
    } else {
      ka[0] = ka[1] = ring + tok * (D / 2) + t * (D / 8);
      ksa = ring + 8 * D + tok * (D / 16);
      va = ring + 9 * D;
      vsa = ring + 17 * D + 4 * t;
    }
  }

  // Issues the copies of the K and V tiles that start `at` units into the pools.
  template <int S0>
  __device__ __forceinline__ void copy(unsigned at, unsigned unit) const {
    if constexpr (EXACT) {
      // rows per 32 chunks: 16 / W; their K places are 2 * (16 / W) / 4 apart
      constexpr int kStep = W == 1 ? 0 : (16 / W / 4) * 2 * 32 * W;
      const uint8_t* k = ksrc + (unsigned long long)at * unit;
      const uint8_t* v = vsrc + (unsigned long long)at * unit;
      const uint8_t* s = ssrc + (unsigned long long)at * unit;
      cp_async16_at<S0, 0>(kd, k);
      if constexpr (W >= 2) cp_async16_at<S0 + kStep, 512>(kd, k);
      if constexpr (W == 4) {
        cp_async16_at<S0 + 2 * kStep, 1024>(kd, k);
        cp_async16_at<S0 + 3 * kStep, 1536>(kd, k);
      }
      cp_async16_at<S0, 0>(vd[0], v);
      if constexpr (W >= 2) cp_async16_at<S0, 512>(vd[1], v);
      if constexpr (W == 4) {
        cp_async16_at<S0, 1024>(vd[2], v);
        cp_async16_at<S0, 1536>(vd[3], v);
      }
      if (W == 4 || (lane & 15) < 4 * W) cp_async16_at<S0, 0>(sd, s);
    } else {
      const unsigned long long off = (unsigned long long)at * unit;
      constexpr int n = 9 * D / 16;
#pragma unroll
      for (int i = 0; i < (n + 31) / 32; ++i) {
        const int x = lane + 32 * i;
        if (x < n) {
          cp_async16_at<S0, 0>(ring + x * 16, ksrc + off + x * 16);
          cp_async16_at<S0, 0>(ring + 9 * D + x * 16, vsrc + off + x * 16);
        }
      }
    }
  }

  // K codes and scales of S^T rows g (r = 0) and g + 8 (r = 1): word i of kw
  // is groups 2 i, 2 i + 1; byte j of ks is group j's scale.
  template <int S0>
  __device__ __forceinline__ void load_k(uint32_t (&kw)[2][2 * W], uint32_t (&ks)[2][W]) const {
    if constexpr (EXACT) {
      constexpr int kRows = 8 * 32 * W;
      if constexpr (W == 4) {
        lds_words<4, S0>(ka[0], kw[0]);
        lds_words<4, S0>(ka[1], kw[0] + 4);
        lds_words<4, S0 + kRows>(ka[0], kw[1]);
        lds_words<4, S0 + kRows>(ka[1], kw[1] + 4);
      } else {
        lds_words<2 * W, S0>(ka[0], kw[0]);
        lds_words<2 * W, S0 + kRows>(ka[0], kw[1]);
      }
      lds_words<W, S0>(ksa, ks[0]);
      lds_words<W, S0 + 8 * W>(ksa, ks[1]);
    } else {
      constexpr int NG = D / 16;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const uint32_t row = ka[0] + 2 * r * (D / 2);
        const uint32_t sc = ksa + 2 * r * NG;
#pragma unroll
        for (int i = 0; i < 2 * W; ++i) {
          kw[r][i] = 0u;
          if constexpr (NG % 2 == 0) {  // whole words
            if (2 * i < NG) lds_words<1, S0>(row + 4 * i, &kw[r][i]);
          } else {
            if (2 * i < NG) kw[r][i] = lds16<S0>(row + 4 * i);
            if (2 * i + 1 < NG) kw[r][i] |= lds16<S0>(row + 4 * i + 2) << 16;
          }
        }
#pragma unroll
        for (int i = 0; i < W; ++i) {
          ks[r][i] = 0u;
          if constexpr (NG % 4 == 0) {
            if (4 * i < NG) lds_words<1, S0>(sc + 4 * i, &ks[r][i]);
          } else if constexpr (NG % 2 == 0) {
            if (4 * i < NG) ks[r][i] = lds16<S0>(sc + 4 * i);
            if (4 * i + 2 < NG) ks[r][i] |= lds16<S0>(sc + 4 * i + 2) << 16;
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (4 * i + j < NG) ks[r][i] |= lds8<S0>(sc + 4 * i + j) << (8 * j);
          }
        }
      }
    }
  }

  // V codes of tokens 4 t + k: word w is channels 8 (g W + w) .. + 7; vs[w]
  // holds the four tokens' scales of those channels.
  template <int S0>
  __device__ __forceinline__ void load_v(uint32_t (&vw)[4][W], uint32_t (&vs)[W]) const {
    if constexpr (EXACT) {
      constexpr int kRows = 4 * 32 * W;
      lds_words<W, S0>(va, vw[0]);
      lds_words<W, S0 + kRows>(va, vw[1]);
      lds_words<W, S0 + 2 * kRows>(va, vw[2]);
      lds_words<W, S0 + 3 * kRows>(va, vw[3]);
      lds_words<1, S0>(vsa, vs);
      if constexpr (W == 2) vs[1] = vs[0];
      if constexpr (W == 4) {
        vs[1] = vs[0];
        lds_words<1, S0 + 16>(vsa, vs + 2);
        vs[3] = vs[2];
      }
    } else {
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const int at = g * W + w;
        const bool in = at < D / 8;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          vw[k][w] = 0u;
          if (in) lds_words<1, S0>(va + (4 * t + k) * (D / 2) + at * 4, &vw[k][w]);
        }
        vs[w] = 0u;
        if (in) lds_words<1, S0>(vsa + (at >> 1) * 16, &vs[w]);
      }
    }
  }
};

// f(0), f(1), ..., f(N - 1) with compile-time arguments, until one is false.
template <int N, int I = 0, typename F>
__device__ __forceinline__ bool each_stage(F&& f) {
  if constexpr (I < N) {
    if (!f(std::integral_constant<int, I>{})) return false;
    return each_stage<N, I + 1>(static_cast<F&&>(f));
  }
  return true;
}

// Addresses of one call: a tile starts at a whole number of units in its pool.
struct Q4Units {
  unsigned unit, page_units, tile_units;  // bytes; units per page, per tile
  int page_limit;   // page ids below this are in the pools
  int head_chunks;  // CTAs per group of query heads
};

template <int D, int NT, int NW, int STAGES, int U, int MINB>
__global__ void __launch_bounds__(NW * 32, MINB) pa_q4_kernel(const Params p, const Q4Units q) {
  using C = Q4Cfg<D, NT, NW, STAGES, U>;
  constexpr int W = Q4Stage<D>::W, NG = D / 16;  // V words per lane, channel groups
  extern __shared__ __align__(128) uint8_t smem[];
  // Every CTA waits for the kernel before this one (which may be this call's
  // append); the merge may be scheduled from here on and waits for this grid.
  pdl_wait_primary();
  pdl_launch_dependents();
  Item it;
  // grid: x = partition, y and z = (sequence, KV head, head chunk)
  const int col = blockIdx.y + blockIdx.z * kGridY;
  if (col >= p.B * p.Hkv * q.head_chunks) return;
  const int row = q.head_chunks == 1 ? col : col / q.head_chunks;
  const ItemKind kind = part_item(p, row, it);
  if (kind == kItemNone) return;
  const int h0 = (col - row * q.head_chunks) * C::kHeads;
  const int nh = min(p.GS - h0, C::kHeads);
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
  const float slack = fminf(kRaise / sl, 1e30f);  // kRaise in units of q . k

  // ── Q fragments: head g of tile nt, channels 16 j + 4 t .. + 3 ──────────
  // Groups go in pairs, a missing one as 0, so that both halves of a word of codes
  // are used (q4x8_to_h2).
  constexpr int NGP = NG + NG % 2;
  uint32_t qf[NGP][NT][2];
  {
    const __half* query = static_cast<const __half*>(p.q);
    const bool al = (reinterpret_cast<uintptr_t>(query) & 7u) == 0;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const bool head = nt * 8 + g < nh;
      const __half* src = query + (row0 + nt * 8 + g) * D + 4 * t;
#pragma unroll
      for (int j = 0; j < NGP; ++j) {
        uint2 u = make_uint2(0u, 0u);
        if (head && j < NG) {
          if (al) {
            u = __ldg(reinterpret_cast<const uint2*>(src + 16 * j));
          } else {
            const unsigned short* s = reinterpret_cast<const unsigned short*>(src + 16 * j);
            u.x = s[0] | ((uint32_t)s[1] << 16);
            u.y = s[2] | ((uint32_t)s[3] << 16);
          }
        }
        if (sign <= 0.f) {
          u.x = h2_mul(u.x, pack_half2(sign, sign));
          u.y = h2_mul(u.y, pack_half2(sign, sign));
        }
        qf[j][nt][0] = u.x;
        qf[j][nt][1] = u.y;
      }
    }
  }

  // ── this warp's steps of U tiles: i = warp, warp + NW, ... of the item ──
  const int spp = p.block_size >> 4;  // tiles per page
  const long long tok_end = min((long long)it.L, (long long)it.page_end * p.block_size);
  const int tok_begin = it.page_begin * p.block_size;
  const int tiles = (int)((tok_end - tok_begin + 15) >> 4);
  const int steps = (tiles + U - 1) / U;
  const int n = steps > warp ? (steps - warp + NW - 1) / NW : 0;
  const long long head_off = (long long)it.kvh * p.kv_head_stride;
  const Q4Stage<D> sg(lane, static_cast<const uint8_t*>(p.k) + head_off,
                      static_cast<const uint8_t*>(p.v) + head_off,
                      smem_u32(smem) + warp * (STAGES * C::kStageBytes));
  const int* table = p.block_tables + (long long)it.b * p.max_blocks + it.page_begin;
  auto entry_ok = [&](int e) { return e >= 0 && e < q.page_limit; };

  constexpr int kBatch = 32 / U;
  constexpr unsigned kNone = 0xffffffffu;
  // lane l: where tile l % U of step i - i % kBatch + l / U starts, in units
  unsigned ent = kNone;
  bool masked = false;  // a page of this warp's is masked
  auto tile_page = [&](int i, int u) { return (U * (warp + i * NW) + u) / spp; };
  auto issue = [&](int i, auto stage) {
    constexpr int S0 = decltype(stage)::value * C::kStageBytes;
    if (i < n) {
      if (i % kBatch == 0) {
        bool bad = false;
        const int j = U * (warp + (i + lane / U) * NW) + lane % U;
        ent = kNone;
        if (j < tiles) {
          const int page = spp == 1 ? j : j / spp;
          const int e = __ldg(table + page);
          bad = !entry_ok(e);
          if (bad)
            raise_status(p, kDevBadPage);
          else
            ent = (unsigned)e * q.page_units + (unsigned)(j - page * spp) * q.tile_units;
        }
        masked |= __any_sync(0xffffffffu, bad);
      }
      const int l = U * (i % kBatch);
      each_stage<U>([&](auto u) {
        constexpr int T0 = S0 + decltype(u)::value * C::kTileBytes;
        const unsigned at = __shfl_sync(0xffffffffu, ent, l + decltype(u)::value);
        if (at != kNone) sg.template copy<T0>(at, q.unit);
        return true;
      });
    }
    cp_async_commit();
  };

  float o[4 * W][NT][4] = {};
  // Heads 2 t, 2 t + 1 of each tile: the reference point m in units of q . k,
  // and the weights' sum.
  float m[NT][2], l[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      m[nt][c] = kNoScore;
      l[nt][c] = 0.f;
    }

  // The warp's i-th step, from ring stage `stage`; false after the last.
  int left = (int)(tok_end - tok_begin) - warp * (16 * U);  // tokens from this step on
  auto step = [&](int i, auto stage) {
    constexpr int S = decltype(stage)::value, S0 = S * C::kStageBytes;
    if (i >= n) return false;
    cp_async_wait<STAGES - 2>();
    __syncwarp();  // every lane's copies of this stage are in; the one before is free
    issue(i + STAGES - 1, std::integral_constant<int, (S + STAGES - 1) % STAGES>{});
    int here[U];  // valid tokens of each tile, when below 16
#pragma unroll
    for (int u = 0; u < U; ++u) here[u] = left - 16 * u;
    left -= 16 * U * NW;
    if (masked) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (here[u] > 0 && !entry_ok(__ldg(table + tile_page(i, u)))) here[u] = 0;
    }
    const bool partial = here[0] < 16 || here[U - 1] < 16;

    // ── S^T = K . Q^T ─────────────────────────────────────────────────────
    float x[U][NT][4] = {};
    {
      uint32_t kw[U][2][2 * W], ks[U][2][W];
      each_stage<U>([&](auto u) {
        constexpr int V = decltype(u)::value;
        sg.template load_k<S0 + V * C::kTileBytes>(kw[V], ks[V]);
        return true;
      });
#pragma unroll
      for (int i2 = 0; i2 < 2 * W; ++i2) {
        if (2 * i2 >= NGP) break;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          uint32_t a[2][4];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            // scales of groups 2 i2 and 2 i2 + 1
            const uint32_t s2 = fp8x2_to_h2<kKvE4M3>(ks[u][r][i2 >> 1] >> (16 * (i2 & 1)));
            q4x8_to_h2(kw[u][r][i2], a[r]);
            a[r][0] = h2_mul_low(a[r][0], s2);
            a[r][1] = h2_mul_low(a[r][1], s2);
            a[r][2] = h2_mul_high(a[r][2], s2);
            a[r][3] = h2_mul_high(a[r][3], s2);
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma_f16_16816(x[u][nt], a[0][0], a[1][0], a[0][1], a[1][1], qf[2 * i2][nt][0],
                          qf[2 * i2][nt][1]);
            mma_f16_16816(x[u][nt], a[0][2], a[1][2], a[0][3], a[1][3], qf[2 * i2 + 1][nt][0],
                          qf[2 * i2 + 1][nt][1]);
          }
        }
      }
    }

    // ── softmax step ──────────────────────────────────────────────────────
    if (partial) {  // tokens sigma(g) and sigma(g + 8)
      const int tok = 4 * (g >> 1) + (g & 1);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          if (tok >= here[u]) x[u][nt][0] = x[u][nt][1] = -INFINITY;
          if (tok + 2 >= here[u]) x[u][nt][2] = x[u][nt][3] = -INFINITY;
        }
    }
    auto top = [&](int nt, int c) {
      float mx = fmaxf(x[0][nt][c], x[0][nt][c + 2]);
#pragma unroll
      for (int u = 1; u < U; ++u) mx = fmaxf(mx, fmaxf(x[u][nt][c], x[u][nt][c + 2]));
      return mx;
    };
    bool raise = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c)
        raise |= top(nt, c) - m[nt][c] > slack;
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float mx = top(nt, c);
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
          mx = fmaxf(mx, m[nt][c]);
          const float f = ex2((m[nt][c] - mx) * sl);
          m[nt][c] = mx;
          l[nt][c] *= f;
#pragma unroll
          for (int mt = 0; mt < 4 * W; ++mt) {
            o[mt][nt][c] *= f;
            o[mt][nt][c + 2] *= f;
          }
        }
    }
    uint32_t pf[U][NT][2], pl[U][NT][2];  // P^T fragments: a weight's fp16 value, and what that leaves
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float e[4];
#pragma unroll
        for (int c = 0; c < 4; ++c)  // a masked score is -inf and its weight 0, whatever m is
          e[c] = ex2(fmaf(x[u][nt][c] - m[nt][c & 1], sl, kShift));
        l[nt][0] += e[0] + e[2];
        l[nt][1] += e[1] + e[3];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint32_t h = pack_half2(e[2 * r], e[2 * r + 1]);
          const float2 f = unpack_half2(h);
          pf[u][nt][r] = movmatrix_trans(h);
          pl[u][nt][r] = movmatrix_trans(pack_half2(e[2 * r] - f.x, e[2 * r + 1] - f.y));
        }
      }

    // ── O^T += V^T . P^T ──────────────────────────────────────────────────
    // scales of tokens past the end become 0, so their V counts as 0
    uint32_t keep[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      keep[u] = 0xffffffffu;
      if (partial) {
        const int nv = here[u] - 4 * t;  // valid tokens among this lane's four
        keep[u] = nv >= 4 ? 0xffffffffu : nv <= 0 ? 0u : (1u << (8 * nv)) - 1u;
      }
    }
    uint32_t vw[U][4][W], vs[U][W];
    each_stage<U>([&](auto u) {
      constexpr int V = decltype(u)::value;
      sg.template load_v<S0 + V * C::kTileBytes>(vw[V], vs[V]);
      return true;
    });
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const uint32_t sw = vs[u][w] & keep[u];
        const uint32_t s01 = fp8x2_to_h2<kKvE4M3>(sw), s23 = fp8x2_to_h2<kKvE4M3>(sw >> 16);
        uint32_t a[4][4];  // [even 01, odd 01, even 23, odd 23][channel pair]
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          // nibbles of two tokens side by side: byte i = channels 2 i / 2 i + 1
          const uint32_t w0 = vw[u][2 * k][w], w1 = vw[u][2 * k + 1][w];
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
            mma_f16_16816(o[4 * w + i2][nt], a0, a1, a2, a3, pf[u][nt][0], pf[u][nt][1]);
            mma_f16_16816(o[4 * w + i2][nt], a0, a1, a2, a3, pl[u][nt][0], pl[u][nt][1]);
          }
        }
      }
    return true;
  };
  each_stage<STAGES - 1>([&](auto s) {
    issue(decltype(s)::value, s);
    return true;
  });
  for (int i = 0; each_stage<STAGES>([&](auto s) { return step(i + decltype(s)::value, s); });)
    i += STAGES;
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
        sml[(warp * C::kHeads + head) * 2] = m[nt][c] == kNoScore ? -INFINITY : m[nt][c];
        sml[(warp * C::kHeads + head) * 2 + 1] = s;
      }
    }
  __syncthreads();
  merge_warps<NW, C::kHeads, C::kRow>(p, it, so, sml, row0, nh, D);
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
#ifndef XPA_Q4_TILES
#define XPA_Q4_TILES 2
#endif
#ifndef XPA_Q4_STAGES
#define XPA_Q4_STAGES 2
#endif
#ifndef XPA_Q4_MIN_CTAS
#define XPA_Q4_MIN_CTAS 4
#endif
#ifndef XPA_Q4_MIN_CTAS_ODD
#define XPA_Q4_MIN_CTAS_ODD 2
#endif
#ifndef XPA_Q4_MIN_CTAS_LARGE
#define XPA_Q4_MIN_CTAS_LARGE 3
#endif

template <int D, int NT>
cudaError_t launch_q4_t(const Params& p, cudaStream_t st) {
  constexpr bool EXACT = Q4Stage<D>::EXACT;
  constexpr int NW = XPA_Q4_WARPS;
  // two tiles a step against one and a ring of four, 64 sequences of 1-8K tokens:
  // D = 64 59 against 61 us, 96 85 / 90, 128 88 / 94, 160 122 / 149, 240 222 / 243
  constexpr int U = XPA_Q4_TILES, STAGES = XPA_Q4_STAGES;
  // Resident CTAs per SM that the registers are held down for. Head sizes without a
  // swizzle of their own take more: four of them at 80 to 112 gain 2-3 % there and
  // lose 5 % on short ragged rows. From 144 to 192 three CTAs take 129, 122, 147, 127
  // us (144, 160, 176, 192; as above), two 143, 134, 161, 141.
  constexpr int MINB = NT > 1              ? 1
                       : EXACT && D <= 128 ? XPA_Q4_MIN_CTAS
                       : D <= 128          ? XPA_Q4_MIN_CTAS_ODD
                       : D <= 192          ? XPA_Q4_MIN_CTAS_LARGE
                                           : 1;
  using C = Q4Cfg<D, NT, NW, STAGES, U>;
  auto kern = pa_q4_kernel<D, NT, NW, STAGES, U, MINB>;
  static std::atomic<unsigned long long> done{0};
  const cudaError_t e = host::smem_limit(kern, C::kSmem, true, done);
  if (e != cudaSuccess) return e;
  // addresses in the largest unit that divides a page's and a tile's bytes
  Q4Units q;
  const unsigned tile = 9u * p.D, page = (unsigned)p.kv_block_stride;
  q.unit = page ? std::gcd(page, tile) : tile;
  q.page_units = page / q.unit;
  q.tile_units = tile / q.unit;
  // page ids whose addresses fit in 32 bits of units; the rest are masked
  const unsigned spp = (unsigned)p.block_size / 16;
  long long limit = 0x7fffffffLL;
  if (q.page_units > 0)
    limit = std::min(limit, (0xfffffffeLL - (long long)spp * q.tile_units) / q.page_units);
  if (p.num_blocks > 0) limit = std::min(limit, p.num_blocks);
  q.page_limit = (int)limit;
  q.head_chunks = (p.GS + C::kHeads - 1) / C::kHeads;
  const long long cols = (long long)p.B * p.Hkv * q.head_chunks;
  const dim3 grid((unsigned)p.max_parts, (unsigned)std::min<long long>(cols, kGridY),
                  (unsigned)((cols + kGridY - 1) / kGridY));
  return launch_pdl(kern, grid, NW * 32, C::kSmem, st, p, q);
}

}  // namespace

cudaError_t launch_q4_attention(const Params& p, cudaStream_t st) {
  // 16 heads per CTA where the group has more than 8 and the accumulators fit
  const bool two = p.GS > 8;
  switch (p.D) {
#define XPA_Q4_SMALL(D) \
  case D:               \
    return two ? launch_q4_t<D, 2>(p, st) : launch_q4_t<D, 1>(p, st)
#define XPA_Q4_LARGE(D) \
  case D:               \
    return launch_q4_t<D, 1>(p, st)
    XPA_Q4_SMALL(16);
    XPA_Q4_SMALL(32);
    XPA_Q4_SMALL(48);
    XPA_Q4_SMALL(64);
    XPA_Q4_SMALL(80);
    XPA_Q4_SMALL(96);
    XPA_Q4_SMALL(112);
    XPA_Q4_SMALL(128);
    XPA_Q4_LARGE(144);
    XPA_Q4_LARGE(160);
    XPA_Q4_LARGE(176);
    XPA_Q4_LARGE(192);
    XPA_Q4_LARGE(208);
    XPA_Q4_LARGE(224);
    XPA_Q4_LARGE(240);
    XPA_Q4_LARGE(256);
#undef XPA_Q4_SMALL
#undef XPA_Q4_LARGE
    default: return cudaErrorInvalidValue;
  }
}

namespace {

// Launches one of a rows kernel's two forms: four pieces a lane from 8 warps of
// them per SM on (8 heads x 128, write and read: 8192 tokens 32 us with four
// pieces, 41 with one; 64 tokens 6.6 against 3.9 us).
cudaError_t launch_rows(void (*one)(Q4RowsParams), void (*four)(Q4RowsParams),
                        const Q4RowsParams& a, cudaStream_t st) {
  Q4RowsParams p = a;
  const int pieces = a.Hkv * (a.D / 4);
  const long long steps = (long long)a.num_tokens * ((pieces + 31) / 32);
  const int P = steps >= 4LL * 8 * a.sms ? 4 : 1;
  p.warps_per_token = (pieces + 32 * P - 1) / (32 * P);
  const unsigned grid = (unsigned)(((long long)a.num_tokens * p.warps_per_token + 3) / 4);
  (P == 4 ? four : one)<<<grid, 128, 0, st>>>(p);
  return cudaGetLastError();
}

}  // namespace

// The head sizes that attention has swizzles of its own for have their address
// arithmetic folded here too (8192 tokens x 8 heads stored and read back, folded /
// not: D = 64 17.9 / 21.3 us, 128 32.0 / 38.2; 4096 tokens, 256 31.4 / 38.3).
cudaError_t launch_q4_write(const Q4RowsParams& a, cudaStream_t st) {
  switch (a.D) {
    case 64: return launch_rows(pa_q4_write_kernel<1, 64>, pa_q4_write_kernel<4, 64>, a, st);
    case 128: return launch_rows(pa_q4_write_kernel<1, 128>, pa_q4_write_kernel<4, 128>, a, st);
    case 256: return launch_rows(pa_q4_write_kernel<1, 256>, pa_q4_write_kernel<4, 256>, a, st);
    default: return launch_rows(pa_q4_write_kernel<1, 0>, pa_q4_write_kernel<4, 0>, a, st);
  }
}

cudaError_t launch_q4_read(const Q4RowsParams& a, cudaStream_t st) {
  switch (a.D) {
    case 64: return launch_rows(pa_q4_read_kernel<1, 64>, pa_q4_read_kernel<4, 64>, a, st);
    case 128: return launch_rows(pa_q4_read_kernel<1, 128>, pa_q4_read_kernel<4, 128>, a, st);
    case 256: return launch_rows(pa_q4_read_kernel<1, 256>, pa_q4_read_kernel<4, 256>, a, st);
    default: return launch_rows(pa_q4_read_kernel<1, 0>, pa_q4_read_kernel<4, 0>, a, st);
  }
}

}  // namespace xpa
