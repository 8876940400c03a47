// pa_q4.cuh — the 4-bit KV format: tile layout, encoding and decoding.
//
// An element is an E2M1 code c (sign, 2 exponent bits, 1 mantissa bit:
// 0, 0.5, 1, 1.5, 2, 3, 4, 6), every 16 channels of a token's row share one
// E4M3 scale s, and the pool has one fp32 scale ps: value = c * s * ps.
//   t = x / ps (fp32; NaN counts as 0),
//   s = E4M3(max |t| / 6), nearest even, at most 448,
//   c = E2M1(t / s), nearest even, at most 6; 0 when s is 0.
// c * s has at most 2 + 4 significand bits and lies in [2^-10, 2688], so it is
// exact in fp16: attention multiplies exact operands and adds in fp32. Neither
// division can hide a tie: s and the E2M1 midpoints have 4 bits, so a 24-bit
// t that is not exactly midpoint * s is at least one unit in its last place
// away, which the quotient's rounding to fp32 keeps on its side.
//
// 16 tokens of one KV head are one tile of 9 * D bytes (D = head size, a
// multiple of 16; 4.5 bits per element):
//   K: 16 rows of D / 2 bytes, then scales [16 tokens][D / 16].
//      A row is four chunks t = 0..3 of D / 16 two-byte units; unit j of
//      chunk t holds channels 16 j + 4 t .. + 3 (low nibble first): lane t of
//      an mma quad reads its share of a row as one contiguous piece.
//   V: 16 rows of D / 2 bytes in channel order, then scales [D / 16][16
//      tokens]: a lane reads the scales of its four tokens as one word.
// Every token's row is its own bytes, so tokens are written independently.
#pragma once

#include <cfloat>

#include "pa_device.cuh"

namespace xpa {

// ── byte offsets inside a tile ──────────────────────────────────────────
// The 8 channels [8 w, 8 w + 8) of token `tok`: two 2-byte K units (at
// q4_k_off and D / 8 bytes further on, the next chunk), or 4 V bytes.
__device__ __forceinline__ int q4_k_off(int D, int tok, int w) {
  return tok * (D / 2) + (w & 1) * (D / 4) + (w >> 1) * 2;
}
__device__ __forceinline__ int q4_v_off(int D, int tok, int w) { return tok * (D / 2) + w * 4; }
__device__ __forceinline__ int q4_k_scale_off(int D, int tok, int grp) {
  return 8 * D + tok * (D / 16) + grp;
}
__device__ __forceinline__ int q4_v_scale_off(int D, int tok, int grp) {
  return 8 * D + grp * 16 + tok;
}

// ── decoding ────────────────────────────────────────────────────────────
// The eight codes of a word -> four fp16x2 (byte i: low nibble in the low half).
// Callers use outputs of both 16-bit halves of the word (0 or 1, and 2 or 3): where
// those of one half alone are used, what ptxas 12.9.86 makes of this gives wrong
// values. Tried on a B200 over all 65536 values of a half: outputs {0, 1}, {2, 3}
// and each by itself are wrong, {0, 2}, {1, 3}, any three and all four right.
// Bytes taken apart by way of 16-bit registers, or one to a statement, are wrong at
// output 2 even with all four in use.
__device__ __forceinline__ void q4x8_to_h2(uint32_t w, uint32_t (&h)[4]) {
  asm("{\n\t.reg .b8 p, q, r, s;\n\tmov.b32 {p, q, r, s}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, p;\n\tcvt.rn.f16x2.e2m1x2 %1, q;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, r;\n\tcvt.rn.f16x2.e2m1x2 %3, s;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
}
__device__ __forceinline__ uint32_t h2_mul(uint32_t a, uint32_t b) {
  const __half2 r =
      __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// a times the low / the high half of s (the multiply selects it: no extra step).
__device__ __forceinline__ uint32_t h2_mul_low(uint32_t a, uint32_t s) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a),
                            __low2half2(*reinterpret_cast<const __half2*>(&s)));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t h2_mul_high(uint32_t a, uint32_t s) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a),
                            __high2half2(*reinterpret_cast<const __half2*>(&s)));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// ── encoding ────────────────────────────────────────────────────────────
// x / y rounded to nearest, from r = 1 / y rounded to nearest: the quotient
// estimate's residual is exact in one fused step and corrects it (Markstein,
// IBM J. Res. Dev. 34, 1990; y > 0, its significand not all ones, nothing near
// the range's ends). The sign of a zero is lost.
__device__ __forceinline__ float div_by(float x, float y, float r) {
  const float q = x * r;
  return fmaf(fmaf(-q, y, x), r, q);
}

// The E4M3 scale of a group whose largest |t| is amax.
__device__ __forceinline__ uint32_t q4_scale(float amax) {
  return float2_to_fp8x2<kKvE4M3>(div_by(amax, 6.f, 1.f / 6.f), 0.f) & 0xffu;
}
// t / s as two E2M1 codes, a in the low nibble.
__device__ __forceinline__ uint32_t q4_pair(float a, float b) {
  uint32_t r;
  asm("{\n\t.reg .b8 t;\n\t.reg .b16 h;\n\tcvt.rn.satfinite.e2m1x2.f32 t, %1, %2;\n\t"
      "mov.b16 h, {t, 0};\n\tcvt.u32.u16 %0, h;\n\t}"
      : "=r"(r)
      : "f"(b), "f"(a));
  return r;
}

// ── asynchronous copies ─────────────────────────────────────────────────
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// ── partitions and their merge over a CTA's warps ───────────────────────
constexpr int kGridY = 32768;
// A warp's reference point before any score above -inf: below every score, and
// finite, so that a score's distance from it is never NaN.
constexpr float kNoScore = -FLT_MAX;

// Partition blockIdx.x of row (sequence, KV head).
__device__ __forceinline__ ItemKind part_item(const Params& p, int row, Item& it) {
  it.part = blockIdx.x;
  it.b = row / p.Hkv;
  it.kvh = row - it.b * p.Hkv;
  int L = __ldg(p.seq_lens + it.b);
  const long long cap = (long long)p.max_blocks * p.block_size;
  if (L < 0 || L > cap) {
    if (it.part == 0 && it.kvh == 0 && threadIdx.x == 0) raise_status(p, kDevSeqClamped);
    L = L < 0 ? 0 : (int)cap;
  }
  it.L = L;
  it.slot0 = 0;
  const long long part_tokens = (long long)p.part_pages * p.block_size;
  it.direct = L <= part_tokens;
  if (L == 0) return it.part == 0 ? kItemZero : kItemNone;
  if (it.part * part_tokens >= L) return kItemNone;
  it.page_begin = it.part * p.part_pages;
  it.page_end = it.page_begin + p.part_pages;
  return kItemWork;
}

// Merges the warps' states and stores the item: the output itself, or a partial.
// A row whose weights' sum is not above 0 (nothing valid, or a NaN score) is 0,
// as in every other kernel here and however the row is split.
// so: [NW][HEADS][ROW] sums of weights times V; sml: [NW][HEADS] reference point
// in units of q . k, p.ml_unit of the exp2 domain each (-inf: no score above
// -inf), and sum of the weights. D is a multiple of 16.
template <int NW, int HEADS, int ROW>
__device__ __forceinline__ void merge_warps(const Params& p, const Item& it, const float* so,
                                            const float* sml, long long row0, int nh, int D) {
  const int nc = D / 8;
  for (int idx = threadIdx.x; idx < nh * nc; idx += NW * 32) {
    const int head = idx / nc, d0 = (idx - head * nc) * 8;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, sml[(w * HEADS + head) * 2]);
    float num[8] = {}, den = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float mw = sml[(w * HEADS + head) * 2];
      // a warp without a score above -inf holds zeros, or NaN sums to pass on
      const float wt = mw == M ? 1.f : ex2((mw - M) * p.ml_unit);
      den = fmaf(wt, sml[(w * HEADS + head) * 2 + 1], den);
      const float4* src =
          reinterpret_cast<const float4*>(so + (size_t)(w * HEADS + head) * ROW + d0);
      const float4 a = src[0], b = src[1];
      num[0] = fmaf(wt, a.x, num[0]);
      num[1] = fmaf(wt, a.y, num[1]);
      num[2] = fmaf(wt, a.z, num[2]);
      num[3] = fmaf(wt, a.w, num[3]);
      num[4] = fmaf(wt, b.x, num[4]);
      num[5] = fmaf(wt, b.y, num[5]);
      num[6] = fmaf(wt, b.z, num[6]);
      num[7] = fmaf(wt, b.w, num[7]);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) num[k] *= p.v_scale;
    if (it.direct) {
#pragma unroll
      for (int k = 0; k < 8; ++k) num[k] = den > 0.f ? num[k] / den : 0.f;
      if (p.vec8) {
        store_out8<__half>(p, row0 + head, d0, num);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) store_out<__half>(p, row0 + head, d0 + k, num[k]);
      }
    } else {
      const long long pr = (row0 + head) * p.slots + it.slot0 + it.part;
      // D is a multiple of 16: the partials' rows start on 16-byte boundaries
      float4* dst = reinterpret_cast<float4*>(p.part_o + pr * D + d0);
      dst[0] = make_float4(num[0], num[1], num[2], num[3]);
      dst[1] = make_float4(num[4], num[5], num[6], num[7]);
      // the merge of partials leaves out one without a score above -inf: NaN
      // sums are not to be lost with it
      if (d0 == 0)
        reinterpret_cast<float2*>(p.part_ml)[pr] = make_float2(isnan(den) ? 0.f : M, den);
    }
  }
}

}  // namespace xpa
