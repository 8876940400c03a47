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

}  // namespace xpa
