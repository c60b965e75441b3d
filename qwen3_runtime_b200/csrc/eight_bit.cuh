// How keys and values are held in 8 bits: the layout of a page and the rounding.
//
// pages [pages][kv_heads][record bytes], a record being, for head size D (a multiple of 16, up to 256) and page size ps,
//   key codes [ps][D] | value codes [ps][D] | key scale | value scale (float32, powers of two) | 8 bytes of nothing
// A code is an 8-bit float: sign, 4 bits of exponent, 3 of mantissa (e4m3: up to 448, steps of 2^-9 below 2^-6, 0x7F not a number), and
// stands for its value times the scale of its page.  A row's pieces of 16 channels stand in the order piece ^ (row & mask), mask 3 for D = 64,
// 7 for 128 and 256, 0 otherwise: rows that a warp reads side by side from shared memory then lie in different banks.
//
// Rounding.  R(x) is x rounded to 4 significant bits, half ways to even; what is not finite, or whose R is not, becomes 0x7F.  The scale is the
// least power of two, 2^-100 at least, with |R(x)| <= 448 scale for every finite x of the page's tokens.  A code stands for R(x) itself from
// 2^-6 scale on (448 / 2^-6: 15 binades), and below that for R(x) cut (towards zero) to a multiple of 2^-9 scale.
// Why cut and not round: cuts onto coarser and coarser grids compose, so a page whose tokens come one by one, and whose scale grows on the
// way, ends with the bytes that it would have had they come together, however prompts are cut into portions.  What is cut is less than 2^-9 of the
// scale, 2^-16 of the page's largest number.  Why powers of two: a code is then exact under a new scale except for that cut, and exact in bfloat16.
#pragma once
#include "common.cuh"

struct Q8Page {  // byte offsets inside a record
  long values, scales, record;
  __host__ __device__ __forceinline__ Q8Page(int D, int ps) : values((long)ps * D), scales(2 * values), record(scales + 16) {}
};
static inline bool q8_sizes_ok(int D, int ps) { return D >= 16 && D <= 256 && D % 16 == 0 && ps >= 1 && ps <= 0x7fffff; }
__host__ __device__ __forceinline__ constexpr int q8_mask(int D) { return D == 64 ? 3 : D == 128 || D == 256 ? 7 : 0; }
// byte of channel c in row `row`
__device__ __forceinline__ int q8_at(int c, int row, int mask) { return (((c >> 4) ^ (row & mask)) << 4) | (c & 15); }

constexpr uint32_t Q8_INFINITE = 0x7F800000u;
constexpr int Q8_LEAST = -100;  // exponent of the least scale

// Bits of |R(x)|; from Q8_INFINITE on: not a number.
__device__ __forceinline__ uint32_t q8_rounded(float x) {
  const uint32_t u = __float_as_uint(x) & 0x7FFFFFFFu;
  return (u + 0x7FFFFu + ((u >> 20) & 1u)) & 0xFFF00000u;
}
__device__ __forceinline__ uint32_t q8_finite(uint32_t rounded) { return rounded < Q8_INFINITE ? rounded : 0u; }
// Exponent of the scale for the largest bits: 448 = 1.75 * 2^8, and mantissas are 1, 1.125 .. 1.875: one more than the exponent less 8 only for
// 1.875, which a one added behind the mantissa carries over.
__device__ __forceinline__ int q8_exponent(uint32_t most) { return max(Q8_LEAST, (int)((most >> 20) + 1 >> 3) - 135); }
__device__ __forceinline__ float q8_power(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }  // -126 .. 127
__device__ __forceinline__ int q8_exponent_of(float scale) {  // of a scale as it is stored (of anything else: something in range)
  return min(120, max(Q8_LEAST, (int)((__float_as_uint(scale) >> 23) & 255u) - 127));
}
// The code of x under 2^-e = down.  2^-6, the least normal number of e4m3, times 2^-120 is float32's, so that float32's own bits, subnormal ones
// among them, shifted by the 20 surplus mantissa bits are the code, cut.
__device__ __forceinline__ uint32_t q8_code(float x, float down) {
  const uint32_t r = q8_rounded(x);
  const uint32_t c = r < Q8_INFINITE ? __float_as_uint(__fmul_rn(__fmul_rn(__uint_as_float(r), down), 0x1p-120f)) >> 20 : 0x7Fu;
  return r < Q8_INFINITE ? c | ((__float_as_uint(x) >> 24) & 0x80u) : c;
}
__device__ __forceinline__ uint32_t q8_word(const float* x, float down) {  // four of them
  return q8_code(x[0], down) | (q8_code(x[1], down) << 8) | (q8_code(x[2], down) << 16) | (q8_code(x[3], down) << 24);
}
// The bits of the largest |R(x)| of eight values, of which those that are not finite are left out, for maxima.  (fmaxf leaves NaN out.)
__device__ __forceinline__ uint32_t q8_most(const float (&x)[8]) {
  float most = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(x[e]));
  uint32_t r = q8_rounded(most);
  if (r >= Q8_INFINITE) {
    r = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) r = max(r, q8_finite(q8_rounded(x[e])));
  }
  return r;
}
// The codes of eight values.  Where none is infinite or rounds to it (from 1.9375 * 2^127 on, which lies within 448 scales of the largest scale alone) and
// none falls below the normal codes, where the cut is not a rounding, the conversion of the hardware (to nearest, half ways to even; NaN 0x7F) gives
// them, two at a time.
__device__ __forceinline__ uint2 q8_words(const float (&x)[8], float down) {
  float y[8], most = 0.f, least = 448.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    y[e] = __fmul_rn(x[e], down);
    most = fmaxf(most, fabsf(y[e]));
    least = fminf(least, fabsf(y[e]));
  }
  if (least >= 0x1p-6f && most <= 464.f && most < __fmul_rn(0x1.Fp127f, down)) {  // (464 lies halfway behind 448)
    uint32_t two[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      asm("{\n\t.reg .b16 t;\n\tcvt.rn.satfinite.e4m3x2.f32 t, %1, %2;\n\tcvt.u32.u16 %0, t;\n\t}" : "=r"(two[e]) : "f"(y[2 * e + 1]), "f"(y[2 * e]));
    return make_uint2(two[0] | (two[1] << 16), two[2] | (two[3] << 16));
  }
  return make_uint2(q8_word(x, down), q8_word(x + 4, down));
}
// Four codes under a scale that is larger: `shrink` is 2^-(growth).
__device__ __forceinline__ uint32_t q8_rescaled(uint32_t w, float shrink) {
  uint32_t y = 0;
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    const uint32_t c = (w >> (8 * b)) & 0x7Fu, sign = (w >> (8 * b)) & 0x80u;
    const uint32_t z = c == 0x7Fu ? c : __float_as_uint(__fmul_rn(__uint_as_float(c << 20), shrink)) >> 20;
    y |= (z | sign) << (8 * b);
  }
  return y;
}
// Two codes (the low one first) as two half-precision numbers, exactly.
__device__ __forceinline__ uint32_t q8_halves(uint32_t two) {
  uint32_t y;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(y) : "r"(two));
  return y;
}
// All four codes of a word: the low two, the high two.
__device__ __forceinline__ void q8_halves(uint32_t word, uint32_t& low, uint32_t& high) {
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\tcvt.rn.f16x2.e4m3x2 %1, hi;\n\t}" : "=r"(low), "=r"(high) : "r"(word));
}
__device__ __forceinline__ void q8_floats(uint32_t word, float (&v)[4]) {  // values of four codes, without the scale
  uint32_t y[2];
  q8_halves(word, y[0], y[1]);
#pragma unroll
  for (int h = 0; h < 2; ++h) asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.f32.f16 %0, lo;\n\tcvt.f32.f16 %1, hi;\n\t}" : "=f"(v[2 * h]), "=f"(v[2 * h + 1]) : "r"(y[h]));
}
