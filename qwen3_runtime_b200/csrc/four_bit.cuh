// How keys and values are held in 4 bits: the layout of a page and the rounding.
//
// A head of D channels (a multiple of 16, up to 256) is G equal groups: the fewest of at most 64 channels that are each made of whole
// words of 8.  A group is 4-bit numbers n, a scale s and a minimum z (bfloat16 both) and stands for z + n * s:
//   z = the largest bfloat16 that is not above the group's minimum, s = the smallest that is not below (maximum - z) / 15,
//   n = (x - z) / s rounded to nearest even and clamped to 0 .. 15 (s = 0: n = 0).
// Both are rounded outwards, so the 16 steps cover every value of the group and none is off by more than s / 2 (and a rounding of the sum).
// A group that holds something not finite, or whose spread is not, gets s = z = NaN: what attends to it is NaN, as it would be otherwise.
//
// pages [pages][kv_heads][record bytes], a record being, for page size ps,
//   key codes [ps][D / 2] | value codes [ps][D / 2] | key parameters [ps][G](s, z) | value parameters [ps][G](s, z)
// rounded up to 16 bytes.  A row of codes is D / 8 words of 32 bits: word i holds channels 8 (i / G) .. + 7 of group i % G, the first in
// its lowest 4 bits.  (The groups' words in turn: a lane of the attention kernel reads 16 bytes of a key and has words of every group, so
// that each matrix instruction stays within one group and the scale can be applied to its sums.)
#pragma once
#include "common.cuh"

__host__ __device__ __forceinline__ int q4_groups(int D) {
  const int words = D / 8;
  int g = (D + 63) / 64;
  while (words % g) ++g;
  return g;
}

struct Q4Page {  // byte offsets inside a record
  int half, par;  // bytes of a token's codes and of its parameters
  long values, kpar, vpar, record;
  __host__ __device__ __forceinline__ Q4Page(int D, int G, int ps) {
    half = D / 2;
    par = 4 * G;
    values = (long)ps * half;
    kpar = 2 * values;
    vpar = kpar + (long)ps * par;
    record = (vpar + (long)ps * par + 15) & ~15L;
  }
};

static inline bool q4_sizes_ok(int D, int ps) { return D >= 16 && D <= 256 && D % 16 == 0 && ps >= 1; }

struct Q4Scale {
  float s, z;
  uint32_t word;  // (s, z) as stored
};

// `lo`: NaN if the group holds one.  (Infinities end up in the scale.)
__device__ __forceinline__ Q4Scale q4_scale(float lo, float hi) {
  const bf16 z = __float2bfloat16_rd(lo);
  const bf16 s = __float2bfloat16_ru(__fdiv_rn(hi - __bfloat162float(z), 15.f));
  Q4Scale y;
  y.s = __bfloat162float(s);
  y.z = __bfloat162float(z);
  if (!(isfinite(y.s) && isfinite(y.z))) {
    y.s = y.z = NAN;
    y.word = 0x7FC07FC0u;
  } else {
    y.word = (uint32_t)__bfloat16_as_ushort(s) | ((uint32_t)__bfloat16_as_ushort(z) << 16);
  }
  return y;
}
// (x - z) / s for several x: with y = 1 / s rounded to nearest, q = x y and its remainder x - q s (exact in one fused step), q + remainder * y
// is the rounded quotient (Markstein, IBM J. Res. Dev. 34, 1990), as long as nothing leaves the range of normal numbers.
__device__ __forceinline__ uint32_t q4_word(const float (&x)[8], const Q4Scale& y) {
  uint32_t w = 0;
  if (!(y.s > 0.f)) return 0;  // one value all over, or NaN
  if (y.s > 0x1p-90f && y.s < 0x1p90f) {
    // a number between 0 and 15 plus 1.5 * 2^23 is rounded to whole numbers, half ways to even ones, and stands in the last bits (no
    // conversions, which are slow); 0x4b400000 in front of it is taken off once: its sum over the eight shifts
    const float inv = __frcp_rn(y.s);
    w = 0u - 0x3f400000u;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float d = x[e] - y.z, q = d * inv;
      const float n = fminf(fmaxf(fmaf(fmaf(-q, y.s, d), inv, q), 0.f), 15.f);
      w += __float_as_uint(__fadd_rn(n, 12582912.f)) << (4 * e);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) w |= (uint32_t)fminf(fmaxf(rintf(__fdiv_rn(x[e] - y.z, y.s)), 0.f), 15.f) << (4 * e);
  }
  return w;
}
__device__ __forceinline__ float q4_s(uint32_t word) { return __uint_as_float(word << 16); }
__device__ __forceinline__ float q4_z(uint32_t word) { return __uint_as_float(word & 0xFFFF0000u); }
