// Attention over prompts whose keys were cut into slices: what a slice leaves of a (token, head), and how the slices are joined.
#pragma once
#include "common.cuh"

// The maximum of a row that has seen nothing: a hidden key's score, -inf, weighs 2^(-inf - MINUS_BIG) = 0.
constexpr float MINUS_BIG = -3.402823466e+38f;

// The sum of a row that sees no key of a slice.  Its place says so and not its maximum: scores that are no number, or -inf, move none either, and what
// they make of the row has to reach its result.
constexpr float NOTHING_SEEN = -1.f;
// Whether a row that sees keys lo .. pos, and those in front of keep, sees one of the tiles j0 .. j1 - 1 of `size` keys, of which the ones from `firsts` on
// lie `skip` tiles further on.
__device__ __forceinline__ bool sees_tiles(int j0, int j1, int firsts, int skip, int size, int pos, int lo, int keep) {
  auto sees = [&](int a, int b) {  // one of keys a .. b - 1
    b = min(b, pos + 1);
    return a < b && (a < keep || lo < b);
  };
  return sees(j0 * size, min(j1, firsts) * size) || sees((max(j0, firsts) + skip) * size, (j1 + skip) * size);
}

struct PromptSlices {
  const float *mid_o, *mid_ml;  // [tokens][nq][splits][D], 2^-maximum times the results, and [tokens][nq][splits][2], maxima (base 2) and sums (or NOTHING_SEEN)
  bf16* out;
  const int* cu_seqlens;
  int num_seqs, least, tokens, nq, D, splits;  // sequences that bring fewer than `least` tokens are left alone
};

// A warp per (token of a sequence that counts, head): joins the slices in order.
static __global__ void __launch_bounds__(128) merge_prompts_kernel(PromptSlices a) {
  pdl_wait();
  pdl_launch_dependents();
  const long at = (long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (at >= (long)a.tokens * a.nq) return;
  const int t = (int)(at / a.nq);
  // the token's sequence: whether it counts
  bool mine = false;
  for (int base = 0; base < a.num_seqs; base += 32) {
    const int b = base + lane;
    const bool in = b < a.num_seqs && a.cu_seqlens[b] <= t && t < a.cu_seqlens[b + 1] && a.cu_seqlens[b + 1] - a.cu_seqlens[b] >= a.least;
    mine = mine || __any_sync(0xffffffffu, in);
  }
  if (!mine) return;
  float top = MINUS_BIG;
  for (int s = lane; s < a.splits; s += 32) top = fmaxf(top, a.mid_ml[2 * (at * a.splits + s)]);
  top = warp_max(top);
  float den = 0.f, y[8] = {};
  bool any = false;  // (a token without a key: zero)
  for (int s = 0; s < a.splits; ++s) {
    const float2 ml = *reinterpret_cast<const float2*>(a.mid_ml + 2 * (at * a.splits + s));
    if (ml.y == NOTHING_SEEN) continue;
    any = true;
    const float f = exp2f(ml.x - top);
    den += f * ml.y;
    const float* o = a.mid_o + (at * a.splits + s) * a.D;
#pragma unroll
    for (int c = 0; c < 8; ++c)
      if (lane + 32 * c < a.D) y[c] += f * o[lane + 32 * c];
  }
  const float inv = any ? 1.f / den : 0.f;
#pragma unroll
  for (int c = 0; c < 8; ++c)
    if (lane + 32 * c < a.D) a.out[at * a.D + lane + 32 * c] = __float2bfloat16_rn(y[c] * inv);
}

static inline cudaError_t merge_prompts(const PromptSlices& a, cudaStream_t stream) {
  return launch_pdl(merge_prompts_kernel, dim3((unsigned)(((long)a.tokens * a.nq + 3) / 4)), dim3(128), 0, stream, a);
}
