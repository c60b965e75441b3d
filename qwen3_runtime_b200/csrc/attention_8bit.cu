// Attention over a cache in 8 bits (layout: eight_bit.cuh), all keys or a window of them and the sequence's first ones: decode attention in
// bfloat16, and a general form.
//
// A code (e4m3) is exact in half precision, so codes become operands of mma.sync by one conversion for two of them, and what a page's tokens
// share, the scales, is applied to sums:
//   scores   K (16 keys) x Q^T (8 queries) on mma.sync m16n8k16.  A query row is multiplied by a power of two that brings its largest value to
//            2^14 .. 2^15 (bfloat16's 8 bits fit half precision's 11; values 2^-28 of the largest and less lose bits, by 2^-40 of it at most):
//              score = (key scale * 2^-S) sum_c q_c 2^S code_c
//   results  V^T (16 channels) x P^T, P^T being the score tile's weights, transposed by movmatrix.  Weights carry the values' scale along and are
//            rounded to half precision, 2^-12 of themselves where bfloat16 would give 2^-9.  That needs them in range whatever the scales are:
//              w_t = 2^(x_t + log2(value scale) - M + 6),  M following the largest x_t + log2(value scale), which is the largest contribution,
//            while the sum of the softmax follows the largest x_t, m, as ever.  Within a page w_t is 2^(x_t - m) times one number per query.
// Keys as the product's 16 rows and the kv head's queries as its 8 columns: a group of up to 8 query heads wastes nothing.
#include <type_traits>

#include "async_tiles.cuh"
#include "eight_bit.cuh"
#include "mma_tiles.cuh"

#define Q3_ERR_WAIT_8BIT 22

namespace {

// The maximum of a row that has seen nothing: no score lies below it, and a hidden key's, -inf, weighs 2^(-inf - MINUS_BIG) = 0.
constexpr float MINUS_BIG = -3.402823466e+38f;

__device__ __forceinline__ uint32_t transposed(uint32_t a) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(a));
  return y;
}
__device__ __forceinline__ float exp2_fast(float x) {  // 2^x to 2 units in the last place; below 2^-126 zero
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  uint32_t y;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
  return y;
}
__device__ __forceinline__ void mma_half(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float log2_of(float scale) { return (float)((int)(__float_as_uint(scale) >> 23) - 127); }  // of a power of two

// What a warp's lanes hold of 16 keys: rows lane / 4 and lane / 4 + 8, and of each row the pieces of 16 channels that lane % 4 takes; of 16
// values the pieces that lane / 4 takes (D = 64: half a piece), of tokens 2 (lane % 4), + 1, + 8, + 9.
template <int D> struct Head {
  static constexpr int PIECES = D / 64;           // of a row, by lane
  static constexpr int MASK = q8_mask(D);
  static constexpr int TILES = D == 256 ? 1 : 2;  // of 16 keys that a warp takes at a time: what is asked and counted once for both costs half
  static __device__ __forceinline__ int key_piece(int j, int l) { return D == 64 ? l : D == 128 ? 2 * l + j : 2 * l + (j & 1) + 8 * (j >> 1); }
};

// The queries' side of the scores: B fragments (column lane / 4, the channels of this lane's pieces in order), and what the sums are to be
// multiplied by for columns 2 (lane % 4) and + 1: 2^-S times the scores' scale.
template <int D> __device__ __forceinline__ void fetch_query(uint4 (&raw)[Head<D>::PIECES][2], const bf16* row, int lane) {
#pragma unroll
  for (int j = 0; j < Head<D>::PIECES; ++j)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      raw[j][e] = make_uint4(0, 0, 0, 0);
      if (row) raw[j][e] = *reinterpret_cast<const uint4*>(row + 16 * Head<D>::key_piece(j, lane & 3) + 8 * e);
    }
}
template <int D> __device__ __forceinline__ void take_query(uint32_t (&b)[Head<D>::PIECES][4][2], float (&undo)[2],
                                                            const uint4 (&raw)[Head<D>::PIECES][2], float scale_log2, int lane) {
  using H = Head<D>;
  float top = 0.f;
#pragma unroll
  for (int j = 0; j < H::PIECES; ++j)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t word[4] = {raw[j][e].x, raw[j][e].y, raw[j][e].z, raw[j][e].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) top = fmaxf(top, fmaxf(fabsf(__uint_as_float(word[i] << 16)), fabsf(__uint_as_float(word[i] & 0xFFFF0000u))));
    }
#pragma unroll
  for (int d = 1; d < 4; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  const int S = min(126, 141 - (int)(__float_as_uint(top) >> 23));  // (an infinite row stays infinite)
  const float up = q8_power(S);
#pragma unroll
  for (int j = 0; j < H::PIECES; ++j)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t word[4] = {raw[j][e].x, raw[j][e].y, raw[j][e].z, raw[j][e].w};
#pragma unroll
      for (int i = 0; i < 4; ++i)  // a piece's word w is channels 4w .. 4w + 3: the first pair meets the low half of the operand
        b[j][2 * e + i / 2][i & 1] = pack_half(__uint_as_float(word[i] << 16) * up, __uint_as_float(word[i] & 0xFFFF0000u) * up);
    }
  const float back = scale_log2 * q8_power(-S);
#pragma unroll
  for (int c = 0; c < 2; ++c) undo[c] = __shfl_sync(0xffffffffu, back, 4 * (2 * (lane & 3) + c));
}

// ---- decode attention -------------------------------------------------------------------------------------------------------------
// Grid (slice, kv head, sequence): a block takes one slice of one sequence's keys for one kv head and the query heads that read it; each of
// its 4 warps takes every fourth step of keys, with a ring of its own and a softmax of its own (no barrier in the loop), and the warps are
// joined at the end.  Where the launch leaves SMs idle, up to 16 slices are the blocks of a cluster, which read each other's results in shared
// memory; else they go through global memory and a second kernel.
//   BULK   page sizes that are a multiple of 16: a tile is 16 tokens of one page, brought by one bulk copy (16 tokens a page) or three
//          that a lane asks for, and has one scale.  Rows behind the slice's end come along and are masked.
//   else   any page size: cp.async token by token, each with its scales; what is not there is zero.
// What bounds it is reading the codes: eight tokens behind 17,000 to 32,768, 64 heads over 8 of 128, 81 to 85 us over other pages each time, 5.8 to 6.0 TB/s, 78
// over the same two sets again and again (pages of 16 bits 162); issue 0.34 a clock, a warp waits for results of mma.sync and for copies about alike.  Smaller launches lose to the blocks' beginnings and ends: eight behind 4,096, 32
// heads over 8, 16.5 us for 10 of reading; one behind 512, 5 us, a chain of lookups, copies and a join.  No more, measured at both: rings of 2 or 4 stages, 1
// or 4 tiles a step, 3 blocks an SM, two accumulators for the scores, values read before the softmax.  Slower: all pairs' steps behind one another, as many for
// each warp of a launch that fills the device, its ring filled across the pairs' borders, the parts joined by a second kernel: 88, 22.5, and 48 sequences of
// 65 to 3,966 44 for 42 -- a warp's every page is another place to read from, 1,184 of them, and the second kernel has many parts to join.
constexpr int WARPS = 4;
constexpr int THREADS = 32 * WARPS;
constexpr int STEP = 16;  // keys of a tile
constexpr int STAGES = 3;
constexpr int MOST_CLUSTER = 16;

// A step's barrier, when the first look finds its bytes still on their way; called by whole warps, which leave it of one mind.  Bounded:
// false after the limit.  The warp then asks for nothing more (the barrier has its arrivals, and must not be given others), waits for what
// it has in flight (wait_for_copies) and goes on to the block's end; the error word says that the result is invalid.
__device__ __noinline__ bool wait_for_tiles(uint32_t bar, uint32_t parity, int* error_word) {
  const long long start = clock64();
  while (!__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) {
    if (__any_sync(0xffffffffu, clock64() - start > Q3_WAIT_LIMIT_CYCLES)) {
      atomicExch(error_word, Q3_ERR_WAIT_8BIT);
      return false;
    }
  }
  return true;
}
// The steps that are asked for and not yet taken, from `stage` on (bounded).
__device__ __noinline__ void wait_for_copies(uint32_t bars, int stage, uint32_t parity) {
  for (int i = 0; i < STAGES - 1; ++i) {
    mbar_wait_drain(bars + 8 * stage, parity);
    if (++stage == STAGES) stage = 0, parity ^= 1;
  }
}

struct Decode {
  const bf16* q;
  int q_stride;
  const unsigned char* pages;
  int num_pages;
  const int *block_table, *kv_lens, *cu_seqlens, *seq_list;
  int max_pages;
  bf16* out;
  float *mid_o, *mid_lse;
  int nq, nkv, ps, window, keep_first, splits, max_len;
  float scale_log2;
  const int* longest;
  int* error_word;
};

// What a sequence's newest token sees: keys lo .. kv_len - 1, and keys 0 .. keep_first - 1.  Both beginnings are rounded to tiles (BULK: a tile
// lies in one page): places count the tiles of the first ones, `first` keys of them, and then those from lo on; key = place + gap from `first`
// on.  Slices are cut by places.  Places per slice, the same for all sequences of the launch: the longest sequence's over the slices
// asked for, in whole rounds of the block.  A shorter sequence has fewer slices.
struct Seen {
  int kv_len, lo, first, gap, places;
  __device__ __forceinline__ Seen(const Decode& a, int seq) {
    kv_len = min(a.kv_lens[seq], a.max_len);
    lo = a.window > 0 ? max(0, kv_len - a.window) : 0;
    const int tiles = (a.keep_first + STEP - 1) & ~(STEP - 1), begins = lo & ~(STEP - 1);
    first = min(tiles, begins), gap = begins - first;
    places = max(0, kv_len - gap);
  }
};
template <int ROUND> struct Slice : Seen {
  int begin, end, per;
  __device__ __forceinline__ Slice(const Decode& a, int seq, int split) : Seen(a, seq) {
    const int tiles = (a.keep_first + STEP - 1) & ~(STEP - 1);
    int longest = a.longest ? min(*a.longest, a.max_len) : a.max_len;
    if (a.window > 0) longest = min(longest, a.window + STEP - 1 + tiles);
    per = max(ROUND, ((longest + a.splits - 1) / a.splits + ROUND - 1) / ROUND * ROUND);
    begin = split * per;
    end = min(places, begin + per);
  }
  __device__ __forceinline__ int count(const Decode& a) const { return min(a.splits, max(0, places + per - 1) / per); }  // slices that have keys
};

// What a warp holds of the queries of one kv head and sequence, and of their attention so far.
template <int D, int NT, bool BULK> struct Taker {
  using H = Head<D>;
  static constexpr int TILES = H::TILES, MT = D / 16, VALUES = STEP * D, SCALES = 2 * VALUES, TILE = SCALES + (BULK ? 16 : 8 * STEP);
  int lane, r, l, k_row, k_swap;
  uint32_t q[NT][H::PIECES][4][2];
  float undo[NT][2];
  // o: 2^(6 - M) times the results so far; sum: of 2^(x - m), this lane's share.  m and M are the same in all lanes of a column.
  float o[NT][MT][4], m[NT][2], M[NT][2], sum[NT][2];
  __device__ __forceinline__ Taker(int lane) : lane(lane), r(lane >> 2), l(lane & 3), k_row((lane >> 2) * D), k_swap((lane >> 2) & H::MASK) {}
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n][0] = m[n][1] = M[n][0] = M[n][1] = MINUS_BIG;
      sum[n][0] = sum[n][1] = 0.f;
#pragma unroll
      for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][j][e] = 0.f;
    }
  }
  // The keys of one step, at places base .. of which those in front of `end` count.  WHOLE: every one of them is visible.
  template <bool WHOLE> __device__ __forceinline__ void take(const Decode& a, const unsigned char* st, int base, const Seen& sl, int end) {
    float x[TILES][NT][4], up[TILES][2];  // up: log2 of the values' scales of rows r and r + 8
    bool in[TILES][2];
    int key0[TILES];
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      const unsigned char* tile = st + t * TILE;
      float acc[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
#pragma unroll
      for (int j = 0; j < H::PIECES; ++j) {
        const int piece = 16 * (H::key_piece(j, l) ^ k_swap);
        const uint4 w0 = *reinterpret_cast<const uint4*>(tile + k_row + piece), w1 = *reinterpret_cast<const uint4*>(tile + k_row + 8 * D + piece);
        const uint32_t k0[4] = {w0.x, w0.y, w0.z, w0.w}, k1[4] = {w1.x, w1.y, w1.z, w1.w};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          uint32_t f[4];
          q8_halves(k0[w], f[0], f[2]);
          q8_halves(k1[w], f[1], f[3]);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_half(acc[n], f, q[n][j][w][0], q[n][j][w][1]);
        }
      }
      float2 s0, s1;  // scales of keys and values, of rows r and r + 8
      if (BULK) {
        s0 = s1 = *reinterpret_cast<const float2*>(tile + SCALES);
      } else {
        s0 = *reinterpret_cast<const float2*>(tile + SCALES + 8 * r), s1 = *reinterpret_cast<const float2*>(tile + SCALES + 8 * (r + 8));
      }
      in[t][0] = in[t][1] = true;
      if (!WHOLE) {
        const int place = base + t * STEP;
        key0[t] = place + (place >= sl.first ? sl.gap : 0);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int key = key0[t] + r + 8 * half;
          in[t][half] = key < sl.kv_len && place + r + 8 * half < end && (key >= sl.lo || key < a.keep_first);
        }
      }
      // (rows that are nobody's may have anything for a scale)
      up[t][0] = WHOLE || in[t][0] ? log2_of(s0.y) : 0.f;
      up[t][1] = BULK && WHOLE ? up[t][0] : WHOLE || in[t][1] ? log2_of(s1.y) : 0.f;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float(&y)[4] = x[t][n];
#pragma unroll
        for (int c = 0; c < 2; ++c) {  // (a product beyond float32's range would make NaN of a sum of zero)
          const float f0 = fminf(s0.x * undo[n][c], 3e38f), f1 = BULK ? f0 : fminf(s1.x * undo[n][c], 3e38f);
          y[c] = acc[n][c] * f0, y[c + 2] = acc[n][c + 2] * f1;
          if (!WHOLE) {
            y[c] = in[t][0] ? y[c] : -INFINITY;
            y[c + 2] = in[t][1] ? y[c + 2] : -INFINITY;
          }
        }
      }
    }
    // Both maxima move only when they would be passed by a factor of 2^8 (a weight is 2^8 at most, which float32 sums do not mind, and 2^14 with
    // the 6 that it is lifted by in half precision, whose numbers end at 2^16); hardly ever after the first tiles.
    float top[NT][2], high[NT][2];
    bool far = false;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        top[n][c] = high[n][c] = -INFINITY;
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
          const float both = fmaxf(x[t][n][c], x[t][n][c + 2]);
          top[n][c] = fmaxf(top[n][c], both);
          high[n][c] = fmaxf(high[n][c], BULK && WHOLE ? both + up[t][0] : fmaxf(x[t][n][c] + up[t][0], x[t][n][c + 2] + up[t][1]));
        }
        far = far || top[n][c] > m[n][c] + 8.f || high[n][c] > M[n][c] + 8.f;
      }
    if (__any_sync(0xffffffffu, far)) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float now = fmaxf(m[n][c], top[n][c]), now_high = fmaxf(M[n][c], high[n][c]);
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) {
            now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, d));
            now_high = fmaxf(now_high, __shfl_xor_sync(0xffffffffu, now_high, d));
          }
          sum[n][c] *= exp2_fast(m[n][c] - now);
          const float f = exp2_fast(M[n][c] - now_high);
          m[n][c] = now, M[n][c] = now_high;
#pragma unroll
          for (int j = 0; j < MT; ++j) o[n][j][c] *= f, o[n][j][c + 2] *= f;
        }
    }
    uint32_t w[TILES][NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int t = 0; t < TILES; ++t) {
        float(&y)[4] = x[t][n];
        float z[4];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          y[c] = exp2_fast(y[c] - m[n][c]), y[c + 2] = exp2_fast(y[c + 2] - m[n][c]);
          sum[n][c] += y[c] + y[c + 2];
          // (a factor beyond 2^126 meets weights that are next to nothing)
          const float lift = (m[n][c] - M[n][c]) + 6.f, f0 = exp2_fast(fminf(up[t][0] + lift, 126.f));
          z[c] = y[c] * f0, z[c + 2] = y[c + 2] * (BULK && WHOLE ? f0 : exp2_fast(fminf(up[t][1] + lift, 126.f)));
        }
        w[t][n][0] = transposed(pack_half(z[0], z[1]));
        w[t][n][1] = transposed(pack_half(z[2], z[3]));
      }
    // ---- results: of each tile the tokens 2l, 2l + 1, 2l + 8, 2l + 9
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      const unsigned char* tile = st + t * TILE + VALUES;
      constexpr int WORDS = D / 32;  // of a token's values that a lane takes
      uint32_t v[4][WORDS];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = 2 * l + (e & 1) + 8 * (e >> 1);
        const unsigned char* from = tile + row * D;
        if constexpr (D == 64) {
          *reinterpret_cast<uint2*>(&v[e][0]) = *reinterpret_cast<const uint2*>(from + 16 * ((r >> 1) ^ (row & H::MASK)) + 8 * (r & 1));
        } else {
#pragma unroll
          for (int i = 0; i < WORDS / 4; ++i)
            *reinterpret_cast<uint4*>(&v[e][4 * i]) = *reinterpret_cast<const uint4*>(from + 16 * ((r + 8 * i) ^ (row & H::MASK)));
        }
        if (!WHOLE) {  // rows that are hidden may hold what is no number
          const int key = key0[t] + row, place = base + t * STEP + row;
          const bool seen = key < sl.kv_len && place < end && (key >= sl.lo || key < a.keep_first);
#pragma unroll
          for (int i = 0; i < WORDS; ++i) v[e][i] = seen ? v[e][i] : 0u;
        }
      }
#pragma unroll
      for (int i = 0; i < WORDS; ++i) {
        const uint32_t a0 = __byte_perm(v[0][i], v[1][i], 0x5140), a1 = __byte_perm(v[0][i], v[1][i], 0x7362);
        const uint32_t b0 = __byte_perm(v[2][i], v[3][i], 0x5140), b1 = __byte_perm(v[2][i], v[3][i], 0x7362);
        uint32_t f[4], g[4];
        q8_halves(a0, f[0], f[1]);
        q8_halves(b0, f[2], f[3]);
        q8_halves(a1, g[0], g[1]);
        q8_halves(b1, g[2], g[3]);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma_half(o[n][2 * i], f, w[t][n][0], w[t][n][1]);
          mma_half(o[n][2 * i + 1], g, w[t][n][0], w[t][n][1]);
        }
      }
    }
  }
  // column c of tile n, from here, as its sum (all lanes of a column) and, by `put`, four channels at a time of 2^-m times the results
  template <typename Put> __device__ __forceinline__ float finished(int n, int c, Put put) const {
    float total = sum[n][c];
#pragma unroll
    for (int d = 4; d < 32; d <<= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
    const float back = exp2_fast((M[n][c] - m[n][c]) - 6.f);
#pragma unroll
    for (int i = 0; i < MT / 2; ++i) {  // channels 4 i .. 4 i + 3 of this lane's, which are pieces r and r + 8 of the head (D = 64: half of one)
      const int channel = D == 64 ? 8 * r + 4 * i : 16 * (r + 8 * (i / 4)) + 4 * (i % 4);
      put(channel, make_float4(o[n][2 * i][c] * back, o[n][2 * i][c + 2] * back, o[n][2 * i + 1][c] * back, o[n][2 * i + 1][c + 2] * back));
    }
    return total;
  }
};

// The copies of a step into a stage, by a warp: `rec` and `at_row` are of the token that this lane has looked up (BULK: the first lanes, a tile's first token),
// `valid` that there is one.
template <int D, bool BULK>
__device__ __forceinline__ void copy_step(const Decode& a, const Q8Page& L, uint32_t dst, uint32_t stage_at, uint32_t bar, const unsigned char* rec, int at_row,
                                          bool valid, int lane) {
  using H = Head<D>;
  constexpr int TILES = H::TILES, VALUES = STEP * D, SCALES = 2 * VALUES, TILE = SCALES + (BULK ? 16 : 8 * STEP);
  if (BULK) {  // each lane arrives once, with the bytes that it asks for
    if (lane >= TILES) return;
    mbar_expect_tx(bar, valid ? TILE : 0);
#ifdef Q3_TEST_WITHHOLD_A_BOX  // (a test build leaves the second tiles out: the stages never fill, a wait runs out)
    if (valid && lane == 0) {
#else
    if (valid) {
#endif
      if (a.ps == STEP) {
        bulk_copy(dst, rec, TILE, bar);
      } else {
        bulk_copy(dst, rec + (long)at_row * D, VALUES, bar);
        bulk_copy(dst + VALUES, rec + L.values + (long)at_row * D, VALUES, bar);
        bulk_copy(dst + SCALES, rec + L.scales, 16, bar);
      }
    }
  } else {
    // Neighbouring lanes bring neighbouring pieces of a row (every lane a row of its own: 32 lines a copy, half the speed).  A row's address comes from
    // the lane that looked it up, with how its pieces are ordered (by the row in the page there, by the tile's here) and whether it exists below it.
    constexpr int PIECES = D / 16, ROWS = 32 / PIECES;
    const unsigned long long mine = reinterpret_cast<unsigned long long>(rec + (valid ? (long)at_row * D : 0)) | (uint32_t)((at_row ^ lane) & H::MASK) | (valid ? 8u : 0u);
#pragma unroll
    for (int i = 0; i < STEP * TILES / ROWS; ++i) {
      const int token = i * ROWS + lane / PIECES, piece = lane % PIECES;
      const unsigned long long from = __shfl_sync(0xffffffffu, mine, token);
      const unsigned char* src = reinterpret_cast<const unsigned char*>(from & ~15ull) + 16 * (piece ^ ((int)from & 7));
      const uint32_t at_tile = stage_at + token / STEP * TILE + token % STEP * D + 16 * piece;
      cp_async16(at_tile, src, from & 8 ? 16 : 0);
      cp_async16(at_tile + VALUES, src + L.values, from & 8 ? 16 : 0);
    }
    if (lane < STEP * TILES)
      asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;\n" ::"r"(dst + SCALES + 8 * (lane & (STEP - 1))), "l"(rec + L.scales), "r"(valid ? 8 : 0));
    cp_async_commit();
  }
}

template <int D, int NT> constexpr int decode_blocks() { return D == 64 ? 4 : 2; }

template <int D, int NT, bool BULK, bool CLUSTER>
__global__ void __launch_bounds__(THREADS, decode_blocks<D, NT>()) decode_8bit_kernel(Decode a) {
  using H = Head<D>;
  constexpr int TILES = H::TILES, ROUND = STEP * TILES * WARPS, QS = 8 * NT, PITCH = D + 4;
  constexpr int VALUES = STEP * D, SCALES = 2 * VALUES;       // of a tile: keys, values, scales (one pair, or a pair of rows)
  constexpr int TILE = SCALES + (BULK ? 16 : 8 * STEP), STAGE = TILES * TILE;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ __align__(8) uint64_t bars[WARPS][STAGES];
  const int split = blockIdx.x, kvh = blockIdx.y, slot = blockIdx.z;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r = lane >> 2, l = lane & 3;
  const int R = a.nq / a.nkv;
  if (BULK) {
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < STAGES; ++i) mbar_init(smem_addr(&bars[warp][i]), TILES);
      mbar_init_fence();
    }
    __syncwarp();
  }
  pdl_wait();
  const int seq = a.seq_list ? a.seq_list[slot] : slot;
  const int tok = a.cu_seqlens[seq];
  const Slice<ROUND> sl(a, seq, split);
  const int begin = sl.begin, end = sl.end;
  const long out_row = (long)tok * a.nq + kvh * R;
  if (!CLUSTER && begin >= end) {
    pdl_launch_dependents();
    if (a.splits == 1)  // no key at all
      for (int i = tid; i < R * D; i += THREADS) a.out[out_row * D + i] = __float2bfloat16_rn(0.f);
    return;
  }
  const Q8Page L(D, a.ps);
  const int* bt = a.block_table + (long)seq * a.max_pages;
  unsigned char* ring = smem + warp * STAGES * STAGE;

  // The token that this lane copies (BULK: the first lanes, a tile's first), as page of the sequence and row, moved on by a round at a time and
  // over the gap once.  Its page is looked up a step before the copy, whose address waits for it.
  const unsigned char* head = a.pages + kvh * L.record;
  const uint32_t page_bytes = (uint32_t)(a.nkv * L.record);
  int at = begin + warp * STEP * TILES + (BULK ? STEP * lane : lane);
  bool behind = at >= sl.first;  // of the gap
  int at_page = (at + (behind ? sl.gap : 0)) / a.ps, at_row = at + (behind ? sl.gap : 0) - at_page * a.ps;
  const int go_pages = ROUND / a.ps, go_rows = ROUND - go_pages * a.ps;
  auto look_up = [&]() { return lane < (BULK ? TILES : STEP * TILES) && at < end ? bt[at_page] : -1; };
  int page = look_up();
  const uint32_t ring_at = smem_addr(ring) + (BULK ? lane : lane / STEP) * TILE, bar_at = smem_addr(&bars[warp][0]);
  auto load_step = [&](int stage) {  // the token looked up last; then the next is
    const uint32_t dst = ring_at + stage * STAGE;
    const bool valid = (uint32_t)page < (uint32_t)a.num_pages;
    const unsigned char* rec = head + (unsigned long long)(uint32_t)(valid ? page : 0) * page_bytes;
    copy_step<D, BULK>(a, L, dst, smem_addr(ring) + stage * STAGE, bar_at + 8 * stage, rec, at_row, valid, lane);
    at += ROUND, at_page += go_pages, at_row += go_rows;
    if (at_row >= a.ps) at_row -= a.ps, ++at_page;
    if (!behind && at >= sl.first) {
      behind = true;
      const int key = at + sl.gap;
      at_page = key / a.ps, at_row = key - at_page * a.ps;
    }
    page = look_up();
  };
  // the queries' rows are on their way together with the first pages
  uint4 raw[NT][H::PIECES][2];
#pragma unroll
  for (int n = 0; n < NT; ++n)
    fetch_query<D>(raw[n], 8 * n + r < R ? a.q + (long)tok * a.q_stride + (long)(kvh * R + 8 * n + r) * D : nullptr, lane);
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) load_step(i);

  Taker<D, NT, BULK> mine(lane);
#pragma unroll
  for (int n = 0; n < NT; ++n) take_query<D>(mine.q[n], mine.undo[n], raw[n], a.scale_log2, lane);
  mine.clear();
  int stage = 0;
  uint32_t parity = 0;
  for (int base = begin + warp * STEP * TILES; base < end; base += ROUND) {
    if (BULK) {
      if (!__all_sync(0xffffffffu, mbar_try_wait(bar_at + 8 * stage, parity)) && !wait_for_tiles(bar_at + 8 * stage, parity, a.error_word)) {
        wait_for_copies(bar_at, stage, parity);
        break;
      }
    } else {
      cp_async_wait<STAGES - 2>();
    }
    __syncwarp();
    const unsigned char* st = ring + stage * STAGE;
    if (base + STEP * TILES <= end && base >= sl.first && base + sl.gap >= sl.lo)  // (of one mind over the warp)
      mine.template take<true>(a, st, base, sl, end);
    else
      mine.template take<false>(a, st, base, sl, end);
    __syncwarp();
    load_step(stage ? stage - 1 : STAGES - 1);
    if (++stage == STAGES) stage = 0, parity ^= 1;
  }
  pdl_launch_dependents();

  // ---- the warps' results, 2^-m times: [warp][query][D + 4] and [warp][query][2] over the rings
  if (!BULK) asm volatile("cp.async.wait_all;\n" ::);
  __syncthreads();
  float* ow = reinterpret_cast<float*>(smem);
  float* ml = ow + WARPS * QS * PITCH;
  float* part = ml + WARPS * QS * 2;  // CLUSTER: [query][D], then [query][2]
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int h = 8 * n + 2 * l + c;
      float* row = ow + (warp * QS + h) * PITCH;
      const float total = mine.finished(n, c, [&](int channel, float4 v) { *reinterpret_cast<float4*>(row + channel) = v; });
      if (r == 0) {
        ml[(warp * QS + h) * 2] = mine.m[n][c];
        ml[(warp * QS + h) * 2 + 1] = total;
      }
    }
  }
  __syncthreads();
  for (int u = tid; u < R * (D / 4); u += THREADS) {
    const int h = u / (D / 4), d = 4 * (u % (D / 4));
    float top = MINUS_BIG;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) top = fmaxf(top, ml[(w * QS + h) * 2]);
    float den = 0.f, y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float f = exp2_fast(ml[(w * QS + h) * 2] - top);
      den += f * ml[(w * QS + h) * 2 + 1];
      const float4 v = *reinterpret_cast<const float4*>(ow + (w * QS + h) * PITCH + d);
      y[0] += f * v.x, y[1] += f * v.y, y[2] += f * v.z, y[3] += f * v.w;
    }
    if (CLUSTER) {
      *reinterpret_cast<float4*>(part + h * D + d) = make_float4(y[0], y[1], y[2], y[3]);
      if (d == 0) part[QS * D + 2 * h] = top, part[QS * D + 2 * h + 1] = den;
    } else if (a.splits > 1) {
      const long where = ((long)slot * a.nq + kvh * R + h) * a.splits + split;
      const float by = den == 0.f ? 1.f : den;  // (all of the slice's scores beyond float32's range below: nothing beside other slices', and 2^-infinity of it)
      *reinterpret_cast<float4*>(a.mid_o + where * D + d) = make_float4(y[0] / by, y[1] / by, y[2] / by, y[3] / by);
      if (d == 0) a.mid_lse[where] = top + log2f(den);
    } else {
      uint2 packed;
      packed.x = pack_bf16(y[0] / den, y[1] / den);
      packed.y = pack_bf16(y[2] / den, y[3] / den);
      *reinterpret_cast<uint2*>(a.out + (out_row + h) * D + d) = packed;
    }
  }
  if (CLUSTER) {  // every block of the cluster joins a share of the rows, slices in order
    cluster_sync_all();
    const uint32_t part_at = smem_addr(part), ml_at = smem_addr(part + QS * D);
    const int count = sl.count(a);
    for (int u = split * THREADS + tid; u < R * (D / 4); u += a.splits * THREADS) {
      const int h = u / (D / 4), d = 4 * (u % (D / 4));
      float2 t[MOST_CLUSTER];
      float4 v[MOST_CLUSTER];
#pragma unroll
      for (int s = 0; s < MOST_CLUSTER; ++s)
        if (s < count) {
          asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(t[s].x), "=f"(t[s].y) : "r"(map_to_cta(ml_at + 8 * h, s)));
          asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                       : "=f"(v[s].x), "=f"(v[s].y), "=f"(v[s].z), "=f"(v[s].w)
                       : "r"(map_to_cta(part_at + 4 * (h * D + d), s)));
        }
      float top = MINUS_BIG, den = 0.f, y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < MOST_CLUSTER; ++s)
        if (s < count) top = fmaxf(top, t[s].x);
#pragma unroll
      for (int s = 0; s < MOST_CLUSTER; ++s)
        if (s < count) {
          const float f = exp2_fast(t[s].x - top);
          den += f * t[s].y;
          y[0] += f * v[s].x, y[1] += f * v[s].y, y[2] += f * v[s].z, y[3] += f * v[s].w;
        }
      const float inv = count > 0 ? 1.f / den : 0.f;
      uint2 packed;
      packed.x = pack_bf16(y[0] * inv, y[1] * inv);
      packed.y = pack_bf16(y[2] * inv, y[3] * inv);
      *reinterpret_cast<uint2*>(a.out + (out_row + h) * D + d) = packed;
    }
    cluster_sync_all();  // a block's results are read until here
  }
}

// Slices of a (sequence, head), in order: a warp per head, four slices' loads in flight.
template <int D> __global__ void __launch_bounds__(THREADS) merge_8bit_kernel(Decode a, int heads) {
  pdl_wait();
  pdl_launch_dependents();
  const int item = blockIdx.x * WARPS + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (item >= heads) return;
  const int slot = item / a.nq, h = item - slot * a.nq;
  const int seq = a.seq_list ? a.seq_list[slot] : slot;
  const int tok = a.cu_seqlens[seq];
  const int slices = Slice<STEP * Head<D>::TILES * WARPS>(a, seq, 0).count(a);
  const float* lses = a.mid_lse + (long)item * a.splits;
  const float* os = a.mid_o + (long)item * a.splits * D;
  float top = MINUS_BIG;
  for (int s = lane; s < slices; s += 32) top = fmaxf(top, lses[s]);
  top = warp_max(top);
  constexpr int C = D >= 128 ? D / 128 : 1, PER = D / 4 < 32 ? D / 4 : 32;
  float den = 0.f, y[C][4] = {};
#pragma unroll 4
  for (int s = 0; s < slices; ++s) {
    const float f = exp2_fast(lses[s] - top);
    den += f;
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (lane < PER) {
        const float4 v = *reinterpret_cast<const float4*>(os + (long)s * D + 128 * c + 4 * lane);
        y[c][0] += f * v.x, y[c][1] += f * v.y, y[c][2] += f * v.z, y[c][3] += f * v.w;
      }
  }
  const float inv = slices > 0 ? 1.f / den : 0.f;
  bf16* row = a.out + ((long)tok * a.nq + h) * D;
#pragma unroll
  for (int c = 0; c < C; ++c)
    if (lane < PER) {
      uint2 packed;
      packed.x = pack_bf16(y[c][0] * inv, y[c][1] * inv);
      packed.y = pack_bf16(y[c][2] * inv, y[c][3] * inv);
      *reinterpret_cast<uint2*>(row + 128 * c + 4 * lane) = packed;
    }
}

template <int D, int NT, bool BULK, bool CLUSTER> constexpr int decode_smem() {
  constexpr int ring = WARPS * STAGES * Head<D>::TILES * (2 * STEP * D + (BULK ? 16 : 8 * STEP));
  constexpr int joined = (WARPS * 8 * NT * (D + 4 + 2) + (CLUSTER ? 8 * NT * (D + 2) : 0)) * 4;
  return ring > joined ? ring : joined;
}
template <int D, int NT, bool BULK, bool CLUSTER> bool decode_ready() {
  auto kernel = decode_8bit_kernel<D, NT, BULK, CLUSTER>;
  static bool once[Q3_MAX_DEVICES];
  const int dev = q3_current_device();
  if (!once[dev]) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, decode_smem<D, NT, BULK, CLUSTER>()) != cudaSuccess) return false;
    if (CLUSTER && cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) return false;
    once[dev] = true;
  }
  return true;
}
// Clusters of `size` blocks that the device holds at a time (which SMs lie together differs between devices).
template <int D, int NT> int decode_clusters(int size) {
  if (!decode_ready<D, NT, true, true>()) return 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(size);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = decode_smem<D, NT, true, true>();
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = size;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int count = 0;
  return cudaOccupancyMaxActiveClusters(&count, decode_8bit_kernel<D, NT, true, true>, &cfg) == cudaSuccess ? count : 0;
}

template <int D, int NT, bool BULK, bool CLUSTER> int launch_decode_as(const Decode& a, int num_seqs, cudaStream_t stream) {
  constexpr int smem = decode_smem<D, NT, BULK, CLUSTER>();
  auto kernel = decode_8bit_kernel<D, NT, BULK, CLUSTER>;
  if (!decode_ready<D, NT, BULK, CLUSTER>()) return Q3_ERR_LAUNCH;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.splits, a.nkv, num_seqs);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (CLUSTER) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = a.splits;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (q3_pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  cudaError_t err = cudaLaunchKernelEx(&cfg, kernel, a);
  if (err == cudaSuccess && !CLUSTER && a.splits > 1) {
    const int heads = num_seqs * a.nq;
    err = launch_pdl(merge_8bit_kernel<D>, dim3((heads + WARPS - 1) / WARPS), dim3(THREADS), 0, stream, a, heads);
  }
  return err == cudaSuccess ? Q3_OK : Q3_ERR_LAUNCH;
}
template <int D, int NT> int launch_decode(const Decode& a, int num_seqs, cudaStream_t stream) {
  const bool bulk = a.ps % STEP == 0, cluster = a.splits > 1 && !a.mid_o;
  if (bulk) return cluster ? launch_decode_as<D, NT, true, true>(a, num_seqs, stream) : launch_decode_as<D, NT, true, false>(a, num_seqs, stream);
  return cluster ? launch_decode_as<D, NT, false, true>(a, num_seqs, stream) : launch_decode_as<D, NT, false, false>(a, num_seqs, stream);
}

// ---- attention in general -----------------------------------------------------------------------------------------------------------------
// float32, and bfloat16 tokens whose head size or group the tiles above do not take: a block takes a (token, kv head, up to NH of its query heads) and
// 256 keys at a time, each of its 8 warps 32 of them, with a softmax of their own: a lane makes a key's scores, channel by channel, from codes that it
// reads itself, then takes two channels (or four, eight) of every value.  No barrier until the warps are joined.  Sums are float32 on the FMA pipes, in an
// order that depends on the keys' places alone: a warp's 32 keys begin at a multiple of 32, what the warps and then the slices of 256 keys have is joined in
// order, by the same block or, where the launch leaves SMs idle, by a second kernel from what one block a slice has left -- the same bits, however a
// sequence is cut into steps and batched with others.  What bounds it is instructions, and for few tokens the chain of a slice: 21 float32 tokens behind up
// to 320, 16 heads over 4 of 64, 10 us (0.17 issued a clock; with barriers between the tiles of a slice 17); eight behind 4,096, 32 over 8 of 128, 52; a prompt of 512 158
// (keys' pieces by neighbouring lanes, each line once: 185).
constexpr int GEN_WARPS = 8;
constexpr int GEN_THREADS = 32 * GEN_WARPS;
constexpr int GEN_SLICE = 32 * GEN_WARPS;

struct General {
  const unsigned char* pages;
  int num_pages;
  const int *block_table, *token_seq, *places;
  int max_pages, num_seqs, nq, nkv, D, ps, window, keep_first, slices;
  long q_stride;
  float scale_log2;
  float *mid_o, *mid_ml;  // slices > 0: [tokens][nq][slices][D] and [tokens][nq][slices][2]
  // the last key that token t sees; -1: none (it belongs to no sequence, or its place lies outside the table), and its row is zero
  __device__ __forceinline__ int last_key(long t) const {
    const int seq = token_seq[t], place = places[t];
    return seq >= 0 && seq < num_seqs && place >= 0 && place / ps < max_pages ? place : -1;
  }
  // the first key of the window of a token that sees keys up to `last`
  __device__ __forceinline__ int window_begin(int last) const { return window > 0 ? max(0, last - window + 1) : 0; }
  // Slices that hold a key which the token sees: 0 .. kept - 1, and those from kept + gap on.
  __device__ __forceinline__ int kept_slices(int lo) const { return min((keep_first + GEN_SLICE - 1) / GEN_SLICE, lo / GEN_SLICE); }
};

// (m, l) <- its join with another slice's, and what results (unnormalised) are multiplied by: o <- o fa + bo fb.  The fused steps are named, so that
// both kernels round alike.
__device__ __forceinline__ void join_sums(float& m, float& l, float bm, float bl, float& fa, float& fb) {
  const float top = fmaxf(m, bm);
  fa = exp2f(m - top), fb = exp2f(bm - top);
  m = top;
  l = __fmaf_rn(l, fa, __fmul_rn(bl, fb));
}
// As many neighbouring codes as `v` has places, from an address that is a multiple of that.
__device__ __forceinline__ void read_codes(const unsigned char* at, float (&v)[2]) {
  float y[4];
  q8_floats(*reinterpret_cast<const uint16_t*>(at), y);
  v[0] = y[0], v[1] = y[1];
}
__device__ __forceinline__ void read_codes(const unsigned char* at, float (&v)[4]) { q8_floats(*reinterpret_cast<const uint32_t*>(at), v); }
__device__ __forceinline__ void read_codes(const unsigned char* at, float (&v)[8]) {
  const uint2 w = *reinterpret_cast<const uint2*>(at);
  float lo[4], hi[4];
  q8_floats(w.x, lo);
  q8_floats(w.y, hi);
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = lo[e], v[4 + e] = hi[e];
}

// NH: heads of a block; CH: channels of a lane (heads of up to 32 CH channels).
template <typename T, int NH, int CH>
__global__ void __launch_bounds__(GEN_THREADS) general_8bit_kernel(General a, const T* __restrict__ q, T* __restrict__ out) {
  extern __shared__ __align__(16) float shared[];
  pdl_wait();
  pdl_launch_dependents();
  const int R = a.nq / a.nkv, chunks = (R + NH - 1) / NH, D = a.D, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, mask = q8_mask(D);
  const int t = blockIdx.x, kvh = blockIdx.y / chunks, h0 = kvh * R + (blockIdx.y - kvh * chunks) * NH, heads = min(NH, kvh * R + R - h0);
  const Q8Page L(D, a.ps);
  float* q_s = shared;                                  // [NH][D]
  float* o_s = q_s + NH * D;                            // [warps][NH][D]
  float* ml_s = o_s + GEN_WARPS * NH * D;               // [warps][NH][2]: maxima and sums
  float* f_s = ml_s + GEN_WARPS * NH * 2;               // [warps + 2][NH]: what the warps' results, the slices so far and this one are multiplied by
  float2* p_s = reinterpret_cast<float2*>(f_s + (GEN_WARPS + 2) * NH) + warp * 32 * NH;  // [32][NH], this warp's weights, twice each
  const int last = a.last_key(t), lo = a.window_begin(last), mine = CH * lane;  // this lane's first channel
  const int* bt = a.block_table + (long)(last >= 0 ? a.token_seq[t] : 0) * a.max_pages;
  for (int i = tid; i < NH * D; i += GEN_THREADS) q_s[i] = i < heads * D ? to_f32(q[t * a.q_stride + (long)h0 * D + i]) * a.scale_log2 : 0.f;
  __syncthreads();
  // thread h keeps head h's joined maximum and sum; a thread the joined results of (head, channel) tid, tid + 256 ...
  constexpr int OWN = NH * CH * 32 / GEN_THREADS;
  float M = MINUS_BIG, S = 0.f, O[OWN];
#pragma unroll
  for (int i = 0; i < OWN; ++i) O[i] = 0.f;
  const int kept = a.kept_slices(lo), gap = lo / GEN_SLICE - kept, count = last < 0 ? 0 : last / GEN_SLICE + 1 - gap;
  int first_slice = 0, stop_slice = count;  // of those that count
  if (a.slices > 0) {
    const int z = blockIdx.z;
    first_slice = z < kept ? z : z - gap;
    stop_slice = (z >= kept && z < kept + gap) || first_slice >= count ? first_slice : first_slice + 1;
  }
  for (int s = first_slice; s < stop_slice; ++s) {
    const int key = (s + (s >= kept ? gap : 0)) * GEN_SLICE + 32 * warp + lane;
    const bool seen = key <= last && (key >= lo || key < a.keep_first);
    // this lane's key: where its codes lie
    const unsigned char* rec = nullptr;
    int row = 0;
    if (seen) {
      const int pi = key / a.ps, page = bt[pi];
      row = key - pi * a.ps;
      if ((uint32_t)page < (uint32_t)a.num_pages) rec = a.pages + ((long)page * a.nkv + kvh) * L.record;
    }
    const uint32_t there = __ballot_sync(0xffffffffu, rec != nullptr);
    float m[NH], l[NH];
    float2 o[NH][CH / 2];
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      m[h] = MINUS_BIG, l[h] = 0.f;
#pragma unroll
      for (int c = 0; c < CH / 2; ++c) o[h][c] = make_float2(0.f, 0.f);
    }
    if (there) {
      float2 x[NH];  // sums over every second channel (two of them an instruction)
#pragma unroll
      for (int h = 0; h < NH; ++h) x[h] = make_float2(0.f, 0.f);
      const unsigned char *codes = rec + (long)row * D, *values = codes + L.values;
      float2 scale = make_float2(0.f, 0.f);
      if (rec) {
        scale = *reinterpret_cast<const float2*>(rec + L.scales);
        asm volatile("prefetch.global.L2 [%0];" ::"l"(values));
        if (D > 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(values + 128));
      }
#pragma unroll 1
      for (int piece0 = 0; piece0 < D / 16; piece0 += 4) {  // four loads at a time
        uint4 w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          w[i] = make_uint4(0, 0, 0, 0);
          if (rec && piece0 + i < D / 16) w[i] = *reinterpret_cast<const uint4*>(codes + 16 * ((piece0 + i) ^ (row & mask)));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (piece0 + i >= D / 16) break;
          const uint32_t word[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
          const float* y_at = q_s + 16 * (piece0 + i);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float v[4];
            q8_floats(word[e], v);
#pragma unroll
            for (int h = 0; h < NH; ++h) {
              const float4 y = *reinterpret_cast<const float4*>(y_at + h * D + 4 * e);
              x[h] = __ffma2_rn(make_float2(y.x, y.y), make_float2(v[0], v[1]), x[h]);
              x[h] = __ffma2_rn(make_float2(y.z, y.w), make_float2(v[2], v[3]), x[h]);
            }
          }
        }
      }
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        const float y = rec ? (x[h].x + x[h].y) * scale.x : -INFINITY;
        m[h] = fmaxf(MINUS_BIG, warp_max(y));
        const float p = exp2f(y - m[h]), w = p * scale.y;  // (a power of two: what the values are to be multiplied by)
        l[h] = warp_sum(p);
        x[h] = make_float2(w, w);
      }
      __syncwarp();
#pragma unroll
      for (int h = 0; h < NH; h += 2) *reinterpret_cast<float4*>(p_s + lane * NH + h) = make_float4(x[h].x, x[h].y, x[h + 1].x, x[h + 1].y);
      __syncwarp();
      // where this lane's value row begins, a multiple of 16, and below that how its pieces are ordered
      const unsigned long long where = reinterpret_cast<unsigned long long>(values) | (uint32_t)(row & mask);
#pragma unroll 1
      for (int k0 = 0; k0 < 32; k0 += 8) {
        if (!(there >> k0 & 255u)) continue;
        float v[8][CH];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const unsigned long long from = __shfl_sync(0xffffffffu, where, k0 + k);
#pragma unroll
          for (int c = 0; c < CH; ++c) v[k][c] = 0.f;
          if ((there >> (k0 + k) & 1u) && mine < D) read_codes(reinterpret_cast<const unsigned char*>(from & ~15ull) + (mine ^ ((int)from << 4 & 0xF0)), v[k]);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          float2 p[NH];
#pragma unroll
          for (int h = 0; h < NH; h += 2) *reinterpret_cast<float4*>(p + h) = *reinterpret_cast<const float4*>(p_s + (k0 + k) * NH + h);
#pragma unroll
          for (int h = 0; h < NH; ++h)
#pragma unroll
            for (int c = 0; c < CH / 2; ++c) o[h][c] = __ffma2_rn(p[h], make_float2(v[k][2 * c], v[k][2 * c + 1]), o[h][c]);
        }
      }
    }
    // the warps' results, joined in order to what came before
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      if (lane == 0) *reinterpret_cast<float2*>(ml_s + 2 * (warp * NH + h)) = make_float2(m[h], l[h]);
#pragma unroll
      for (int c = 0; c < CH / 2; ++c)
        if (mine < D) *reinterpret_cast<float2*>(o_s + (warp * NH + h) * D + mine + 2 * c) = o[h][c];
    }
    __syncthreads();
    if (tid < NH) {
      float top = MINUS_BIG, sum = 0.f;
#pragma unroll
      for (int w = 0; w < GEN_WARPS; ++w) top = fmaxf(top, ml_s[2 * (w * NH + tid)]);
#pragma unroll
      for (int w = 0; w < GEN_WARPS; ++w) {
        const float f = exp2f(ml_s[2 * (w * NH + tid)] - top);
        f_s[w * NH + tid] = f;
        sum = __fmaf_rn(f, ml_s[2 * (w * NH + tid) + 1], sum);
      }
      join_sums(M, S, top, sum, f_s[GEN_WARPS * NH + tid], f_s[(GEN_WARPS + 1) * NH + tid]);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
      const int u = tid + GEN_THREADS * i, h = u / D;
      if (u < NH * D) {
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < GEN_WARPS; ++w) sum = __fmaf_rn(f_s[w * NH + h], o_s[w * NH * D + u], sum);
        O[i] = __fmaf_rn(O[i], f_s[GEN_WARPS * NH + h], __fmul_rn(sum, f_s[(GEN_WARPS + 1) * NH + h]));
      }
    }
    __syncthreads();
  }
  if (tid < NH) ml_s[tid] = S;
  if (a.slices > 0 && tid < heads) *reinterpret_cast<float2*>(a.mid_ml + 2 * (((long)t * a.nq + h0 + tid) * a.slices + blockIdx.z)) = make_float2(M, S);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < OWN; ++i) {
    const int u = tid + GEN_THREADS * i, h = u / D, c = u - h * D;
    if (u >= heads * D) continue;
    if (a.slices > 0) {
      const long at = ((long)t * a.nq + h0 + h) * a.slices + blockIdx.z;
      a.mid_o[at * D + c] = O[i];
    } else {
      out[((long)t * a.nq + h0 + h) * D + c] = from_f32<T>(last >= 0 ? O[i] / ml_s[h] : 0.f);
    }
  }
}

// One block per (token, head): joins the slices that hold a key which the token sees, in order, a thread per channel.
template <typename T> __global__ void general_8bit_merge_kernel(General a, T* __restrict__ out) {
  pdl_wait();
  pdl_launch_dependents();
  const long at = blockIdx.x;
  const int last = a.last_key(at / a.nq), lo = a.window_begin(last);
  const int kept = a.kept_slices(lo), gap = lo / GEN_SLICE - kept, count = last < 0 ? 0 : min(last / GEN_SLICE + 1, a.slices) - gap;
  for (int c = threadIdx.x; c < a.D; c += blockDim.x) {
    float M = MINUS_BIG, S = 0.f, O = 0.f;
    for (int s0 = 0; s0 < count; s0 += 8) {  // eight slices' loads at a time
      float m[8], l[8], o[8];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (s0 + u < count) {
          const long i = at * a.slices + s0 + u + (s0 + u >= kept ? gap : 0);
          m[u] = a.mid_ml[2 * i], l[u] = a.mid_ml[2 * i + 1], o[u] = a.mid_o[i * a.D + c];
        }
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (s0 + u < count) {
          float fa, fb;
          join_sums(M, S, m[u], l[u], fa, fb);
          O = __fmaf_rn(O, fa, __fmul_rn(o[u], fb));
        }
    }
    out[at * a.D + c] = from_f32<T>(last >= 0 ? O / S : 0.f);
  }
}

template <typename T, int NH, int CH> int launch_general_as(const General& a, const T* q, T* out, int tokens, cudaStream_t stream) {
  const int chunks = (a.nq / a.nkv + NH - 1) / NH;
  const int smem = 4 * (NH * a.D * (1 + GEN_WARPS) + NH * (GEN_WARPS * (2 + 1 + 64) + 2));
  static bool once[Q3_MAX_DEVICES];
  const int dev = q3_current_device();
  if (!once[dev]) {
    if (cudaFuncSetAttribute(general_8bit_kernel<T, NH, CH>, cudaFuncAttributeMaxDynamicSharedMemorySize, 96 * 1024) != cudaSuccess) return Q3_ERR_LAUNCH;
    once[dev] = true;
  }
  cudaError_t err = launch_pdl(general_8bit_kernel<T, NH, CH>, dim3(tokens, a.nkv * chunks, a.slices > 0 ? a.slices : 1), dim3(GEN_THREADS), smem, stream,
                               a, q, out);
  if (err == cudaSuccess && a.slices > 0)
    err = launch_pdl(general_8bit_merge_kernel<T>, dim3((unsigned)((long)tokens * a.nq)), dim3(a.D <= 128 ? 128 : 256), 0, stream, a, out);
  return err == cudaSuccess ? Q3_OK : Q3_ERR_LAUNCH;
}
template <typename T> int launch_general(const General& a, const T* q, T* out, int tokens, cudaStream_t stream) {
  if (a.nq / a.nkv <= 4) {
    if (a.D <= 64) return launch_general_as<T, 4, 2>(a, q, out, tokens, stream);
    return a.D <= 128 ? launch_general_as<T, 4, 4>(a, q, out, tokens, stream) : launch_general_as<T, 4, 8>(a, q, out, tokens, stream);
  }
  if (a.D <= 64) return launch_general_as<T, 8, 2>(a, q, out, tokens, stream);
  return a.D <= 128 ? launch_general_as<T, 8, 4>(a, q, out, tokens, stream) : launch_general_as<T, 8, 8>(a, q, out, tokens, stream);
}

}  // namespace

Q3_EXPORT int q3_decode_attention_8bit(const void* q, int q_stride, const void* pages, int num_pages, const int* block_table, int max_pages,
                                       const int* kv_lens, const int* cu_seqlens, const int* seq_list, void* out, float* mid_o,
                                       float* mid_lse, int num_seqs, int nq, int nkv, int D, int ps, float scale, int window, int keep_first,
                                       int splits, int max_len, const int* longest, int* error_word, cudaStream_t stream) {
  if (num_seqs < 1) return Q3_OK;
  if (!q || !pages || !block_table || !kv_lens || !cu_seqlens || !out || nq < 1 || nkv < 1 || nq % nkv || !q8_sizes_ok(D, ps) || splits < 1 ||
      !error_word || (splits > MOST_CLUSTER && !mid_o) || (mid_o && !mid_lse) || max_len > (long)max_pages * ps || keep_first < 0)
    return Q3_ERR_ARGUMENT;
  const int R = nq / nkv;
  if (R > 16 || q_stride % 8 || (reinterpret_cast<uintptr_t>(q) & 15) || (reinterpret_cast<uintptr_t>(pages) & 15) ||
      (reinterpret_cast<uintptr_t>(out) & 7) || num_seqs > 65535 || nkv > 65535 || Q8Page(D, ps).record * nkv > 0x7fffffffL ||
      (long)window + keep_first > 0x7ffffff0L)
    return Q3_ERR_UNSUPPORTED;
  Decode a{(const bf16*)q, q_stride, (const unsigned char*)pages, num_pages, block_table, kv_lens, cu_seqlens, seq_list, max_pages,
           (bf16*)out, mid_o, mid_lse, nq, nkv, ps, window, window > 0 ? keep_first : 0, splits, max_len, scale * LOG2_E, longest, error_word};
  if (D == 64) return R <= 8 ? launch_decode<64, 1>(a, num_seqs, stream) : launch_decode<64, 2>(a, num_seqs, stream);
  if (D == 128) return R <= 8 ? launch_decode<128, 1>(a, num_seqs, stream) : launch_decode<128, 2>(a, num_seqs, stream);
  if (D == 256) return R <= 8 ? launch_decode<256, 1>(a, num_seqs, stream) : launch_decode<256, 2>(a, num_seqs, stream);
  return Q3_ERR_UNSUPPORTED;
}

// How many clusters of `size` blocks of decode attention run at a time, for groups of up to 8 query heads or (wide) more; 0: not known.
Q3_EXPORT int q3_decode_clusters_8bit(int D, int wide, int size) {
  if (size < 1 || size > MOST_CLUSTER) return 0;
  if (D == 64) return wide ? decode_clusters<64, 2>(size) : decode_clusters<64, 1>(size);
  if (D == 128) return wide ? decode_clusters<128, 2>(size) : decode_clusters<128, 1>(size);
  if (D == 256) return wide ? decode_clusters<256, 2>(size) : decode_clusters<256, 1>(size);
  return 0;
}

// `slices` 0: a block goes through all of a token's keys; else mid_o [tokens][nq][slices][D] and mid_ml [tokens][nq][slices][2] are given and
// slices * 256 covers the longest sequence.
Q3_EXPORT int q3_general_attention_8bit(int dtype, const void* q, long q_stride, const void* pages, int num_pages, const int* block_table,
                                        int max_pages, int num_seqs, const int* token_seq, const int* places, void* out, float* mid_o,
                                        float* mid_ml, int slices, int tokens, int nq, int nkv, int D, int ps, float scale, int window,
                                        int keep_first, cudaStream_t stream) {
  if (tokens < 1) return Q3_OK;
  if (!q || !pages || !block_table || !token_seq || !places || !out || nq < 1 || nkv < 1 || nq % nkv || !q8_sizes_ok(D, ps) || max_pages < 1 ||
      slices < 0 || (slices > 0 && (!mid_o || !mid_ml)) || keep_first < 0)
    return Q3_ERR_ARGUMENT;
  if (dtype != Q3_DTYPE_F32 && dtype != Q3_DTYPE_BF16) return Q3_ERR_ARGUMENT;
  if ((long)nkv * ((nq / nkv + 3) / 4) > 65535 || slices > 65535 || (long)tokens * nq > 0x7fffffffL ||
      (reinterpret_cast<uintptr_t>(pages) & 15))
    return Q3_ERR_UNSUPPORTED;
  General a{(const unsigned char*)pages, num_pages, block_table, token_seq, places, max_pages, num_seqs, nq, nkv, D, ps, window,
            window > 0 ? keep_first : 0, slices, q_stride, scale * LOG2_E, mid_o, mid_ml};
  return dtype == Q3_DTYPE_F32 ? launch_general(a, (const float*)q, (float*)out, tokens, stream)
                               : launch_general(a, (const bf16*)q, (bf16*)out, tokens, stream);
}
