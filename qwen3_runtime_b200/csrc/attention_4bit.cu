// Attention over a cache in 4 bits (layout: four_bit.cuh): decode attention in bfloat16, and the sums of attention weights per cached
// token that eviction goes by.
//
// Numbers stay in 4 bits up to the registers, and what all channels of a group share is applied to sums:
// A number n = 0 .. 15 in the low bits of a bfloat16 is n * 2^-133 (subnormal), and four bits further up 16 n * 2^-133 (subnormal up to 7,
// the lowest exponent from 8 on: both have the same step).  mma.sync takes subnormal operands exactly, so a word of 8 numbers becomes
// four operands by four masks and one shift, x & 0x000F000F, x & 0x00F000F0 and the same of x >> 8, and the other operand brings the
// power of two that lifts the products into float32's range:
//   scores   K (16 keys) x Q^T (8 queries) on mma.sync m16n8k16, one accumulator per group g of channels; a query row times 2^S, its
//            largest near 2^110:
//              score = sum_g  s_g 2^(133 - S) acc_g + z_g sum_(c in g) q_c
//   results  V^T (16 channels) x P^T.  P^T is the score tile times the tokens' scales, w_t = bf16(p_t s_t) 2^T, transposed by movmatrix;
//            T follows the largest scale seen, as the softmax follows the largest score:
//              o_c = 2^(133 - T) (sum_t w_t n_tc - sum_t 8 w_t) + sum_t p_t (z_t + 8 s_t)
//            The second sum is one more product with constant rows, the third runs in float32.  The one rounding of a weight thus
//            weighs on n - 8, as small as the values about their middle (with w_t n_tc and z_t alone results were twice as far off).
// (Numbers as 1 + n / 16, a shift and a mask each, took 118 us where this takes 73, eight sequences of 17,000 to 32,768 tokens, 64 heads
// over 8 of 128; as 8-bit floats, whose byte n is n * 2^-9 without any conversion, 137: mma.sync converts those by instructions.)
// Keys as the product's 16 rows and the kv head's queries as its 8 columns: a group of up to 8 query heads wastes nothing (the other way
// round, 16 rows of queries, computes twice as much, and the conversion would meet half as many values per instruction).
#include <type_traits>

#include "async_tiles.cuh"
#include "four_bit.cuh"
#include "mma_tiles.cuh"

#define Q3_ERR_WAIT_4BIT 21

namespace {

// The maximum of a row that has seen nothing: no score lies below it, and a hidden key's, -inf, weighs 2^(-inf - MINUS_BIG) = 0.
constexpr float MINUS_BIG = -3.402823466e+38f;
constexpr float LN_2 = 0.6931471805599453f;

// Numbers J and J + 4 of a word `w` (`high`: w >> 8), or number J of two tokens whose halves were put side by side, as two bfloat16:
// times 2^-133 (J even) or 2^-129 (J odd).
template <int J> __device__ __forceinline__ uint32_t tiny_of(uint32_t w, uint32_t high) {
  return (J < 2 ? w : high) & (J & 1 ? 0x00F000F0u : 0x000F000Fu);
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }  // -126 .. 127
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
// c[16 x 8] = a[16 x 16] b[16 x 8]: a sum's first product
__device__ __forceinline__ void mma_bf16_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void cp_async8(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;\n" ::"r"(dst), "l"(src), "r"(bytes));
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(dst), "l"(src), "r"(bytes));
}

// What a warp's lanes hold of 16 keys: rows lane / 4 and lane / 4 + 8, and of each row the words that lane % 4 takes.
// D = 64: 2 words (one group); 128: 4 (two groups in turn); 256: two pieces of 4 (four groups in turn each).
template <int D> struct Head {
  static constexpr int G = D / 64;         // groups
  static constexpr int WORDS = D / 32;     // words of a row that a lane holds
  static constexpr int ROW = D / 2;        // bytes of a row of codes
  static constexpr int PAR = 4 * G;
  static constexpr int TILE = 16 * (D + 2 * PAR);  // bytes of 16 tokens' keys and values
  // word j of lane l: which group, and which 8 channels of it
  static __device__ __forceinline__ int group(int j) { return D == 64 ? 0 : j % G; }
  static __device__ __forceinline__ int index(int j, int l) {
    return D == 64 ? 2 * l + j : D == 128 ? 2 * l + j / 2 : l + 4 * (j / 4);
  }
};

// The queries' side of the scores: B fragments (n = lane / 4: the query, k: the channels that word j's pairs stand for; b[j][0..3]: of word j,
// channels (0, 4), (1, 5), (2, 6), (3, 7) of its eight), times 2^S, the channels that meet 2^-129 a 16th of it.  `undo`: what the sums
// are to be multiplied by, for columns 2 (lane % 4) and + 1; `sum`: the channels' sums per group, both times the scores' scale.
template <int D> __device__ __forceinline__ void fetch_query(uint4 (&raw)[Head<D>::WORDS], const bf16* row, int lane) {
#pragma unroll
  for (int j = 0; j < Head<D>::WORDS; ++j) {
    raw[j] = make_uint4(0, 0, 0, 0);
    if (row) raw[j] = *reinterpret_cast<const uint4*>(row + 64 * Head<D>::group(j) + 8 * Head<D>::index(j, lane & 3));
  }
}
template <int D> __device__ __forceinline__ void take_query(uint32_t (&b)[Head<D>::WORDS][4], float (&undo)[2], float (&sum)[Head<D>::G][2],
                                                            const uint4 (&raw)[Head<D>::WORDS], float scale_log2, int lane) {
  using H = Head<D>;
  float v[H::WORDS][8], top = 0.f, part[H::G];
#pragma unroll
  for (int g = 0; g < H::G; ++g) part[g] = 0.f;
#pragma unroll
  for (int j = 0; j < H::WORDS; ++j) {
    const uint32_t word[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
#pragma unroll
    for (int e = 0; e < 4; ++e) v[j][2 * e] = __uint_as_float(word[e] << 16), v[j][2 * e + 1] = __uint_as_float(word[e] & 0xFFFF0000u);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      top = fmaxf(top, fabsf(v[j][e]));
      part[H::group(j)] += v[j][e];
    }
  }
#pragma unroll
  for (int d = 1; d < 4; d <<= 1) {
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
#pragma unroll
    for (int g = 0; g < H::G; ++g) part[g] += __shfl_xor_sync(0xffffffffu, part[g], d);
  }
  // S = 110 less the largest's exponent; 120 at most (smaller rows need no more), and an infinite row stays infinite
  const int S = min(120, 237 - (int)(__float_as_uint(top) >> 23));
  const float even = power_of_two(S), odd = power_of_two(S - 4);
#pragma unroll
  for (int j = 0; j < H::WORDS; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) b[j][e] = pack_bf16(v[j][e] * (e & 1 ? odd : even), v[j][e + 4] * (e & 1 ? odd : even));
  // (scores beyond 2^100 of rows beyond 2^104 come out too small, and still tell one key from all others)
  const float back = scale_log2 * power_of_two(min(120, 133 - S));
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int from = 4 * (2 * (lane & 3) + c);
    undo[c] = __shfl_sync(0xffffffffu, back, from);
#pragma unroll
    for (int g = 0; g < H::G; ++g) sum[g][c] = __shfl_sync(0xffffffffu, part[g], from) * scale_log2;
  }
}
template <int D> __device__ __forceinline__ void load_query_tiny(uint32_t (&b)[Head<D>::WORDS][4], float (&undo)[2], float (&sum)[Head<D>::G][2],
                                                                 const bf16* row, float scale_log2, int lane) {
  uint4 raw[Head<D>::WORDS];
  fetch_query<D>(raw, row, lane);
  take_query<D>(b, undo, sum, raw, scale_log2, lane);
}

// ---- decode attention -------------------------------------------------------------------------------------------------------------
// Grid (slice, kv head, sequence): a block takes one slice of one sequence's keys for one kv head and the query heads that read it; each of
// its 4 warps takes every fourth 32 keys, with a ring of its own and a softmax of its own (no barrier in the loop), and the warps are
// joined at the end.  Where the launch leaves SMs idle, up to 16 slices are the blocks of a cluster, which read each other's results in shared
// memory; else they go through global memory and a second kernel (a B200 holds 45 clusters of 11 of these blocks at a
// time, 495 of the 592 blocks that it holds otherwise).
//   BULK   page sizes that are a multiple of 16: a tile is 16 tokens of one page, brought by one bulk copy (16 tokens a page) or four
//          that a lane asks for.  Rows behind the slice's end come along and are masked.
//   else   any page size: cp.async token by token, what is not there is zero.
// What bounds it: instructions.  16 tokens of 128 channels, 2304 bytes, take 100 clocks of an SM to stream; their shifts and logic run at 2
// a clock, 128 of them for the conversion alone.
constexpr int WARPS = 4;
constexpr int THREADS = 32 * WARPS;
constexpr int STEP = 16;            // keys of a tile
constexpr int TILES = 2;            // tiles that a warp takes at a time: what is asked and counted once for both costs half
constexpr int ROUND = STEP * TILES * WARPS;
constexpr int STAGES = 3;
constexpr int MOST_CLUSTER = 16;

// A step's barrier, when the first look finds its bytes still on their way; called by whole warps, which leave it of one mind.  Bounded:
// false after the limit.  The warp then asks for nothing more (the barrier has its arrivals, and must not be given others), waits for what
// it has in flight (wait_for_copies) and goes on to the block's end; the error word says that the result is invalid.
__device__ __noinline__ bool wait_for_tiles(uint32_t bar, uint32_t parity, int* error_word) {
  const long long start = clock64();
  while (!__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) {
    if (__any_sync(0xffffffffu, clock64() - start > Q3_WAIT_LIMIT_CYCLES)) {
      atomicExch(error_word, Q3_ERR_WAIT_4BIT);
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

// Which token is row r of a tile (r < 8; row r + 8 is token + 8).  Any order will do, as keys and values agree on it; these let the rows
// that one shared-memory access meets lie in different banks (D = 128: values two-way at worst).
template <int D> __device__ __forceinline__ int token_of(int r) {
  const int l = r >> 1;
  return r & 1 ? 4 + (D == 64 ? (l + 2) & 3 : l ^ 1) : l;
}

struct Decode {
  const bf16* q;
  int q_stride;
  const unsigned char* pages;
  int num_pages;
  const int *block_table, *kv_lens, *cu_seqlens, *seq_list;
  int max_pages;
  bf16* out;
  float *mid_o, *mid_lse, *lse;
  int nq, nkv, ps, window, splits, max_len;
  float scale_log2;
  const int* longest;
  int* error_word;
};

// Slices are cut from the first visible key, rounded down to a tile (BULK: a tile lies in one page).  Keys per slice, the same for all
// sequences of the launch: the longest sequence's keys over the slices asked for, in whole rounds of the block.  A shorter sequence has
// fewer slices.
struct Slice {
  int kv_len, lo, begin, end, per;
  __device__ __forceinline__ Slice(const Decode& a, int seq, int split) {
    kv_len = min(a.kv_lens[seq], a.max_len);
    lo = a.window > 0 ? max(0, kv_len - a.window) : 0;
    int longest = a.longest ? min(*a.longest, a.max_len) : a.max_len;
    if (a.window > 0) longest = min(longest, a.window + STEP - 1);
    per = max(ROUND, ((longest + a.splits - 1) / a.splits + ROUND - 1) / ROUND * ROUND);
    begin = (lo & ~(STEP - 1)) + split * per;
    end = min(kv_len, begin + per);
  }
  __device__ __forceinline__ int count(const Decode& a) const {  // slices that have keys
    return min(a.splits, max(0, kv_len - (lo & ~(STEP - 1)) + per - 1) / per);
  }
};

template <int D, int NT> constexpr int decode_blocks() { return D == 64 ? (NT == 1 ? 5 : 4) : D == 128 ? (NT == 1 ? 4 : 2) : NT == 1 ? 2 : 1; }

template <int D, int NT, bool BULK, bool CLUSTER>
__global__ void __launch_bounds__(THREADS, decode_blocks<D, NT>()) decode_4bit_kernel(Decode a) {
  using H = Head<D>;
  constexpr int QS = 8 * NT, PITCH = D + 4;
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
  const Slice sl(a, seq, split);
  const int begin = sl.begin, end = sl.end;
  const long out_row = (long)tok * a.nq + kvh * R;
  if (!CLUSTER && begin >= end) {
    pdl_launch_dependents();
    if (a.splits == 1) {  // no key at all
      for (int i = tid; i < R * D; i += THREADS) a.out[out_row * D + i] = __float2bfloat16_rn(0.f);
      if (a.lse && tid < R) a.lse[out_row + tid] = -INFINITY;
    }
    return;
  }
  const Q4Page L(D, H::G, a.ps);
  const int* bt = a.block_table + (long)seq * a.max_pages;
  constexpr int STAGE = TILES * H::TILE;
  unsigned char* ring = smem + warp * STAGES * STAGE;

  // The token that this lane copies (BULK: lanes 0 and 1, a tile's first), as page of the sequence and row, moved on by a round at a time.
  // Its page is looked up a step before the copy, whose address waits for it.
  const unsigned char* head = a.pages + kvh * L.record;
  const uint32_t page_bytes = (uint32_t)(a.nkv * L.record);
  int at = begin + warp * STEP * TILES + (BULK ? STEP * lane : lane), at_page = at / a.ps, at_row = at - at_page * a.ps;
  const int go_pages = ROUND / a.ps, go_rows = ROUND - go_pages * a.ps;
  auto look_up = [&]() { return at < end ? bt[at_page] : -1; };
  int page = -1;
  if (!BULK || lane < TILES) page = look_up();
  const uint32_t ring_at = smem_addr(ring) + (BULK ? lane * H::TILE : (lane >> 4) * H::TILE), bar_at = smem_addr(&bars[warp][0]);
  auto load_step = [&](int stage) {  // the token looked up last; then the next is
    if (BULK && lane >= TILES) return;
    const uint32_t dst = ring_at + stage * STAGE;
    const bool valid = (uint32_t)page < (uint32_t)a.num_pages;
    const unsigned char* rec = head + (unsigned long long)(uint32_t)(valid ? page : 0) * page_bytes;
    if (BULK) {  // each lane arrives once, with the bytes that it asks for
      const uint32_t bar = bar_at + 8 * stage;
      mbar_expect_tx(bar, valid ? H::TILE : 0);
#ifdef Q3_TEST_WITHHOLD_A_BOX  // (a test build leaves the second tiles out: the stages never fill, a wait runs out)
      if (valid && lane == 0) {
#else
      if (valid) {
#endif
        if (a.ps == STEP) {
          bulk_copy(dst, rec, H::TILE, bar);
        } else {
          bulk_copy(dst, rec + at_row * H::ROW, STEP * H::ROW, bar);
          bulk_copy(dst + STEP * H::ROW, rec + L.values + at_row * H::ROW, STEP * H::ROW, bar);
          bulk_copy(dst + 2 * STEP * H::ROW, rec + L.kpar + at_row * H::PAR, STEP * H::PAR, bar);
          bulk_copy(dst + 2 * STEP * H::ROW + STEP * H::PAR, rec + L.vpar + at_row * H::PAR, STEP * H::PAR, bar);
        }
      }
    } else {
      const unsigned char* src = rec + (valid ? at_row : 0) * H::ROW;
#pragma unroll
      for (int c = 0; c < H::ROW / 16; ++c) {
        cp_async16(dst + (lane & 15) * H::ROW + 16 * c, src + 16 * c, valid ? 16 : 0);
        cp_async16(dst + (STEP + (lane & 15)) * H::ROW + 16 * c, src + L.values + 16 * c, valid ? 16 : 0);
      }
      const uint32_t par = dst + 2 * STEP * H::ROW + (lane & 15) * H::PAR;
      src = rec + L.kpar + (valid ? at_row : 0) * H::PAR;
      const long vpar = L.vpar - L.kpar;
      if (D == 64) cp_async4(par, src, valid ? 4 : 0), cp_async4(par + STEP * H::PAR, src + vpar, valid ? 4 : 0);
      if (D == 128) cp_async8(par, src, valid ? 8 : 0), cp_async8(par + STEP * H::PAR, src + vpar, valid ? 8 : 0);
      if (D == 256) cp_async16(par, src, valid ? 16 : 0), cp_async16(par + STEP * H::PAR, src + vpar, valid ? 16 : 0);
      cp_async_commit();
    }
    at += ROUND, at_page += go_pages, at_row += go_rows;
    if (at_row >= a.ps) at_row -= a.ps, ++at_page;
    page = look_up();
  };
  // the queries' rows are on their way together with the first pages
  uint4 raw[NT][H::WORDS];
#pragma unroll
  for (int n = 0; n < NT; ++n)
    fetch_query<D>(raw[n], 8 * n + r < R ? a.q + (long)tok * a.q_stride + (long)(kvh * R + 8 * n + r) * D : nullptr, lane);
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) load_step(i);

  uint32_t q[NT][H::WORDS][4];
  float qsum[NT][H::G][2], undo[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) take_query<D>(q[n], undo[n], qsum[n], raw[n], a.scale_log2, lane);
  // o: sums of w n (times 2^-133, odd j 2^-129); oz: of -8 w (2^-133); oc: of p (z + 8 s), this lane's share; all of 16 p in place of p.
  // lift = 2^T is set so that the largest scale seen lies in 2^100 .. 2^115, beyond which it is set anew.
  float o[NT][H::G][4][4], oz[NT][H::G][4], oc[NT][H::G][2], m[NT][2], sum[NT][2];
  float most_scale = -1.f, lift = 1.f;
  int T = 0;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    m[n][0] = m[n][1] = MINUS_BIG;
    sum[n][0] = sum[n][1] = 0.f;
#pragma unroll
    for (int g = 0; g < H::G; ++g) {
      oc[n][g][0] = oc[n][g][1] = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        oz[n][g][e] = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[n][g][j][e] = 0.f;
      }
    }
  }
  uint32_t eight[4];  // -8 * 2^-133, kept in registers: as a constant it is built anew for every product
#pragma unroll
  for (int e = 0; e < 4; ++e) asm volatile("mov.b32 %0, 0x80088008;" : "=r"(eight[e]));
  const int tr = token_of<D>(r);
  const int k_at = tr * H::ROW + (D == 64 ? 8 * l : 16 * l), par_at = 2 * STEP * H::ROW + tr * H::PAR;
  const int va_at = (STEP + token_of<D>(2 * l)) * H::ROW + (D / 16) * r, vb_at = (STEP + token_of<D>(2 * l + 1)) * H::ROW + (D / 16) * r;

  int stage = 0;
  uint32_t parity = 0;
  // WHOLE: every key of both tiles is visible
  auto take = [&](auto whole_tiles, const unsigned char* st, int base) {
    constexpr bool WHOLE = decltype(whole_tiles)::value;
    float x[TILES][NT][4];
    uint32_t vp[TILES][2][H::G];
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      const unsigned char* tile = st + t * H::TILE;
      uint32_t kw[2][H::WORDS], kp[2][H::G];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const unsigned char *kr = tile + k_at + 8 * half * H::ROW, *pr = tile + par_at + 8 * half * H::PAR;
        if constexpr (D == 64) {
          *reinterpret_cast<uint2*>(&kw[half][0]) = *reinterpret_cast<const uint2*>(kr);
          kp[half][0] = *reinterpret_cast<const uint32_t*>(pr);
          vp[t][half][0] = *reinterpret_cast<const uint32_t*>(pr + STEP * H::PAR);
        } else if constexpr (D == 128) {
          *reinterpret_cast<uint4*>(&kw[half][0]) = *reinterpret_cast<const uint4*>(kr);
          *reinterpret_cast<uint2*>(&kp[half][0]) = *reinterpret_cast<const uint2*>(pr);
          *reinterpret_cast<uint2*>(&vp[t][half][0]) = *reinterpret_cast<const uint2*>(pr + STEP * H::PAR);
        } else {
          *reinterpret_cast<uint4*>(&kw[half][0]) = *reinterpret_cast<const uint4*>(kr);
          *reinterpret_cast<uint4*>(&kw[half][4]) = *reinterpret_cast<const uint4*>(kr + 64);
          *reinterpret_cast<uint4*>(&kp[half][0]) = *reinterpret_cast<const uint4*>(pr);
          *reinterpret_cast<uint4*>(&vp[t][half][0]) = *reinterpret_cast<const uint4*>(pr + STEP * H::PAR);
        }
      }
      float acc[NT][H::G][4];
#pragma unroll
      for (int j = 0; j < H::WORDS; ++j) {
        const uint32_t w0 = kw[0][j], w1 = kw[1][j], u0 = w0 >> 8, u1 = w1 >> 8;
        const uint32_t a0[4] = {tiny_of<0>(w0, u0), tiny_of<0>(w1, u1), tiny_of<1>(w0, u0), tiny_of<1>(w1, u1)};
        const uint32_t a1[4] = {tiny_of<2>(w0, u0), tiny_of<2>(w1, u1), tiny_of<3>(w0, u0), tiny_of<3>(w1, u1)};
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if (j < H::G)  // the words of the groups come in turn: the first of each starts its sum
            mma_bf16_first(acc[n][H::group(j)], a0, q[n][j][0], q[n][j][1]);
          else
            mma_bf16(acc[n][H::group(j)], a0, q[n][j][0], q[n][j][1]);
          mma_bf16(acc[n][H::group(j)], a1, q[n][j][2], q[n][j][3]);
        }
      }
      bool in[2] = {true, true};
      if (!WHOLE) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int key = base + t * STEP + tr + 8 * half;
          in[half] = key < end && key >= sl.lo;
#pragma unroll
          for (int g = 0; g < H::G; ++g)
            if (!in[half]) kp[half][g] = vp[t][half][g] = 0;  // rows that are nobody's may hold anything
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float(&y)[4] = x[t][n];
#pragma unroll
        for (int g = 0; g < H::G; ++g) {
          const float s0 = q4_s(kp[0][g]), s1 = q4_s(kp[1][g]);
          y[0] = g ? y[0] + s0 * acc[n][g][0] : s0 * acc[n][g][0];
          y[1] = g ? y[1] + s0 * acc[n][g][1] : s0 * acc[n][g][1];
          y[2] = g ? y[2] + s1 * acc[n][g][2] : s1 * acc[n][g][2];
          y[3] = g ? y[3] + s1 * acc[n][g][3] : s1 * acc[n][g][3];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] *= undo[n][e & 1];
#pragma unroll
        for (int g = 0; g < H::G; ++g) {
          const float z0 = q4_z(kp[0][g]), z1 = q4_z(kp[1][g]);
          y[0] += z0 * qsum[n][g][0];
          y[1] += z0 * qsum[n][g][1];
          y[2] += z1 * qsum[n][g][0];
          y[3] += z1 * qsum[n][g][1];
        }
        if (!WHOLE) {
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = in[e >> 1] ? y[e] : -INFINITY;
        }
      }
    }
    // The maximum moves only when it would be passed by a factor of 2^8 (a weight is 2^8 at most, which float32 sums do not mind), the
    // lift when a scale would leave its range; hardly ever after the first tiles.
    float top[NT][2], scale = 0.f;
    bool far = false;
#pragma unroll
    for (int t = 0; t < TILES; ++t)
#pragma unroll
      for (int g = 0; g < H::G; ++g) scale = fmaxf(scale, fmaxf(q4_s(vp[t][0][g]), q4_s(vp[t][1][g])));
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        top[n][c] = fmaxf(fmaxf(x[0][n][c], x[0][n][c + 2]), fmaxf(x[1][n][c], x[1][n][c + 2]));
        far = far || top[n][c] > m[n][c] + 8.f;
      }
    if (__any_sync(0xffffffffu, far || scale > most_scale)) {
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) scale = fmaxf(scale, __shfl_xor_sync(0xffffffffu, scale, d));
      float down = 1.f;
      if (scale > most_scale) {
        const int now = min(120, 227 - (int)(__float_as_uint(scale) >> 23));  // 100 less its exponent
        down = most_scale < 0.f ? 1.f : power_of_two(max(-126, now - T));
        T = now;
        lift = power_of_two(T);
        most_scale = power_of_two(min(127, 115 - T));
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float now = fmaxf(m[n][c], top[n][c]);
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, d));
          const float f = exp2_fast(m[n][c] - now), fd = f * down;
          m[n][c] = now;
          sum[n][c] *= f;
#pragma unroll
          for (int g = 0; g < H::G; ++g) {
            oc[n][g][c] *= f, oz[n][g][c] *= fd, oz[n][g][c + 2] *= fd;
#pragma unroll
            for (int j = 0; j < 4; ++j) o[n][g][j][c] *= fd, o[n][g][j][c + 2] *= fd;
          }
        }
    }
    uint32_t w[TILES][NT][H::G][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float off[2] = {4.f - m[n][0], 4.f - m[n][1]};
#pragma unroll
      for (int t = 0; t < TILES; ++t) {
        float(&y)[4] = x[t][n];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = exp2_fast(y[e] + off[e & 1]);
        sum[n][0] += y[0] + y[2];
        sum[n][1] += y[1] + y[3];
#pragma unroll
        for (int g = 0; g < H::G; ++g) {
          const float s0 = q4_s(vp[t][0][g]), s1 = q4_s(vp[t][1][g]);
          const float c0 = q4_z(vp[t][0][g]) + 8.f * s0, c1 = q4_z(vp[t][1][g]) + 8.f * s1;
          oc[n][g][0] += y[0] * c0 + y[2] * c1;
          oc[n][g][1] += y[1] * c0 + y[3] * c1;
          // weight times scale is rounded to bfloat16 for the product, as weights are everywhere in this engine's 16-bit attention
          const float l0 = s0 * lift, l1 = s1 * lift;
          w[t][n][g][0] = transposed(pack_bf16(y[0] * l0, y[1] * l0));
          w[t][n][g][1] = transposed(pack_bf16(y[2] * l1, y[3] * l1));
        }
      }
    }
    // ---- results: of each tile the tokens of rows 2l, 2l + 1, 2l + 8, 2l + 9
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      const unsigned char* tile = st + t * H::TILE;
      uint32_t vw[4][H::G];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const unsigned char* vr = tile + (e & 1 ? vb_at : va_at) + 8 * (e >> 1) * H::ROW;
        if constexpr (D == 64) vw[e][0] = *reinterpret_cast<const uint32_t*>(vr);
        if constexpr (D == 128) *reinterpret_cast<uint2*>(&vw[e][0]) = *reinterpret_cast<const uint2*>(vr);
        if constexpr (D == 256) *reinterpret_cast<uint4*>(&vw[e][0]) = *reinterpret_cast<const uint4*>(vr);
      }
#pragma unroll
      for (int g = 0; g < H::G; ++g) {
        const uint32_t lo0 = __byte_perm(vw[0][g], vw[1][g], 0x5410), hi0 = __byte_perm(vw[0][g], vw[1][g], 0x7632);
        const uint32_t lo1 = __byte_perm(vw[2][g], vw[3][g], 0x5410), hi1 = __byte_perm(vw[2][g], vw[3][g], 0x7632);
        const uint32_t lu0 = lo0 >> 8, hu0 = hi0 >> 8, lu1 = lo1 >> 8, hu1 = hi1 >> 8;
        const uint32_t v0[4] = {tiny_of<0>(lo0, lu0), tiny_of<0>(hi0, hu0), tiny_of<0>(lo1, lu1), tiny_of<0>(hi1, hu1)};
        const uint32_t v1[4] = {tiny_of<1>(lo0, lu0), tiny_of<1>(hi0, hu0), tiny_of<1>(lo1, lu1), tiny_of<1>(hi1, hu1)};
        const uint32_t v2[4] = {tiny_of<2>(lo0, lu0), tiny_of<2>(hi0, hu0), tiny_of<2>(lo1, lu1), tiny_of<2>(hi1, hu1)};
        const uint32_t v3[4] = {tiny_of<3>(lo0, lu0), tiny_of<3>(hi0, hu0), tiny_of<3>(lo1, lu1), tiny_of<3>(hi1, hu1)};
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma_bf16(oz[n][g], eight, w[t][n][g][0], w[t][n][g][1]);
          mma_bf16(o[n][g][0], v0, w[t][n][g][0], w[t][n][g][1]);
          mma_bf16(o[n][g][1], v1, w[t][n][g][0], w[t][n][g][1]);
          mma_bf16(o[n][g][2], v2, w[t][n][g][0], w[t][n][g][1]);
          mma_bf16(o[n][g][3], v3, w[t][n][g][0], w[t][n][g][1]);
        }
      }
    }
  };
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
    if (base + STEP * TILES <= end && base >= sl.lo)  // (of one mind over the warp)
      take(std::true_type(), st, base);
    else
      take(std::false_type(), st, base);
    __syncwarp();
    load_step(stage ? stage - 1 : STAGES - 1);
    if (++stage == STAGES) stage = 0, parity ^= 1;
  }
  pdl_launch_dependents();

  // ---- the warps' results: [warp][query][D + 4] and [warp][query][2] over the rings
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
      float total = sum[n][c];
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) {
        total += __shfl_xor_sync(0xffffffffu, total, d);
#pragma unroll
        for (int g = 0; g < H::G; ++g) oc[n][g][c] += __shfl_xor_sync(0xffffffffu, oc[n][g][c], d);
      }
      if (r == 0) {
        ml[(warp * QS + h) * 2] = m[n][c];
        ml[(warp * QS + h) * 2 + 1] = total;
      }
      float* row = ow + (warp * QS + h) * PITCH;
      const float up = power_of_two(69 - T), up_odd = up * 0.0625f;  // 2^(133 - T) in two steps
#pragma unroll
      for (int g = 0; g < H::G; ++g) {
        const float base = oz[n][g][c] * 0x1p64f * up + oc[n][g][c];
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = o[n][g][e & 3][c + (e >> 2) * 2] * 0x1p64f * (e & 1 ? up_odd : up) + base;
        store8(row + 64 * g + 8 * r, y);
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
      *reinterpret_cast<float4*>(a.mid_o + where * D + d) = make_float4(y[0] / den, y[1] / den, y[2] / den, y[3] / den);
      if (d == 0) a.mid_lse[where] = top + log2f(den) - 4.f;
    } else {
      uint2 packed;
      packed.x = pack_bf16(y[0] / den, y[1] / den);
      packed.y = pack_bf16(y[2] / den, y[3] / den);
      *reinterpret_cast<uint2*>(a.out + (out_row + h) * D + d) = packed;
      if (a.lse && d == 0) a.lse[out_row + h] = (top + log2f(den) - 4.f) * LN_2;
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
      if (a.lse && d == 0) a.lse[out_row + h] = count > 0 ? (top + log2f(den) - 4.f) * LN_2 : -INFINITY;
    }
    cluster_sync_all();  // a block's results are read until here
  }
}

// Slices of a (sequence, head), in order: a warp per head, four slices' loads in flight.
template <int D> __global__ void __launch_bounds__(THREADS) merge_4bit_kernel(Decode a, int heads) {
  pdl_wait();
  pdl_launch_dependents();
  const int item = blockIdx.x * WARPS + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (item >= heads) return;
  const int slot = item / a.nq, h = item - slot * a.nq;
  const int seq = a.seq_list ? a.seq_list[slot] : slot;
  const int tok = a.cu_seqlens[seq];
  const int slices = Slice(a, seq, 0).count(a);
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
  if (a.lse && lane == 0) a.lse[(long)tok * a.nq + h] = slices > 0 ? (top + log2f(den)) * LN_2 : -INFINITY;
}

template <int D, int NT, bool BULK, bool CLUSTER> int launch_decode_as(const Decode& a, int num_seqs, cudaStream_t stream) {
  constexpr int ring = WARPS * STAGES * TILES * Head<D>::TILE;
  constexpr int joined = (WARPS * 8 * NT * (D + 4 + 2) + (CLUSTER ? 8 * NT * (D + 2) : 0)) * 4;
  constexpr int smem = ring > joined ? ring : joined;
  auto kernel = decode_4bit_kernel<D, NT, BULK, CLUSTER>;
  static bool once[Q3_MAX_DEVICES];
  const int dev = q3_current_device();
  if (!once[dev]) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return Q3_ERR_LAUNCH;
    if (CLUSTER && cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) return Q3_ERR_LAUNCH;
    once[dev] = true;
  }
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
    err = launch_pdl(merge_4bit_kernel<D>, dim3((heads + WARPS - 1) / WARPS), dim3(THREADS), 0, stream, a, heads);
  }
  return err == cudaSuccess ? Q3_OK : Q3_ERR_LAUNCH;
}
template <int D, int NT> int launch_decode(const Decode& a, int num_seqs, cudaStream_t stream) {
  const bool bulk = a.ps % STEP == 0, cluster = a.splits > 1 && !a.mid_o;
  if (bulk) return cluster ? launch_decode_as<D, NT, true, true>(a, num_seqs, stream) : launch_decode_as<D, NT, true, false>(a, num_seqs, stream);
  return cluster ? launch_decode_as<D, NT, false, true>(a, num_seqs, stream) : launch_decode_as<D, NT, false, false>(a, num_seqs, stream);
}

// ---- sums of attention weights -----------------------------------------------------------------------------------------------------
// mass[key] += sum over a sequence's last `observe` tokens and the query heads of the kv head of 2^(score - log sum of the row).  Rows are
// (token, head of the group), token by token; the scores' tiles are those of decode attention.  A cached token's sum belongs to one warp's
// lane: no atomics, the same bits every time.  Sums are float32; a weight is 2^x to 2 units in the last place (2^-22 of itself), and the
// log sum that is taken off, a float32 too, is good to 2^-23 of the row's scores: beyond some 2^20 weights are no more than a guess, but
// no sum gets more than one for each row.
//   few rows (up to 16: single tokens)  mass_few_kernel: the queries stay in registers, keys stream past them, 16 a warp at a time, the next
//                                       ones' bytes on their way; reads half of what the attention reads.  Instructions bound it: 96,700
//                                       tokens of 8 kv heads of 128 channels in 29 us (2.0 TB/s); with two tiles on their way no less.
//   more                                mass_rows_kernel: the rows' log sums, keys cut into slices so that all SMs have some (left out
//                                       where the attention has them); mass_columns_kernel: a warp keeps 16 keys and goes through the
//                                       rows, which the block has turned into operands in shared memory.
struct Mass {
  const bf16* q;
  int q_stride;
  const unsigned char* pages;
  int num_pages;
  const int *block_table, *kv_lens, *cu_seqlens;
  int max_pages, nq, nkv, ps, max_len, observe, slices, num_seqs;
  float scale_log2;
  float* lse;    // [tokens][nq], natural logarithms
  float2* part;  // null (the log sums are in lse), or [tokens][nq][slices]: maximum and sum
  float* mass;
};

constexpr int ROWS_STEP = STEP * WARPS;  // keys of a block at a time

template <int D> struct KeyBytes {  // what a lane holds of 16 keys as they are stored
  uint32_t w[2][Head<D>::WORDS], p[2][Head<D>::G];
  // rows of keys first + r and first + r + 8; what is not there is zero.  `page`, `row`: where they lie
  __device__ __forceinline__ void load(const Mass& m, const Q4Page& L, int kvh, const int (&page)[2], const int (&row)[2], int lane) {
    using H = Head<D>;
    const int l = lane & 3;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
      for (int j = 0; j < H::WORDS; ++j) w[half][j] = 0;
#pragma unroll
      for (int g = 0; g < H::G; ++g) p[half][g] = 0;
      if ((uint32_t)page[half] < (uint32_t)m.num_pages) {
        const unsigned char* rec = m.pages + ((long)page[half] * m.nkv + kvh) * L.record;
        const unsigned char* codes = rec + (long)row[half] * H::ROW;
        const unsigned char* par = rec + L.kpar + (long)row[half] * H::PAR;
        if constexpr (D == 64) {
          *reinterpret_cast<uint2*>(&w[half][0]) = *reinterpret_cast<const uint2*>(codes + 8 * l);
          p[half][0] = *reinterpret_cast<const uint32_t*>(par);
        } else if constexpr (D == 128) {
          *reinterpret_cast<uint4*>(&w[half][0]) = *reinterpret_cast<const uint4*>(codes + 16 * l);
          *reinterpret_cast<uint2*>(&p[half][0]) = *reinterpret_cast<const uint2*>(par);
        } else {
          *reinterpret_cast<uint4*>(&w[half][0]) = *reinterpret_cast<const uint4*>(codes + 16 * l);
          *reinterpret_cast<uint4*>(&w[half][4]) = *reinterpret_cast<const uint4*>(codes + 16 * (l + 4));
          *reinterpret_cast<uint4*>(&p[half][0]) = *reinterpret_cast<const uint4*>(par);
        }
      }
    }
  }
  // keys first + r and first + r + 8 of a sequence, as far as they lie in front of `end`
  __device__ __forceinline__ void load_at(const Mass& m, const Q4Page& L, const int* bt, int kvh, int first, int end, int lane) {
    int page[2], row[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int key = first + (lane >> 2) + 8 * half, i = key / m.ps;
      page[half] = key < end ? bt[i] : -1;
      row[half] = key - i * m.ps;
    }
    load(m, L, kvh, page, row, lane);
  }
};

// Sixteen keys of one page (page sizes that are multiples of 16): one place for all of them.
template <int D> struct PageKeys {
  long code_at, par_at;  // this lane's first bytes in a tile
  __device__ __forceinline__ PageKeys(const Q4Page& L, int lane)
      : code_at((lane >> 2) * Head<D>::ROW + (D == 64 ? 8 : 16) * (lane & 3)), par_at(L.kpar + (lane >> 2) * Head<D>::PAR) {}
  __device__ __forceinline__ void load(KeyBytes<D>& b, const Mass& m, const Q4Page& L, int kvh, int page, int row) const {
    using H = Head<D>;
    if ((uint32_t)page >= (uint32_t)m.num_pages) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int j = 0; j < H::WORDS; ++j) b.w[half][j] = 0;
#pragma unroll
        for (int g = 0; g < H::G; ++g) b.p[half][g] = 0;
      }
      return;
    }
    const unsigned char* rec = m.pages + ((long)page * m.nkv + kvh) * L.record;
    const unsigned char *codes = rec + ((long)row * H::ROW + code_at), *par = rec + ((long)row * H::PAR + par_at);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if constexpr (D == 64) {
        *reinterpret_cast<uint2*>(&b.w[half][0]) = *reinterpret_cast<const uint2*>(codes + 8 * half * H::ROW);
        b.p[half][0] = *reinterpret_cast<const uint32_t*>(par + 8 * half * H::PAR);
      } else if constexpr (D == 128) {
        *reinterpret_cast<uint4*>(&b.w[half][0]) = *reinterpret_cast<const uint4*>(codes + 8 * half * H::ROW);
        *reinterpret_cast<uint2*>(&b.p[half][0]) = *reinterpret_cast<const uint2*>(par + 8 * half * H::PAR);
      } else {
        *reinterpret_cast<uint4*>(&b.w[half][0]) = *reinterpret_cast<const uint4*>(codes + 8 * half * H::ROW);
        *reinterpret_cast<uint4*>(&b.w[half][4]) = *reinterpret_cast<const uint4*>(codes + 8 * half * H::ROW + 64);
        *reinterpret_cast<uint4*>(&b.p[half][0]) = *reinterpret_cast<const uint4*>(par + 8 * half * H::PAR);
      }
    }
  }
};

template <int D> struct KeyTile {  // 16 keys as A fragments
  uint32_t a[Head<D>::WORDS][2][4];
  float s[2][Head<D>::G], z[2][Head<D>::G];
  __device__ __forceinline__ void take(const KeyBytes<D>& b) {
    using H = Head<D>;
    const auto& w = b.w;
    const auto& p = b.p;
#pragma unroll
    for (int g = 0; g < H::G; ++g) {
      s[0][g] = q4_s(p[0][g]), s[1][g] = q4_s(p[1][g]);
      z[0][g] = q4_z(p[0][g]), z[1][g] = q4_z(p[1][g]);
    }
#pragma unroll
    for (int j = 0; j < H::WORDS; ++j) {
      const uint32_t w0 = w[0][j], w1 = w[1][j], u0 = w0 >> 8, u1 = w1 >> 8;
      a[j][0][0] = tiny_of<0>(w0, u0), a[j][0][1] = tiny_of<0>(w1, u1), a[j][0][2] = tiny_of<1>(w0, u0), a[j][0][3] = tiny_of<1>(w1, u1);
      a[j][1][0] = tiny_of<2>(w0, u0), a[j][1][1] = tiny_of<2>(w1, u1), a[j][1][2] = tiny_of<3>(w0, u0), a[j][1][3] = tiny_of<3>(w1, u1);
    }
  }
  // scores (times scale, in powers of two): x[0], x[1] of key r and queries 2l, 2l + 1; x[2], x[3] of key r + 8
  __device__ __forceinline__ void scores(float (&x)[4], const uint32_t (&q)[Head<D>::WORDS][4], const float (&undo)[2],
                                         const float (&qsum)[Head<D>::G][2]) const {
    using H = Head<D>;
    float acc[H::G][4];
#pragma unroll
    for (int j = 0; j < H::WORDS; ++j) {
      if (j < H::G)
        mma_bf16_first(acc[H::group(j)], a[j][0], q[j][0], q[j][1]);
      else
        mma_bf16(acc[H::group(j)], a[j][0], q[j][0], q[j][1]);
      mma_bf16(acc[H::group(j)], a[j][1], q[j][2], q[j][3]);
    }
    x[0] = x[1] = x[2] = x[3] = 0.f;
#pragma unroll
    for (int g = 0; g < H::G; ++g) {
      x[0] += s[0][g] * acc[g][0];
      x[1] += s[0][g] * acc[g][1];
      x[2] += s[1][g] * acc[g][2];
      x[3] += s[1][g] * acc[g][3];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] *= undo[e & 1];
#pragma unroll
    for (int g = 0; g < H::G; ++g) {
      x[0] += z[0][g] * qsum[g][0];
      x[1] += z[0][g] * qsum[g][1];
      x[2] += z[1][g] * qsum[g][0];
      x[3] += z[1][g] * qsum[g][1];
    }
  }
};

// The observed rows of a sequence: first token, how many tokens, and the sequence's length without them.
struct Rows {
  int first, count, before;
  __device__ __forceinline__ Rows(const Mass& a, int seq) {
    const int q_len = a.cu_seqlens[seq + 1] - a.cu_seqlens[seq];
    const int kv_len = min(a.kv_lens[seq], a.max_len);
    count = max(0, min(min(a.observe, q_len), kv_len));
    first = a.cu_seqlens[seq + 1] - count;
    before = kv_len - count;
  }
};

__device__ __forceinline__ float at_most(float y, int rows) { return y > (float)rows ? (float)rows : y; }  // (what is no number stays none)

// Log sums: grid (slice, block of 8 NT rows, sequence x kv head); a warp takes every fourth 16 keys of the slice.
template <int D, int NT> __global__ void __launch_bounds__(THREADS) mass_rows_kernel(Mass a) {
  using H = Head<D>;
  pdl_wait();
  pdl_launch_dependents();
  const int seq = blockIdx.z / a.nkv, kvh = blockIdx.z % a.nkv, slice = blockIdx.x, row0 = blockIdx.y * 8 * NT;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r = lane >> 2, l = lane & 3, R = a.nq / a.nkv;
  const Rows rows(a, seq);
  if (row0 >= rows.count * R) return;
  const int kv_len = rows.before + rows.count;
  const int per = ((kv_len + a.slices - 1) / a.slices + 63) & ~63;
  const int begin = slice * per, end = min(kv_len, begin + per);
  const Q4Page L(D, H::G, a.ps);
  const int* bt = a.block_table + (long)seq * a.max_pages;
  uint32_t q[NT][H::WORDS][4];
  float qsum[NT][H::G][2], undo[NT][2], m[NT][2], sum[NT][2];
  int sees[NT][2];  // the last key that the row's token sees
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int row = row0 + 8 * n + r, i = row / R;
    load_query_tiny<D>(q[n], undo[n], qsum[n], i < rows.count ? a.q + (long)(rows.first + i) * a.q_stride + (long)(kvh * R + row % R) * D : nullptr,
                       a.scale_log2, lane);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      m[n][c] = MINUS_BIG, sum[n][c] = 0.f;
      sees[n][c] = min(end - 1, rows.before + (row0 + 8 * n + 2 * l + c) / R);
    }
  }
  KeyBytes<D> bytes;
  bytes.load_at(a, L, bt, kvh, begin + STEP * warp, end, lane);
  for (int first = begin + STEP * warp; first < end; first += STEP * WARPS) {
    KeyTile<D> k;
    k.take(bytes);
    bytes.load_at(a, L, bt, kvh, first + STEP * WARPS, end, lane);  // (on its way while this tile is worked on)
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float x[4];
      k.scores(x, q[n], undo[n], qsum[n]);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float x0 = first + r <= sees[n][c] ? x[c] : -INFINITY, x1 = first + r + 8 <= sees[n][c] ? x[c + 2] : -INFINITY;
        const float top = fmaxf(m[n][c], fmaxf(x0, x1));
        sum[n][c] = sum[n][c] * exp2_fast(m[n][c] - top) + exp2_fast(x0 - top) + exp2_fast(x1 - top);
        m[n][c] = top;
      }
    }
  }
  __shared__ float2 joined[WARPS][8 * NT];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) {
        const float om = __shfl_xor_sync(0xffffffffu, m[n][c], d), os = __shfl_xor_sync(0xffffffffu, sum[n][c], d);
        const float top = fmaxf(m[n][c], om);
        sum[n][c] = sum[n][c] * exp2_fast(m[n][c] - top) + os * exp2_fast(om - top);
        m[n][c] = top;
      }
      if (r == 0) joined[warp][8 * n + 2 * l + c] = make_float2(m[n][c], sum[n][c]);
    }
  __syncthreads();
  const int row = row0 + tid;
  if (tid < 8 * NT && row < rows.count * R) {
    float top = MINUS_BIG, den = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) top = fmaxf(top, joined[w][tid].x);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) den += joined[w][tid].y * exp2_fast(joined[w][tid].x - top);
    const long at = (long)(rows.first + row / R) * a.nq + kvh * R + row % R;
    if (a.part)
      a.part[at * a.slices + slice] = make_float2(top, den);
    else
      a.lse[at] = (top + log2f(den)) * LN_2;
  }
}

// The log sum of a row in powers of two: as the attention wrote it, or its slices joined.
__device__ __forceinline__ float row_log2(const Mass& a, long at) {
  if (!a.part) return a.lse[at] * LOG2_E;
  float top = MINUS_BIG, den = 0.f;
  for (int s = 0; s < a.slices; s += 8) {  // eight loads at a time
    float2 y[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) y[u] = s + u < a.slices ? a.part[at * a.slices + s + u] : make_float2(MINUS_BIG, 0.f);
    float now = top;
#pragma unroll
    for (int u = 0; u < 8; ++u) now = fmaxf(now, y[u].x);
    den *= exp2_fast(top - now);
#pragma unroll
    for (int u = 0; u < 8; ++u) den += y[u].y * exp2_fast(y[u].x - now);
    top = now;
  }
  return top + log2f(den);
}

// Column sums of many rows: grid (blocks of 16 * COLUMN_WARPS keys, kv head, sequence).
constexpr int COLUMN_WARPS = 8;
constexpr int COLUMN_TILES = 8;  // tiles of 8 rows in shared memory at a time

template <int D> struct RowTile {  // 8 rows as operands, as each lane reads them
  uint32_t q[Head<D>::WORDS][32][4];
  float undo[32][2], sums[Head<D>::G][32][2], lse2[32][2];
  int sees[32][2];
};

template <int D> __global__ void __launch_bounds__(32 * COLUMN_WARPS) mass_columns_kernel(Mass a) {
  using H = Head<D>;
  extern __shared__ __align__(128) unsigned char smem[];
  RowTile<D>* tiles = reinterpret_cast<RowTile<D>*>(smem);
  pdl_wait();
  pdl_launch_dependents();
  const int seq = blockIdx.z, kvh = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, l = lane & 3, R = a.nq / a.nkv;
  const Rows rows(a, seq);
  const int kv_len = rows.before + rows.count;
  const int block_first = blockIdx.x * COLUMN_WARPS * STEP, first = block_first + warp * STEP;
  if (block_first >= kv_len || rows.count == 0) return;
  const Q4Page L(D, H::G, a.ps);
  const int* bt = a.block_table + (long)seq * a.max_pages;
  KeyTile<D> k;
  {
    KeyBytes<D> bytes;
    bytes.load_at(a, L, bt, kvh, first, kv_len, lane);
    k.take(bytes);
  }
  float total[2] = {0.f, 0.f};
  // rows of tokens that see none of the block's keys are left out
  const int start = max(0, block_first - rows.before) * R & ~7, stop = rows.count * R;
  for (int portion = start; portion < stop; portion += 8 * COLUMN_TILES) {
    __syncthreads();
    for (int n = warp; n < COLUMN_TILES && portion + 8 * n < stop; n += COLUMN_WARPS) {
      RowTile<D>& t = tiles[n];
      uint32_t q[H::WORDS][4];
      float undo[2], sums[H::G][2];
      const int own = portion + 8 * n + r, own_i = own / R;
      load_query_tiny<D>(q, undo, sums,
                         own_i < rows.count ? a.q + (long)(rows.first + own_i) * a.q_stride + (long)(kvh * R + own % R) * D : nullptr,
                         a.scale_log2, lane);
#pragma unroll
      for (int j = 0; j < H::WORDS; ++j) *reinterpret_cast<uint4*>(t.q[j][lane]) = make_uint4(q[j][0], q[j][1], q[j][2], q[j][3]);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int row = portion + 8 * n + 2 * l + c, i = row / R;
        const bool is = i < rows.count;
        t.undo[lane][c] = undo[c];
#pragma unroll
        for (int g = 0; g < H::G; ++g) t.sums[g][lane][c] = sums[g][c];
        t.lse2[lane][c] = is ? row_log2(a, (long)(rows.first + i) * a.nq + kvh * R + row % R) : 0.f;
        t.sees[lane][c] = is ? rows.before + i : -1;
      }
    }
    __syncthreads();
    if (first >= kv_len) continue;
    for (int n = 0; n < COLUMN_TILES && portion + 8 * n < stop; ++n) {
      const RowTile<D>& t = tiles[n];
      uint32_t q[H::WORDS][4];
      float sums[H::G][2];
#pragma unroll
      for (int j = 0; j < H::WORDS; ++j) {
        const uint4 v = *reinterpret_cast<const uint4*>(t.q[j][lane]);
        q[j][0] = v.x, q[j][1] = v.y, q[j][2] = v.z, q[j][3] = v.w;
      }
      const float2 undo2 = *reinterpret_cast<const float2*>(t.undo[lane]), lse2 = *reinterpret_cast<const float2*>(t.lse2[lane]);
      const int2 sees = *reinterpret_cast<const int2*>(t.sees[lane]);
#pragma unroll
      for (int g = 0; g < H::G; ++g) sums[g][0] = t.sums[g][lane][0], sums[g][1] = t.sums[g][lane][1];
      const float undo[2] = {undo2.x, undo2.y};
      float x[4];
      k.scores(x, q, undo, sums);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = first + r + 8 * (e >> 1);
        total[e >> 1] += key <= (e & 1 ? sees.y : sees.x) ? exp2_fast(x[e] - (e & 1 ? lse2.y : lse2.x)) : 0.f;
      }
    }
  }
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    float y = total[half];
    y += __shfl_xor_sync(0xffffffffu, y, 1);
    y += __shfl_xor_sync(0xffffffffu, y, 2);
    y = at_most(y, rows.count * R);
    const int key = first + r + 8 * half;
    if (l == 0 && key < kv_len) {
      const int page = bt[key / a.ps];
      if (page >= 0 && page < a.num_pages) a.mass[((long)page * a.nkv + kvh) * a.ps + key % a.ps] += y;
    }
  }
}

// Few rows: grid (slice, kv head, sequence); a warp takes every fourth 16 keys of the slice.  Two tiles are on their way while one is
// worked on: the first one's bytes, and the pages of the second, whose bytes wait for them.  NT tiles of 8 rows.
// WHOLE: page sizes that are multiples of 16, so that a tile's keys lie in one page and have one lookup (29 us; a lookup a key takes 33).
template <int D, int NT, bool WHOLE> __global__ void __launch_bounds__(THREADS, D == 256 ? 2 : 4) mass_few_kernel(Mass a) {
  using H = Head<D>;
  pdl_wait();
  pdl_launch_dependents();
  const int seq = blockIdx.z, kvh = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, l = lane & 3, R = a.nq / a.nkv;
  const Rows rows(a, seq);
  const int kv_len = rows.before + rows.count;
  const int per = ((a.max_len + (int)gridDim.x - 1) / (int)gridDim.x + ROWS_STEP - 1) / ROWS_STEP * ROWS_STEP;
  const int begin = blockIdx.x * per, end = min(kv_len, begin + per);
  if (begin >= end || rows.count == 0) return;
  const Q4Page L(D, H::G, a.ps);
  const int* bt = a.block_table + (long)seq * a.max_pages;
  // this lane's two keys of the tile to come (or the whole tile): page of the sequence and row, moved on by a step of the block at a time
  constexpr int PLACES = WHOLE ? 1 : 2;
  int at_page[PLACES], row[PLACES];
#pragma unroll
  for (int half = 0; half < PLACES; ++half) {
    const int key = begin + warp * STEP + (WHOLE ? 0 : r + 8 * half);
    at_page[half] = key / a.ps, row[half] = key - at_page[half] * a.ps;
  }
  const int go_pages = ROWS_STEP / a.ps, go_rows = ROWS_STEP - go_pages * a.ps;
  int page[PLACES], next_row[PLACES];
  auto look_up = [&](int first) {
#pragma unroll
    for (int half = 0; half < PLACES; ++half) {
      page[half] = first + (WHOLE ? 0 : r + 8 * half) < end ? bt[at_page[half]] : -1;
      next_row[half] = row[half];
      at_page[half] += go_pages, row[half] += go_rows;
      if (row[half] >= a.ps) row[half] -= a.ps, ++at_page[half];
    }
  };
  const PageKeys<D> tile(L, lane);
  KeyBytes<D> bytes;
  float* cell[2];
  float old[2];
  auto fetch = [&](int first) {  // the bytes and sums of the keys looked up last
    if constexpr (WHOLE)
      tile.load(bytes, a, L, kvh, page[0], next_row[0]);
    else
      bytes.load(a, L, kvh, page, next_row, lane);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int at = WHOLE ? 0 : half;
      const bool own = l == 0 && (uint32_t)page[at] < (uint32_t)a.num_pages && (!WHOLE || first + r + 8 * half < end);
      cell[half] = own ? a.mass + ((long)page[at] * a.nkv + kvh) * a.ps + next_row[at] + (WHOLE ? r + 8 * half : 0) : nullptr;
      old[half] = own ? *cell[half] : 0.f;
    }
  };
  int first = begin + warp * STEP;
  look_up(first);
  uint32_t q[NT][H::WORDS][4];
  float qsum[NT][H::G][2], undo[NT][2], lse2[NT][2];
  int sees[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int own = 8 * n + r, own_i = own / R;
    load_query_tiny<D>(q[n], undo[n], qsum[n],
                       own_i < rows.count ? a.q + (long)(rows.first + own_i) * a.q_stride + (long)(kvh * R + own % R) * D : nullptr, a.scale_log2, lane);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int at = 8 * n + 2 * l + c, i = at / R;
      const bool is = i < rows.count;
      lse2[n][c] = is ? row_log2(a, (long)(rows.first + i) * a.nq + kvh * R + at % R) : 0.f;
      sees[n][c] = is ? rows.before + i : -1;
    }
  }
  fetch(first);
  look_up(first + ROWS_STEP);
  for (; first < end; first += ROWS_STEP) {
    KeyTile<D> k;
    k.take(bytes);
    float* const mine[2] = {cell[0], cell[1]};
    const float was[2] = {old[0], old[1]};
    fetch(first + ROWS_STEP);
    look_up(first + 2 * ROWS_STEP);
    float total[2] = {0.f, 0.f};
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float x[4];
      k.scores(x, q[n], undo[n], qsum[n]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = first + r + 8 * (e >> 1);
        total[e >> 1] += key <= sees[n][e & 1] ? exp2_fast(x[e] - lse2[n][e & 1]) : 0.f;
      }
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float y = total[half];
      y += __shfl_xor_sync(0xffffffffu, y, 1);
      y += __shfl_xor_sync(0xffffffffu, y, 2);
      if (mine[half]) *mine[half] = was[half] + at_most(y, rows.count * R);
    }
  }
}

// float32, and head sizes that the tiles do not take: the same sums on the FMA pipes.
template <typename T>
__device__ __forceinline__ float score_of(const T* q, const unsigned char* rec, const Q4Page& L, int row, int D, int G) {
  const uint32_t* code = reinterpret_cast<const uint32_t*>(rec + (long)row * L.half);
  const uint32_t* par = reinterpret_cast<const uint32_t*>(rec + L.kpar + (long)row * L.par);
  const int per = D / 8 / G;
  float sum = 0.f;
  for (int g = 0; g < G; ++g) {
    const float s = q4_s(par[g]), z = q4_z(par[g]);
    for (int i = 0; i < per; ++i) {
      const uint32_t w = code[i * G + g];
      float x[8];
      load8(q + (g * per + i) * 8, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += x[e] * (z + (float)((w >> (4 * e)) & 15u) * s);
    }
  }
  return sum;
}

template <typename T> __global__ void mass_rows_general_kernel(Mass a, const T* q, int D, int G) {  // grid (observed token, head, sequence)
  pdl_wait();
  pdl_launch_dependents();
  const int seq = blockIdx.z, h = blockIdx.y, kvh = h / (a.nq / a.nkv);
  const Rows rows(a, seq);
  if ((int)blockIdx.x >= rows.count) return;
  const int t = rows.first + blockIdx.x, keys = rows.before + blockIdx.x + 1;
  const Q4Page L(D, G, a.ps);
  const int* bt = a.block_table + (long)seq * a.max_pages;
  const T* row = q + (long)t * a.q_stride + (long)h * D;
  float m = MINUS_BIG, sum = 0.f;
  for (int key = threadIdx.x; key < keys; key += blockDim.x) {
    const int page = bt[key / a.ps];
    if (page < 0 || page >= a.num_pages) continue;
    const float x = score_of(row, a.pages + ((long)page * a.nkv + kvh) * L.record, L, key % a.ps, D, G) * a.scale_log2;
    const float top = fmaxf(m, x);
    sum = sum * exp2f(m - top) + exp2f(x - top);
    m = top;
  }
  __shared__ float red[34];
  const float top = block_max(m, red);
  const float den = block_sum(sum * exp2f(m - top), red);
  if (threadIdx.x == 0) a.lse[(long)t * a.nq + h] = (top + log2f(den)) * LN_2;
}

template <typename T> __global__ void mass_columns_general_kernel(Mass a, const T* q, int D, int G) {  // grid (keys / threads, kv head, sequence)
  pdl_wait();
  pdl_launch_dependents();
  const int seq = blockIdx.z, kvh = blockIdx.y, R = a.nq / a.nkv;
  const Rows rows(a, seq);
  const int key = blockIdx.x * blockDim.x + threadIdx.x;
  if (key >= rows.before + rows.count) return;
  const int page = a.block_table[(long)seq * a.max_pages + key / a.ps];
  if (page < 0 || page >= a.num_pages) return;
  const Q4Page L(D, G, a.ps);
  const unsigned char* rec = a.pages + ((long)page * a.nkv + kvh) * L.record;
  float total = 0.f;
  for (int i = max(0, key - rows.before); i < rows.count; ++i)
    for (int h = kvh * R; h < (kvh + 1) * R; ++h) {
      const long t = rows.first + i;
      const float x = score_of(q + t * a.q_stride + (long)h * D, rec, L, key % a.ps, D, G) * a.scale_log2;
      total += exp2f(x - a.lse[t * a.nq + h] * LOG2_E);
    }
  if (rows.count) a.mass[((long)page * a.nkv + kvh) * a.ps + key % a.ps] += at_most(total, rows.count * R);
}

template <int D, int NT> int launch_mass(const Mass& a, bool want_rows, int most_tokens, int few_slices, cudaStream_t stream) {
  const int rows = most_tokens * (a.nq / a.nkv);
  cudaError_t err = cudaSuccess;
  if (want_rows)
    err = launch_pdl(mass_rows_kernel<D, NT>, dim3(a.slices, (rows + 8 * NT - 1) / (8 * NT), a.num_seqs * a.nkv), dim3(THREADS), 0, stream, a);
  if (err != cudaSuccess) return Q3_ERR_LAUNCH;
  if (rows <= 16) {
    const dim3 grid(few_slices, a.nkv, a.num_seqs);
    if (a.ps % STEP == 0)
      err = rows <= 8 ? launch_pdl(mass_few_kernel<D, 1, true>, grid, dim3(THREADS), 0, stream, a)
                      : launch_pdl(mass_few_kernel<D, 2, true>, grid, dim3(THREADS), 0, stream, a);
    else
      err = rows <= 8 ? launch_pdl(mass_few_kernel<D, 1, false>, grid, dim3(THREADS), 0, stream, a)
                      : launch_pdl(mass_few_kernel<D, 2, false>, grid, dim3(THREADS), 0, stream, a);
  } else {
    constexpr int KEYS = COLUMN_WARPS * STEP;
    constexpr int smem = COLUMN_TILES * sizeof(RowTile<D>);
    static bool once[Q3_MAX_DEVICES];
    const int dev = q3_current_device();
    if (!once[dev]) {
      if (cudaFuncSetAttribute(mass_columns_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return Q3_ERR_LAUNCH;
      once[dev] = true;
    }
    err = launch_pdl(mass_columns_kernel<D>, dim3((a.max_len + KEYS - 1) / KEYS, a.nkv, a.num_seqs), dim3(32 * COLUMN_WARPS), smem, stream, a);
  }
  return err == cudaSuccess ? Q3_OK : Q3_ERR_LAUNCH;
}

// ---- attention in general -----------------------------------------------------------------------------------------------------------------
// float32, and bfloat16 tokens whose head size or group the tiles above do not take: a block of 256 threads takes a (token, kv head, up to 8
// of its query heads); 64 keys at a time come to shared memory as they are stored, the next ones while these are worked on; four threads
// make a key's scores, a warp a head's weights, a thread two channels' results.  Sums are float32 on the FMA pipes, in an order that
// depends on the keys' places alone: tiles begin at multiples of 64, slices of 256 keys have a softmax of their own and are joined in
// order, by the same block or, where the launch leaves SMs idle, by a second kernel from what one block a slice has left -- the same bits,
// however a sequence is cut into steps and batched with others.  What bounds it is instructions.  Slices of 512, 256, 128 keys, in us
// (16 heads over 4 of 64, float32): 21 tokens behind up to 320 keys 20, 20, 16; 8 behind 4,096 35, 38, 44; one behind 32,768 40, 48, 63;
// a prompt of 512 134, 139, 148.  (A tile brought without looking ahead, a division a word, a thread a channel: 35, 62, 75 and 227 at 512.)
constexpr int GEN_THREADS = 256;
constexpr int GEN_TILE = 64;
constexpr int GEN_SLICE = 256;
constexpr int GEN_HEADS = 8;
// bytes of a token's codes and parameters in shared memory
__host__ __device__ __forceinline__ int general_pitch(const Q4Page& L) { return (int)(L.half + L.par + 7) & ~7; }

struct General {
  const unsigned char* pages;
  int num_pages;
  const int *block_table, *token_seq, *places;
  int max_pages, num_seqs, nq, nkv, D, G, ps, window, slices;
  long q_stride;
  float scale_log2;
  float *mid_o, *mid_ml;  // slices > 0: [tokens][nq][slices][D] and [tokens][nq][slices][2]
  int tiles_at;           // byte of shared memory
  // the last key that token t sees; -1: none (it belongs to no sequence, or its place lies outside the table), and its row is zero
  __device__ __forceinline__ int last_key(long t) const {
    const int seq = token_seq[t], place = places[t];
    return seq >= 0 && seq < num_seqs && place >= 0 && place / ps < max_pages ? place : -1;
  }
};

// (m, l, o) <- its join with another's; o and b are unnormalised.  The fused steps are named, so that both kernels round alike.
__device__ __forceinline__ void join_slices(float& m, float& l, float& o, float bm, float bl, float bo) {
  const float top = fmaxf(m, bm), fa = exp2f(m - top), fb = exp2f(bm - top);
  m = top;
  l = __fmaf_rn(l, fa, __fmul_rn(bl, fb));
  o = __fmaf_rn(o, fa, __fmul_rn(bo, fb));
}

template <typename T>
__global__ void __launch_bounds__(GEN_THREADS) general_4bit_kernel(General a, const T* __restrict__ q, T* __restrict__ out) {
  extern __shared__ __align__(128) unsigned char smem[];
  pdl_wait();
  pdl_launch_dependents();
  const int R = a.nq / a.nkv, chunks = (R + GEN_HEADS - 1) / GEN_HEADS;
  const int t = blockIdx.x, kvh = blockIdx.y / chunks, h0 = kvh * R + (blockIdx.y % chunks) * GEN_HEADS;
  const int heads = min(GEN_HEADS, kvh * R + R - h0);
  const int D = a.D, G = a.G, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const Q4Page L(D, G, a.ps);
  float* q_s = reinterpret_cast<float*>(smem);                   // [8][D]
  float* x_s = q_s + GEN_HEADS * D;                              // [8][64] scores
  float* p_s = x_s + GEN_HEADS * GEN_TILE;                       // [64][8] weights
  float* f_s = p_s + GEN_HEADS * GEN_TILE;                       // [8]: what the results so far shrink by; then the slice's maximum and sum
  float* v_s = f_s + 32;                                         // [groups of threads][8][D] at the end of a slice
  unsigned char* k_s = smem + a.tiles_at;                        // two tiles: 64 rows of keys' codes and parameters, then of values
  const int pitch = general_pitch(L), bytes = 2 * GEN_TILE * pitch;
  const int last = a.last_key(t), lo = a.window > 0 ? max(0, last - a.window + 1) : 0;
  const int* bt = a.block_table + (long)(last >= 0 ? a.token_seq[t] : 0) * a.max_pages;
  for (int i = tid; i < heads * D; i += GEN_THREADS) q_s[i] = to_f32(q[t * a.q_stride + (long)h0 * D + i]) * a.scale_log2;
  // a thread owns channels c and c + 1, which share a byte, of the keys g, g + parts, g + 2 parts ... of each tile
  const int parts = 2 * GEN_THREADS / D, c = 2 * (tid % (D / 2)), part = tid / (D / 2);
  const bool owner = part < parts;
  const int c_group = c / (D / G), c_in = c % (D / G), c_byte = 4 * ((c_in / 8) * G + c_group) + (c_in % 8) / 2;
  // two threads bring a row (64 of keys, then 64 of values), 8 bytes of codes or a group's parameters in turn, a tile ahead of its use, into
  // two buffers in turn; what is not there is zero
  const int my_row = tid & (2 * GEN_TILE - 1), my_half = tid >> 7, my_v = my_row >= GEN_TILE;
  auto fetch = [&](int base, int stop) {
    const int key = base + (my_row & (GEN_TILE - 1));
    const unsigned char *codes = a.pages, *pars = a.pages;
    int there = 0;
    if (key >= lo && key < stop) {
      const int pi = key / a.ps, page = bt[pi];
      if ((uint32_t)page < (uint32_t)a.num_pages) {
        const long pr = key - pi * a.ps;
        const unsigned char* rec = a.pages + ((long)page * a.nkv + kvh) * L.record;
        codes = rec + (my_v ? L.values : 0) + pr * L.half;
        pars = rec + (my_v ? L.vpar : L.kpar) + pr * L.par;
        there = 1;
      }
    }
    const uint32_t dst = smem_addr(k_s) + (base / GEN_TILE & 1) * bytes + my_row * pitch;
    for (int at = 8 * my_half; at < L.half; at += 16) cp_async8(dst + at, codes + at * there, 8 * there);
    for (int at = 4 * my_half; at < L.par; at += 8) cp_async4(dst + L.half + at, pars + at * there, 4 * there);
    cp_async_commit();
  };
  float M[GEN_HEADS], S[GEN_HEADS], O[GEN_HEADS][2];
#pragma unroll
  for (int h = 0; h < GEN_HEADS; ++h) M[h] = MINUS_BIG, S[h] = 0.f, O[h][0] = O[h][1] = 0.f;
  const int slice0 = a.slices > 0 ? blockIdx.z : lo / GEN_SLICE, slice1 = a.slices > 0 ? blockIdx.z : last / GEN_SLICE;
  const int stop = min(last + 1, (slice1 + 1) * GEN_SLICE);
  fetch(max(lo, slice0 * GEN_SLICE) / GEN_TILE * GEN_TILE, stop);
  for (int slice = slice0; slice <= slice1 && last >= 0; ++slice) {
    const int begin = max(lo, slice * GEN_SLICE) / GEN_TILE * GEN_TILE, end = min(last + 1, (slice + 1) * GEN_SLICE);
    float o[GEN_HEADS][2];
#pragma unroll
    for (int h = 0; h < GEN_HEADS; ++h) o[h][0] = o[h][1] = 0.f;
    float m = MINUS_BIG, l = 0.f;  // warp h: of head h, the same in every lane
    for (int base = begin; base < end; base += GEN_TILE) {
      __syncthreads();
      fetch(base + GEN_TILE, stop);
      cp_async_wait<1>();
      __syncthreads();
      const unsigned char* tile = k_s + (base / GEN_TILE & 1) * bytes;
      {  // four threads a key, each every fourth word; 8 channels of a word in order, the four threads' sums in pairs
        const int key = tid >> 2, sub = tid & 3;
        const uint32_t* row = reinterpret_cast<const uint32_t*>(tile + key * pitch);
        const uint32_t* par = reinterpret_cast<const uint32_t*>(tile + key * pitch + L.half);
        float x[GEN_HEADS];
#pragma unroll
        for (int h = 0; h < GEN_HEADS; ++h) x[h] = 0.f;
        for (int w = sub; w < D / 8; w += 4) {
          const uint32_t code = row[w];
          const int g = w % G, first = g * (D / G) + 8 * (w / G);
          const float s = q4_s(par[g]), z = q4_z(par[g]);
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = z + (float)((code >> (4 * e)) & 15u) * s;
#pragma unroll
          for (int h = 0; h < GEN_HEADS; ++h)
            if (h < heads) {
              const float4 qa = *reinterpret_cast<const float4*>(q_s + h * D + first), qb = *reinterpret_cast<const float4*>(q_s + h * D + first + 4);
              x[h] = fmaf(qa.x, v[0], x[h]), x[h] = fmaf(qa.y, v[1], x[h]), x[h] = fmaf(qa.z, v[2], x[h]), x[h] = fmaf(qa.w, v[3], x[h]);
              x[h] = fmaf(qb.x, v[4], x[h]), x[h] = fmaf(qb.y, v[5], x[h]), x[h] = fmaf(qb.z, v[6], x[h]), x[h] = fmaf(qb.w, v[7], x[h]);
            }
        }
        const bool seen = base + key >= lo && base + key < end;
#pragma unroll
        for (int h = 0; h < GEN_HEADS; ++h) {
          x[h] += __shfl_xor_sync(0xffffffffu, x[h], 1);
          x[h] += __shfl_xor_sync(0xffffffffu, x[h], 2);
          if (sub == (h & 3) && h < heads) x_s[h * GEN_TILE + key] = seen ? x[h] : -INFINITY;
        }
      }
      __syncthreads();
      if (warp < heads) {
        const float x0 = x_s[warp * GEN_TILE + lane], x1 = x_s[warp * GEN_TILE + 32 + lane];
        const float top = fmaxf(m, warp_max(fmaxf(x0, x1))), f = exp2f(m - top);
        const float p0 = exp2f(x0 - top), p1 = exp2f(x1 - top);
        p_s[GEN_HEADS * lane + warp] = p0, p_s[GEN_HEADS * (lane + 32) + warp] = p1;
        l = l * f + warp_sum(p0 + p1);
        m = top;
        if (lane == 0) f_s[warp] = f;
      }
      __syncthreads();
      if (owner) {
#pragma unroll
        for (int h = 0; h < GEN_HEADS; ++h)
          if (h < heads) o[h][0] *= f_s[h], o[h][1] *= f_s[h];
        const unsigned char* rows = tile + GEN_TILE * pitch;
        for (int key = part; key < GEN_TILE; key += parts) {
          const unsigned char* row = rows + key * pitch;
          const uint32_t par = *reinterpret_cast<const uint32_t*>(row + L.half + 4 * c_group), code = row[c_byte];
          const float v0 = q4_z(par) + (float)(code & 15) * q4_s(par), v1 = q4_z(par) + (float)(code >> 4) * q4_s(par);
          float w[GEN_HEADS];
          *reinterpret_cast<float4*>(w) = *reinterpret_cast<const float4*>(p_s + GEN_HEADS * key);
          if (heads > 4) *reinterpret_cast<float4*>(w + 4) = *reinterpret_cast<const float4*>(p_s + GEN_HEADS * key + 4);
#pragma unroll
          for (int h = 0; h < GEN_HEADS; ++h)
            if (h < heads) o[h][0] = fmaf(w[h], v0, o[h][0]), o[h][1] = fmaf(w[h], v1, o[h][1]);
        }
      }
    }
    // the threads' shares of a channel, in order; then the slice joins what came before it
    __syncthreads();
    if (owner) {
#pragma unroll
      for (int h = 0; h < GEN_HEADS; ++h)
        if (h < heads) *reinterpret_cast<float2*>(v_s + (part * GEN_HEADS + h) * D + c) = make_float2(o[h][0], o[h][1]);
    }
    if (warp < heads && lane == 0) f_s[8 + 2 * warp] = m, f_s[9 + 2 * warp] = l;
    __syncthreads();
    if (owner && part == 0) {
#pragma unroll
      for (int h = 0; h < GEN_HEADS; ++h)
        if (h < heads) {
          float2 y = *reinterpret_cast<const float2*>(v_s + h * D + c);
          for (int g = 1; g < parts; ++g) {
            const float2 z = *reinterpret_cast<const float2*>(v_s + (g * GEN_HEADS + h) * D + c);
            y.x += z.x, y.y += z.y;
          }
          float m = M[h], l = S[h];
          join_slices(m, l, O[h][0], f_s[8 + 2 * h], f_s[9 + 2 * h], y.x);
          join_slices(M[h], S[h], O[h][1], f_s[8 + 2 * h], f_s[9 + 2 * h], y.y);
        }
    }
  }
  cp_async_wait<0>();  // (the tile behind the last one: zeros)
  if (owner && part == 0) {
#pragma unroll
    for (int h = 0; h < GEN_HEADS; ++h)
      if (h < heads) {
        if (a.slices > 0) {
          const long at = ((long)t * a.nq + h0 + h) * a.slices + blockIdx.z;
          a.mid_o[at * D + c] = O[h][0], a.mid_o[at * D + c + 1] = O[h][1];
          if (c == 0) a.mid_ml[2 * at] = M[h], a.mid_ml[2 * at + 1] = S[h];
        } else {
          T* y = out + ((long)t * a.nq + h0 + h) * D + c;
          y[0] = from_f32<T>(last >= 0 ? O[h][0] / S[h] : 0.f), y[1] = from_f32<T>(last >= 0 ? O[h][1] / S[h] : 0.f);
        }
      }
  }
}

// One block per (token, head): joins the slices in order, a thread per channel.
template <typename T> __global__ void general_4bit_merge_kernel(General a, T* __restrict__ out) {
  pdl_wait();
  pdl_launch_dependents();
  const long at = blockIdx.x;
  const int last = a.last_key(at / a.nq), lo = a.window > 0 ? max(0, last - a.window + 1) : 0;
  for (int c = threadIdx.x; c < a.D; c += blockDim.x) {
    float M = MINUS_BIG, S = 0.f, O = 0.f;
    const int stop = last >= 0 ? min(last / GEN_SLICE + 1, a.slices) : 0;
    for (int s0 = lo / GEN_SLICE; s0 < stop; s0 += 8) {  // eight slices' loads at a time
      float m[8], l[8], o[8];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (s0 + u < stop) {
          const long i = at * a.slices + s0 + u;
          m[u] = a.mid_ml[2 * i], l[u] = a.mid_ml[2 * i + 1], o[u] = a.mid_o[i * a.D + c];
        }
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (s0 + u < stop) join_slices(M, S, O, m[u], l[u], o[u]);
    }
    out[at * a.D + c] = from_f32<T>(last >= 0 ? O / S : 0.f);
  }
}

template <typename T> int launch_general(General a, const T* q, T* out, int tokens, cudaStream_t stream) {
  const Q4Page L(a.D, a.G, a.ps);
  const int R = a.nq / a.nkv, chunks = (R + GEN_HEADS - 1) / GEN_HEADS, parts = 2 * GEN_THREADS / a.D;
  const int tiles_at = ((GEN_HEADS * (a.D + 2 * GEN_TILE) + 32 + parts * GEN_HEADS * a.D) * 4 + 15) & ~15;
  a.tiles_at = tiles_at;
  const int smem = tiles_at + 2 * 2 * GEN_TILE * general_pitch(L);
  static bool once[Q3_MAX_DEVICES];
  const int dev = q3_current_device();
  if (!once[dev]) {
    if (cudaFuncSetAttribute(general_4bit_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, 96 * 1024) != cudaSuccess) return Q3_ERR_LAUNCH;
    once[dev] = true;
  }
  cudaError_t err = launch_pdl(general_4bit_kernel<T>, dim3(tokens, a.nkv * chunks, a.slices > 0 ? a.slices : 1), dim3(GEN_THREADS), smem, stream,
                               a, q, out);
  if (err == cudaSuccess && a.slices > 0)
    err = launch_pdl(general_4bit_merge_kernel<T>, dim3((unsigned)((long)tokens * a.nq)), dim3(a.D <= 128 ? 128 : 256), 0, stream, a, out);
  return err == cudaSuccess ? Q3_OK : Q3_ERR_LAUNCH;
}

}  // namespace

// `lse` holds the observed rows' log sums (have_lse) or is scratch for them; `part` [tokens][nq][slices] pairs of floats when slices > 1.
Q3_EXPORT int q3_attention_mass_4bit(int dtype, const void* q, int q_stride, const void* pages, int num_pages, const int* block_table,
                                     int max_pages, const int* kv_lens, const int* cu_seqlens, float* mass, float* lse, int have_lse,
                                     void* part, int slices, int num_seqs, int nq, int nkv, int D, int ps, float scale, int max_len,
                                     int observe, int most_tokens, int few_slices, cudaStream_t stream) {
  if (num_seqs < 1 || most_tokens < 1 || max_len < 1) return Q3_OK;
  if (!q || !pages || !block_table || !kv_lens || !cu_seqlens || !mass || !lse || nq < 1 || nkv < 1 || nq % nkv || !q4_sizes_ok(D, ps) ||
      slices < 1 || few_slices < 1 || (slices > 1 && !part) || observe < 1 || max_len > (long)max_pages * ps)
    return Q3_ERR_ARGUMENT;
  if (dtype != Q3_DTYPE_F32 && dtype != Q3_DTYPE_BF16) return Q3_ERR_ARGUMENT;
  if (q_stride % 8 || (reinterpret_cast<uintptr_t>(q) & 15) || (reinterpret_cast<uintptr_t>(pages) & 15) ||
      (long)num_seqs * nkv > 65535 || nq > 65535)
    return Q3_ERR_UNSUPPORTED;
  Mass a{(const bf16*)q, q_stride, (const unsigned char*)pages, num_pages, block_table, kv_lens, cu_seqlens, max_pages, nq, nkv, ps,
         max_len, observe, slices, num_seqs, scale * LOG2_E, lse, have_lse || slices == 1 ? nullptr : (float2*)part, mass};
  if (dtype == Q3_DTYPE_BF16 && (D == 64 || D == 128 || D == 256)) {
    if ((long)most_tokens * (nq / nkv) > 65535L * 16) return Q3_ERR_UNSUPPORTED;
    if (D == 64) return launch_mass<64, 4>(a, !have_lse, most_tokens, few_slices, stream);
    if (D == 128) return launch_mass<128, 4>(a, !have_lse, most_tokens, few_slices, stream);
    return launch_mass<256, 2>(a, !have_lse, most_tokens, few_slices, stream);
  }
  const int G = q4_groups(D);
  cudaError_t err = cudaSuccess;
  const dim3 columns((max_len + 127) / 128, nkv, num_seqs);
  if (dtype == Q3_DTYPE_BF16) {
    if (!have_lse)
      err = launch_pdl(mass_rows_general_kernel<bf16>, dim3(most_tokens, nq, num_seqs), dim3(128), 0, stream, a, (const bf16*)q, D, G);
    if (err == cudaSuccess) err = launch_pdl(mass_columns_general_kernel<bf16>, columns, dim3(128), 0, stream, a, (const bf16*)q, D, G);
  } else {
    if (!have_lse)
      err = launch_pdl(mass_rows_general_kernel<float>, dim3(most_tokens, nq, num_seqs), dim3(128), 0, stream, a, (const float*)q, D, G);
    if (err == cudaSuccess) err = launch_pdl(mass_columns_general_kernel<float>, columns, dim3(128), 0, stream, a, (const float*)q, D, G);
  }
  return err == cudaSuccess ? Q3_OK : Q3_ERR_LAUNCH;
}

Q3_EXPORT int q3_decode_attention_4bit(const void* q, int q_stride, const void* pages, int num_pages, const int* block_table, int max_pages,
                                       const int* kv_lens, const int* cu_seqlens, const int* seq_list, void* out, float* mid_o,
                                       float* mid_lse, float* lse, int num_seqs, int nq, int nkv, int D, int ps, float scale, int window,
                                       int splits, int max_len, const int* longest, int* error_word, cudaStream_t stream) {
  if (num_seqs < 1) return Q3_OK;
  if (!q || !pages || !block_table || !kv_lens || !cu_seqlens || !out || nq < 1 || nkv < 1 || nq % nkv || !q4_sizes_ok(D, ps) || splits < 1 ||
      !error_word || (splits > MOST_CLUSTER && !mid_o) || (mid_o && !mid_lse) || max_len > (long)max_pages * ps)
    return Q3_ERR_ARGUMENT;
  const int R = nq / nkv;
  if (R > 16 || q_stride % 8 || (reinterpret_cast<uintptr_t>(q) & 15) || (reinterpret_cast<uintptr_t>(pages) & 15) ||
      (reinterpret_cast<uintptr_t>(out) & 7) || num_seqs > 65535 || nkv > 65535 || Q4Page(D, q4_groups(D), ps).record * nkv > 0x7fffffffL)
    return Q3_ERR_UNSUPPORTED;
  Decode a{(const bf16*)q, q_stride, (const unsigned char*)pages, num_pages, block_table, kv_lens, cu_seqlens, seq_list, max_pages,
           (bf16*)out, mid_o, mid_lse, lse, nq, nkv, ps, window, splits, max_len, scale * LOG2_E, longest, error_word};
  if (D == 64) return R <= 8 ? launch_decode<64, 1>(a, num_seqs, stream) : launch_decode<64, 2>(a, num_seqs, stream);
  if (D == 128) return R <= 8 ? launch_decode<128, 1>(a, num_seqs, stream) : launch_decode<128, 2>(a, num_seqs, stream);
  if (D == 256) return R <= 8 ? launch_decode<256, 1>(a, num_seqs, stream) : launch_decode<256, 2>(a, num_seqs, stream);
  return Q3_ERR_UNSUPPORTED;
}

// `slices` 0: a block goes through all of a token's keys; else mid_o [tokens][nq][slices][D] and mid_ml [tokens][nq][slices][2] are given and
// slices * 256 covers the longest sequence.
Q3_EXPORT int q3_general_attention_4bit(int dtype, const void* q, long q_stride, const void* pages, int num_pages, const int* block_table,
                                        int max_pages, int num_seqs, const int* token_seq, const int* places, void* out, float* mid_o,
                                        float* mid_ml, int slices, int tokens, int nq, int nkv, int D, int ps, float scale, int window,
                                        cudaStream_t stream) {
  if (tokens < 1) return Q3_OK;
  if (!q || !pages || !block_table || !token_seq || !places || !out || nq < 1 || nkv < 1 || nq % nkv || !q4_sizes_ok(D, ps) || max_pages < 1 ||
      slices < 0 || (slices > 0 && (!mid_o || !mid_ml)))
    return Q3_ERR_ARGUMENT;
  if (dtype != Q3_DTYPE_F32 && dtype != Q3_DTYPE_BF16) return Q3_ERR_ARGUMENT;
  if ((long)nkv * ((nq / nkv + GEN_HEADS - 1) / GEN_HEADS) > 65535 || slices > 65535 || (long)tokens * nq > 0x7fffffffL ||
      (reinterpret_cast<uintptr_t>(pages) & 15))
    return Q3_ERR_UNSUPPORTED;
  General a{(const unsigned char*)pages, num_pages, block_table, token_seq, places, max_pages, num_seqs, nq, nkv, D, q4_groups(D), ps, window,
            slices, q_stride, scale * LOG2_E, mid_o, mid_ml};
  return dtype == Q3_DTYPE_F32 ? launch_general(a, (const float*)q, (float*)out, tokens, stream)
                               : launch_general(a, (const bf16*)q, (bf16*)out, tokens, stream);
}
