// Attention over a cache in 4 bits (layout: four_bit.cuh): decode attention in bfloat16, and the sums of attention weights per cached
// token that eviction goes by.
//
// Numbers never leave 4 bits before the registers: a 32-bit word of 8 of them becomes four pairs of bfloat16 by a shift and a
// (x & 0x000F000F) | 0x43004300 each, which is 128 + n exactly, and the scale, the minimum and the 128 are applied to sums:
//   scores   K (16 keys) x Q^T (8 queries) on mma.sync m16n8k16, one accumulator per group g of channels that starts at
//            -128 * sum_c q_c:     score = sum_g  s_g * acc_g + z_g * sum_(c in g) q_c
//   results  V^T (16 channels) x P^T: P^T is the transposed score tile (movmatrix), times the tokens' scales per group, rounded to
//            w_t = bf16(p_t s_t); what is the same for all channels of a group joins as three more products with constant rows:
//              o_c = sum_t w_t (128 + n_tc)  -  136 sum_t w_t  +  sum_t p_t (z_t + 8 s_t)
//            so that the rounding of w weighs on n - 8, which is as small as the values about their middle, and not on n (taken off
//            as 128 with sum_t p_t z_t alone, results were 0.003 to 0.005 off, relative; so 0.0023, of which 0.0017 is the result's own
//            rounding).
// Keys as the product's 16 rows and the kv head's queries as its 8 columns: a group of up to 8 query heads wastes nothing (the other way
// round, 16 rows of queries, computes twice as much, and the conversion would meet half as many values per instruction).
#include "four_bit.cuh"
#include "mma_tiles.cuh"

namespace {

constexpr float MINUS_BIG = -1e30f;  // of a row that has seen nothing: a hidden key's score is -inf and weighs 2^(-inf - MINUS_BIG) = 0
constexpr float LN_2 = 0.6931471805599453f;

template <int J> __device__ __forceinline__ uint32_t pair_of(uint32_t w) {  // numbers J and J + 4 of a word, plus 128, as two bfloat16
  return ((w >> (4 * J)) & 0x000F000Fu) | 0x43004300u;
}
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  const __nv_bfloat162 y = __hmul2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&y);
}
__device__ __forceinline__ uint32_t transposed(uint32_t a) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(a));
  return y;
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
  static constexpr int STAGE = 16 * (D + 2 * PAR);  // bytes of 16 tokens' keys and values
  // word j of lane l: which group, and which 8 channels of it
  static __device__ __forceinline__ int group(int j) { return D == 64 ? 0 : j % G; }
  static __device__ __forceinline__ int index(int j, int l) {
    return D == 64 ? 2 * l + j : D == 128 ? 2 * l + j / 2 : l + 4 * (j / 4);
  }
};

// The queries' side of the scores: B fragments (n = lane / 4: the query, k: the channels that word j's pairs stand for).
// b[j][0..3]: of word j, channels (0, 4), (1, 5), (2, 6), (3, 7) of its eight.
template <int D> __device__ __forceinline__ void load_query(uint32_t (&b)[Head<D>::WORDS][4], const bf16* row, int lane) {
#pragma unroll
  for (int j = 0; j < Head<D>::WORDS; ++j) {
    uint4 v = make_uint4(0, 0, 0, 0);
    if (row) v = *reinterpret_cast<const uint4*>(row + 64 * Head<D>::group(j) + 8 * Head<D>::index(j, lane & 3));
    // v: channels (0,1) (2,3) (4,5) (6,7)
    b[j][0] = __byte_perm(v.x, v.z, 0x5410);
    b[j][1] = __byte_perm(v.x, v.z, 0x7632);
    b[j][2] = __byte_perm(v.y, v.w, 0x5410);
    b[j][3] = __byte_perm(v.y, v.w, 0x7632);
  }
}

// Sums of the queries' channels per group, in the accumulators' layout (columns 2 (lane % 4), + 1): a product with ones.
template <int D> __device__ __forceinline__ void query_sums(float (&sum)[Head<D>::G][2], const uint32_t (&b)[Head<D>::WORDS][4]) {
  const uint32_t one[4] = {0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u};
  float c[Head<D>::G][4];
#pragma unroll
  for (int g = 0; g < Head<D>::G; ++g) c[g][0] = c[g][1] = c[g][2] = c[g][3] = 0.f;
#pragma unroll
  for (int j = 0; j < Head<D>::WORDS; ++j) {
    mma_bf16(c[Head<D>::group(j)], one, b[j][0], b[j][1]);
    mma_bf16(c[Head<D>::group(j)], one, b[j][2], b[j][3]);
  }
#pragma unroll
  for (int g = 0; g < Head<D>::G; ++g) sum[g][0] = c[g][0], sum[g][1] = c[g][1];
}

// ---- decode attention -------------------------------------------------------------------------------------------------------------
// Grid (slice, kv head, sequence): a block takes one slice of one sequence's keys for one kv head and the query heads that read it; each of
// its 4 warps takes every fourth 16 keys, with a ring of its own that cp.async fills (no barrier in the loop) and a softmax of its own;
// the warps are joined at the end, the slices by whoever reads the partial results (merge kernel).
constexpr int WARPS = 4;
constexpr int THREADS = 32 * WARPS;
constexpr int STEP = 16;  // keys a warp takes at a time
constexpr int STAGES = 4;

// Rows of values are read by tokens 2l, 2l + 1 (lane % 4 = l) in pieces of lane / 4: places that let the lanes of one request hit different banks.
template <int D> __device__ __forceinline__ int value_place(int t, int chunk) {
  if (D == 64) return ((t & 8) + (t & 1) * 4 + ((t >> 1) & 3)) * 32 + chunk * 16;
  if (D == 128) return (t >> 1) * 128 + (((t & 1) ^ ((t >> 1) & 1)) * 64) + (chunk ^ (((t >> 2) & 1) << 1)) * 16;
  return t * 128 + (chunk ^ (((t >> 1) & 3) << 1)) * 16;
}
template <int D> __device__ __forceinline__ int key_place(int t, int chunk) {
  return t * Head<D>::ROW + (D == 256 ? chunk ^ ((t & 1) << 2) : chunk) * 16;
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
};

// Keys per slice, the same for all sequences of the launch: the longest sequence's keys over the slices asked for, in whole rounds of the
// block.  A shorter sequence has fewer slices.
__device__ __forceinline__ int slice_keys(const Decode& a) {
  int longest = a.longest ? min(*a.longest, a.max_len) : a.max_len;
  if (a.window > 0) longest = min(longest, a.window);
  const int per = (longest + a.splits - 1) / a.splits;
  return max(64, (per + 63) & ~63);
}

template <int D, int NT>
__global__ void __launch_bounds__(THREADS) decode_4bit_kernel(Decode a) {
  using H = Head<D>;
  extern __shared__ __align__(128) unsigned char smem[];
  const int split = blockIdx.x, kvh = blockIdx.y, slot = blockIdx.z;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r = lane >> 2, l = lane & 3;
  const int R = a.nq / a.nkv;
  pdl_wait();
  const int seq = a.seq_list ? a.seq_list[slot] : slot;
  const int kv_len = min(a.kv_lens[seq], a.max_len), tok = a.cu_seqlens[seq];
  const int lo = a.window > 0 ? max(0, kv_len - a.window) : 0;
  const int per = slice_keys(a);
  const int begin = lo + split * per, end = min(kv_len, begin + per);
  const long out_row = (long)tok * a.nq + kvh * R;
  if (begin >= end) {
    pdl_launch_dependents();
    if (split == 0) {  // no key at all
      if (a.splits > 1) {
        if (tid < R) a.mid_lse[((long)slot * a.nq + kvh * R + tid) * a.splits] = -INFINITY;
      } else {
        for (int i = tid; i < R * D; i += THREADS) a.out[out_row * D + i] = __float2bfloat16_rn(0.f);
        if (a.lse && tid < R) a.lse[out_row + tid] = -INFINITY;
      }
    }
    return;
  }
  const Q4Page L(D, H::G, a.ps);
  const int* bt = a.block_table + (long)seq * a.max_pages;
  unsigned char* ring = smem + warp * STAGES * H::STAGE;
  const int steps = (end - begin + STEP * WARPS - 1) / (STEP * WARPS);

  // A lane copies half of the pieces of token lane / 2 of the 16.  The page is looked up a step ahead: the copies' addresses wait for it.
  auto look_up = [&](int i) {
    const int key = begin + (i * WARPS + warp) * STEP + (lane >> 1);
    return key < end ? bt[key / a.ps] : -1;
  };
  auto load_step = [&](int i, int page) {
    unsigned char* st = ring + (i % STAGES) * H::STAGE;
    const int t = lane >> 1, key = begin + (i * WARPS + warp) * STEP + t;
    const bool valid = page >= 0 && page < a.num_pages;  // (a page that was given back reads as zeros, like what lies behind the slice)
    const unsigned char* rec = a.pages + ((long)(valid ? page : 0) * a.nkv + kvh) * L.record;
    const int row = valid ? key % a.ps : 0;
    constexpr int CH = H::ROW / 16;  // pieces of a row: 2, 4 or 8
#pragma unroll
    for (int c = 0; c < CH / 2; ++c) {
      const int chunk = (lane & 1) * (CH / 2) + c;
      cp_async16(smem_u32(st + key_place<D>(t, chunk)), rec + (long)row * H::ROW + 16 * chunk, valid ? 16 : 0);
      cp_async16(smem_u32(st + STEP * H::ROW + value_place<D>(t, chunk)), rec + L.values + (long)row * H::ROW + 16 * chunk, valid ? 16 : 0);
    }
    const uint32_t par = smem_u32(st + 2 * STEP * H::ROW + (lane & 1) * STEP * H::PAR + t * H::PAR);
    const unsigned char* src = rec + (lane & 1 ? L.vpar : L.kpar) + (long)row * H::PAR;
    if (D == 64) cp_async4(par, src, valid ? 4 : 0);
    if (D == 128) cp_async8(par, src, valid ? 8 : 0);
    if (D == 256) cp_async16(par, src, valid ? 16 : 0);
  };
  int next[STAGES - 1];
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) next[i] = look_up(i);
  int ahead = look_up(STAGES - 1);
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) {
    load_step(i, next[i]);
    cp_async_commit();
  }

  uint32_t qf[NT][H::WORDS][4];
  float qsum[NT][H::G][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int h = 8 * n + r;
    load_query<D>(qf[n], h < R ? a.q + (long)tok * a.q_stride + (long)(kvh * R + h) * D : nullptr, lane);
    query_sums<D>(qsum[n], qf[n]);
  }
  float o[NT][H::G][4][4], oz[NT][H::G][4], m[NT][2], sum[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    m[n][0] = m[n][1] = MINUS_BIG;
    sum[n][0] = sum[n][1] = 0.f;
#pragma unroll
    for (int g = 0; g < H::G; ++g)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        oz[n][g][e] = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[n][g][j][e] = 0.f;
      }
  }

  for (int i = 0; i < steps; ++i) {
    cp_async_wait<STAGES - 2>();
    __syncwarp();
    const unsigned char* st = ring + (i % STAGES) * Head<D>::STAGE;
    const int base = begin + (i * WARPS + warp) * STEP;
    if (base < end) {
      const unsigned char* par_k = st + 2 * STEP * H::ROW;
      const unsigned char* par_v = par_k + STEP * H::PAR;
      // ---- scores of 16 keys
      uint32_t kw[2][H::WORDS], kp[2][H::G];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int t = r + 8 * half;
        if constexpr (D == 64) {
          *reinterpret_cast<uint2*>(&kw[half][0]) = *reinterpret_cast<const uint2*>(st + t * H::ROW + 8 * l);
          kp[half][0] = *reinterpret_cast<const uint32_t*>(par_k + t * 4);
        } else if constexpr (D == 128) {
          *reinterpret_cast<uint4*>(&kw[half][0]) = *reinterpret_cast<const uint4*>(st + key_place<D>(t, l));
          *reinterpret_cast<uint2*>(&kp[half][0]) = *reinterpret_cast<const uint2*>(par_k + t * 8);
        } else {
          *reinterpret_cast<uint4*>(&kw[half][0]) = *reinterpret_cast<const uint4*>(st + key_place<D>(t, l));
          *reinterpret_cast<uint4*>(&kw[half][4]) = *reinterpret_cast<const uint4*>(st + key_place<D>(t, l + 4));
          *reinterpret_cast<uint4*>(&kp[half][0]) = *reinterpret_cast<const uint4*>(par_k + t * 16);
        }
      }
      float acc[NT][H::G][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int g = 0; g < H::G; ++g) {
          acc[n][g][0] = acc[n][g][2] = -128.f * qsum[n][g][0];
          acc[n][g][1] = acc[n][g][3] = -128.f * qsum[n][g][1];
        }
#pragma unroll
      for (int j = 0; j < H::WORDS; ++j) {
        const uint32_t a0[4] = {pair_of<0>(kw[0][j]), pair_of<0>(kw[1][j]), pair_of<1>(kw[0][j]), pair_of<1>(kw[1][j])};
        const uint32_t a1[4] = {pair_of<2>(kw[0][j]), pair_of<2>(kw[1][j]), pair_of<3>(kw[0][j]), pair_of<3>(kw[1][j])};
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma_bf16(acc[n][H::group(j)], a0, qf[n][j][0], qf[n][j][1]);
          mma_bf16(acc[n][H::group(j)], a1, qf[n][j][2], qf[n][j][3]);
        }
      }
      const bool in0 = base + r < end, in1 = base + r + 8 < end;
      uint32_t p[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int g = 0; g < H::G; ++g) {
          const float s0 = q4_s(kp[0][g]), z0 = q4_z(kp[0][g]), s1 = q4_s(kp[1][g]), z1 = q4_z(kp[1][g]);
          x[0] += s0 * acc[n][g][0] + z0 * qsum[n][g][0];
          x[1] += s0 * acc[n][g][1] + z0 * qsum[n][g][1];
          x[2] += s1 * acc[n][g][2] + z1 * qsum[n][g][0];
          x[3] += s1 * acc[n][g][3] + z1 * qsum[n][g][1];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = (e < 2 ? in0 : in1) ? x[e] * a.scale_log2 : -INFINITY;
        // the maximum moves only when it would be passed by a factor of 2^8: a weight is 2^8 at most, which float32 sums do not mind
        const bool far = fmaxf(x[0], x[2]) > m[n][0] + 8.f || fmaxf(x[1], x[3]) > m[n][1] + 8.f;
        if (__any_sync(0xffffffffu, far)) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float top = fmaxf(m[n][c], fmaxf(x[c], x[c + 2]));
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            const float f = exp2f(m[n][c] - top);
            m[n][c] = top;
            sum[n][c] *= f;
#pragma unroll
            for (int g = 0; g < H::G; ++g) {
              oz[n][g][c] *= f, oz[n][g][c + 2] *= f;
#pragma unroll
              for (int j = 0; j < 4; ++j) o[n][g][j][c] *= f, o[n][g][j][c + 2] *= f;
            }
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = exp2f(x[e] - m[n][e & 1]);
        sum[n][0] += x[0] + x[2];
        sum[n][1] += x[1] + x[3];
        // weights are rounded to bfloat16 for the product, as everywhere in this engine's 16-bit attention
        p[n][0] = transposed(pack_bf16(x[0], x[1]));
        p[n][1] = transposed(pack_bf16(x[2], x[3]));
      }
      // ---- results: tokens 2l, 2l + 1, 2l + 8, 2l + 9
      uint32_t vw[4][H::G], vp[4][H::G];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int t = 2 * l + (e & 1) + 8 * (e >> 1);
        const unsigned char* vs = st + STEP * H::ROW;
        if constexpr (D == 64) {
          vw[e][0] = *reinterpret_cast<const uint32_t*>(vs + value_place<D>(t, r >> 2) + 4 * (r & 3));
          vp[e][0] = *reinterpret_cast<const uint32_t*>(par_v + t * 4);
        } else if constexpr (D == 128) {
          *reinterpret_cast<uint2*>(&vw[e][0]) = *reinterpret_cast<const uint2*>(vs + value_place<D>(t, r >> 1) + 8 * (r & 1));
          *reinterpret_cast<uint2*>(&vp[e][0]) = *reinterpret_cast<const uint2*>(par_v + t * 8);
        } else {
          *reinterpret_cast<uint4*>(&vw[e][0]) = *reinterpret_cast<const uint4*>(vs + value_place<D>(t, r));
          *reinterpret_cast<uint4*>(&vp[e][0]) = *reinterpret_cast<const uint4*>(par_v + t * 16);
        }
      }
#pragma unroll
      for (int g = 0; g < H::G; ++g) {
        const uint32_t lo0 = __byte_perm(vw[0][g], vw[1][g], 0x5410), hi0 = __byte_perm(vw[0][g], vw[1][g], 0x7632);
        const uint32_t lo1 = __byte_perm(vw[2][g], vw[3][g], 0x5410), hi1 = __byte_perm(vw[2][g], vw[3][g], 0x7632);
        const uint32_t s0 = __byte_perm(vp[0][g], vp[1][g], 0x5410), z0 = __byte_perm(vp[0][g], vp[1][g], 0x7632);
        const uint32_t s1 = __byte_perm(vp[2][g], vp[3][g], 0x5410), z1 = __byte_perm(vp[2][g], vp[3][g], 0x7632);
        const uint32_t az[4] = {z0, z0, z1, z1};
        const __nv_bfloat162 eight = __floats2bfloat162_rn(8.f, 8.f);
        const uint32_t e0 = mul_bf16x2(s0, *reinterpret_cast<const uint32_t*>(&eight)), e1 = mul_bf16x2(s1, *reinterpret_cast<const uint32_t*>(&eight));
        const uint32_t as[4] = {e0, e0, e1, e1};
        const uint32_t off[4] = {0xC308C308u, 0xC308C308u, 0xC308C308u, 0xC308C308u};  // -136
        const uint32_t v0[4] = {pair_of<0>(lo0), pair_of<0>(hi0), pair_of<0>(lo1), pair_of<0>(hi1)};
        const uint32_t v1[4] = {pair_of<1>(lo0), pair_of<1>(hi0), pair_of<1>(lo1), pair_of<1>(hi1)};
        const uint32_t v2[4] = {pair_of<2>(lo0), pair_of<2>(hi0), pair_of<2>(lo1), pair_of<2>(hi1)};
        const uint32_t v3[4] = {pair_of<3>(lo0), pair_of<3>(hi0), pair_of<3>(lo1), pair_of<3>(hi1)};
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const uint32_t w0 = mul_bf16x2(p[n][0], s0), w1 = mul_bf16x2(p[n][1], s1);
          mma_bf16(oz[n][g], az, p[n][0], p[n][1]);
          mma_bf16(oz[n][g], as, p[n][0], p[n][1]);
          mma_bf16(oz[n][g], off, w0, w1);
          mma_bf16(o[n][g][0], v0, w0, w1);
          mma_bf16(o[n][g][1], v1, w0, w1);
          mma_bf16(o[n][g][2], v2, w0, w1);
          mma_bf16(o[n][g][3], v3, w0, w1);
        }
      }
    }
    __syncwarp();
    load_step(i + STAGES - 1, ahead);
    ahead = look_up(i + STAGES);
    cp_async_commit();
  }
  pdl_launch_dependents();

  // ---- the warps' results: [warp][query][D + 4] and [warp][query][2] over the rings
  asm volatile("cp.async.wait_all;\n" ::);
  __syncthreads();
  constexpr int QS = 8 * NT, PITCH = D + 4;
  float* ow = reinterpret_cast<float*>(smem);
  float* ml = ow + WARPS * QS * PITCH;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int h = 8 * n + 2 * l + c;
      float total = sum[n][c];
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
      if (r == 0) {
        ml[(warp * QS + h) * 2] = m[n][c];
        ml[(warp * QS + h) * 2 + 1] = total;
      }
      float* row = ow + (warp * QS + h) * PITCH;
#pragma unroll
      for (int g = 0; g < H::G; ++g) {
        const float add = oz[n][g][c];
        *reinterpret_cast<float4*>(row + 64 * g + 8 * r) =
            make_float4(o[n][g][0][c] + add, o[n][g][1][c] + add, o[n][g][2][c] + add, o[n][g][3][c] + add);
        *reinterpret_cast<float4*>(row + 64 * g + 8 * r + 4) =
            make_float4(o[n][g][0][c + 2] + add, o[n][g][1][c + 2] + add, o[n][g][2][c + 2] + add, o[n][g][3][c + 2] + add);
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
      const float f = exp2f(ml[(w * QS + h) * 2] - top);
      den += f * ml[(w * QS + h) * 2 + 1];
      const float4 v = *reinterpret_cast<const float4*>(ow + (w * QS + h) * PITCH + d);
      y[0] += f * v.x, y[1] += f * v.y, y[2] += f * v.z, y[3] += f * v.w;
    }
    const float lse2 = top + log2f(den);
    if (a.splits > 1) {
      const long at = ((long)slot * a.nq + kvh * R + h) * a.splits + split;
      *reinterpret_cast<float4*>(a.mid_o + at * D + d) = make_float4(y[0] / den, y[1] / den, y[2] / den, y[3] / den);
      if (d == 0) a.mid_lse[at] = lse2;
    } else {
      uint2 packed;
      packed.x = pack_bf16(y[0] / den, y[1] / den);
      packed.y = pack_bf16(y[2] / den, y[3] / den);
      *reinterpret_cast<uint2*>(a.out + (out_row + h) * D + d) = packed;
      if (a.lse && d == 0) a.lse[out_row + h] = lse2 * LN_2;
    }
  }
}

// Slices of a (sequence, head), in order: a warp per head.
template <int D> __global__ void __launch_bounds__(THREADS) merge_4bit_kernel(Decode a, int heads) {
  pdl_wait();
  pdl_launch_dependents();
  const int item = blockIdx.x * WARPS + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (item >= heads) return;
  const int slot = item / a.nq, h = item - slot * a.nq;
  const int seq = a.seq_list ? a.seq_list[slot] : slot;
  const int kv_len = min(a.kv_lens[seq], a.max_len), tok = a.cu_seqlens[seq];
  const int lo = a.window > 0 ? max(0, kv_len - a.window) : 0;
  const int per = slice_keys(a);
  const int slices = min(a.splits, (kv_len - lo + per - 1) / per);
  const float* lses = a.mid_lse + (long)item * a.splits;
  const float* os = a.mid_o + (long)item * a.splits * D;
  float top = MINUS_BIG;
  for (int s = 0; s < slices; ++s) top = fmaxf(top, lses[s]);
  float den = 0.f, y[D / 128 > 0 ? D / 128 : 1][4] = {};
  constexpr int PER = D / 4 < 32 ? D / 4 : 32;
  for (int s = 0; s < slices; ++s) {
    const float f = exp2f(lses[s] - top);
    den += f;
#pragma unroll
    for (int c = 0; c < (D >= 128 ? D / 128 : 1); ++c)
      if (lane < PER) {
        const float4 v = *reinterpret_cast<const float4*>(os + (long)s * D + 128 * c + 4 * lane);
        y[c][0] += f * v.x, y[c][1] += f * v.y, y[c][2] += f * v.z, y[c][3] += f * v.w;
      }
  }
  const float inv = slices > 0 ? 1.f / den : 0.f;
  bf16* row = a.out + ((long)tok * a.nq + h) * D;
#pragma unroll
  for (int c = 0; c < (D >= 128 ? D / 128 : 1); ++c)
    if (lane < PER) {
      uint2 packed;
      packed.x = pack_bf16(y[c][0] * inv, y[c][1] * inv);
      packed.y = pack_bf16(y[c][2] * inv, y[c][3] * inv);
      *reinterpret_cast<uint2*>(row + 128 * c + 4 * lane) = packed;
    }
  if (a.lse && lane == 0) a.lse[(long)tok * a.nq + h] = slices > 0 ? (top + log2f(den)) * LN_2 : -INFINITY;
}

template <int D, int NT> int launch_decode(const Decode& a, int num_seqs, cudaStream_t stream) {
  constexpr int ring = WARPS * STAGES * Head<D>::STAGE;
  constexpr int joined = WARPS * 8 * NT * (D + 4 + 2) * 4;
  constexpr int smem = ring > joined ? ring : joined;
  static bool once[Q3_MAX_DEVICES];
  const int dev = q3_current_device();
  if (!once[dev]) {
    if (cudaFuncSetAttribute(decode_4bit_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
      return Q3_ERR_LAUNCH;
    once[dev] = true;
  }
  cudaError_t err = launch_pdl(decode_4bit_kernel<D, NT>, dim3(a.splits, a.nkv, num_seqs), dim3(THREADS), smem, stream, a);
  if (err == cudaSuccess && a.splits > 1) {
    const int heads = num_seqs * a.nq;
    err = launch_pdl(merge_4bit_kernel<D>, dim3((heads + WARPS - 1) / WARPS), dim3(THREADS), 0, stream, a, heads);
  }
  return err == cudaSuccess ? Q3_OK : Q3_ERR_LAUNCH;
}

// ---- sums of attention weights -----------------------------------------------------------------------------------------------------
// mass[key] += sum over a sequence's last `observe` tokens and the query heads of the kv head of 2^(score - log sum of the row).  Three
// kernels: the rows' log sums (left out when the attention has them), their slices joined, and the columns' sums.  Rows are
// (token, head of the group), token by token; the scores' tiles are those of decode attention, with the numbers as 1 + n / 16: what
// has to be taken off the sums is then no larger than they are, and the sums keep float32's precision (with 128 + n seven bits of it go).
// A cached token's sum belongs to one lane: no atomics, the same bits every time.
template <int J> __device__ __forceinline__ uint32_t sixteenths_of(uint32_t w) {
  const uint32_t x = J == 0 ? w << 3 : w >> (4 * J - 3 > 0 ? 4 * J - 3 : 0);
  return (x & 0x00780078u) | 0x3F803F80u;
}

struct Mass {
  const bf16* q;
  int q_stride;
  const unsigned char* pages;
  int num_pages;
  const int *block_table, *kv_lens, *cu_seqlens;
  int max_pages, nq, nkv, ps, max_len, observe, slices, num_seqs;
  float scale_log2;
  float* lse;    // [tokens][nq], natural logarithms
  float2* part;  // [tokens][nq][slices]: maximum and sum
  float* mass;
};

template <int D> struct KeyTile {  // 16 keys as A fragments
  uint32_t a[Head<D>::WORDS][2][4];
  float s[2][Head<D>::G], z[2][Head<D>::G];  // 16 * scale, minimum
  // rows of keys first + r and first + r + 8; what is not there is zero
  __device__ __forceinline__ void load(const Mass& m, const Q4Page& L, const int* bt, int kvh, int first, int end, int lane) {
    using H = Head<D>;
    const int r = lane >> 2, l = lane & 3;
    uint32_t w[2][H::WORDS], p[2][H::G];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int key = first + r + 8 * half;
      int page = key < end ? bt[key / m.ps] : -1;
      const bool valid = page >= 0 && page < m.num_pages;
#pragma unroll
      for (int j = 0; j < H::WORDS; ++j) w[half][j] = 0;
#pragma unroll
      for (int g = 0; g < H::G; ++g) p[half][g] = 0;
      if (valid) {
        const unsigned char* rec = m.pages + ((long)page * m.nkv + kvh) * L.record;
        const unsigned char* row = rec + (long)(key % m.ps) * H::ROW;
        const unsigned char* par = rec + L.kpar + (long)(key % m.ps) * H::PAR;
        if constexpr (D == 64) {
          *reinterpret_cast<uint2*>(&w[half][0]) = *reinterpret_cast<const uint2*>(row + 8 * l);
          p[half][0] = *reinterpret_cast<const uint32_t*>(par);
        } else if constexpr (D == 128) {
          *reinterpret_cast<uint4*>(&w[half][0]) = *reinterpret_cast<const uint4*>(row + 16 * l);
          *reinterpret_cast<uint2*>(&p[half][0]) = *reinterpret_cast<const uint2*>(par);
        } else {
          *reinterpret_cast<uint4*>(&w[half][0]) = *reinterpret_cast<const uint4*>(row + 16 * l);
          *reinterpret_cast<uint4*>(&w[half][4]) = *reinterpret_cast<const uint4*>(row + 16 * (l + 4));
          *reinterpret_cast<uint4*>(&p[half][0]) = *reinterpret_cast<const uint4*>(par);
        }
      }
    }
#pragma unroll
    for (int g = 0; g < H::G; ++g) {
      s[0][g] = 16.f * q4_s(p[0][g]), s[1][g] = 16.f * q4_s(p[1][g]);
      z[0][g] = q4_z(p[0][g]), z[1][g] = q4_z(p[1][g]);
    }
#pragma unroll
    for (int j = 0; j < H::WORDS; ++j) {
      a[j][0][0] = sixteenths_of<0>(w[0][j]), a[j][0][1] = sixteenths_of<0>(w[1][j]);
      a[j][0][2] = sixteenths_of<1>(w[0][j]), a[j][0][3] = sixteenths_of<1>(w[1][j]);
      a[j][1][0] = sixteenths_of<2>(w[0][j]), a[j][1][1] = sixteenths_of<2>(w[1][j]);
      a[j][1][2] = sixteenths_of<3>(w[0][j]), a[j][1][3] = sixteenths_of<3>(w[1][j]);
    }
  }
  // scores (times scale, in powers of two): x[0], x[1] of key r and queries 2l, 2l + 1; x[2], x[3] of key r + 8
  __device__ __forceinline__ void scores(float (&x)[4], const uint32_t (&q)[Head<D>::WORDS][4], const float (&qsum)[Head<D>::G][2],
                                         float scale_log2) const {
    using H = Head<D>;
    float acc[H::G][4];
#pragma unroll
    for (int g = 0; g < H::G; ++g) {
      acc[g][0] = acc[g][2] = -qsum[g][0];
      acc[g][1] = acc[g][3] = -qsum[g][1];
    }
#pragma unroll
    for (int j = 0; j < H::WORDS; ++j) {
      mma_bf16(acc[H::group(j)], a[j][0], q[j][0], q[j][1]);
      mma_bf16(acc[H::group(j)], a[j][1], q[j][2], q[j][3]);
    }
    x[0] = x[1] = x[2] = x[3] = 0.f;
#pragma unroll
    for (int g = 0; g < H::G; ++g) {
      x[0] += s[0][g] * acc[g][0] + z[0][g] * qsum[g][0];
      x[1] += s[0][g] * acc[g][1] + z[0][g] * qsum[g][1];
      x[2] += s[1][g] * acc[g][2] + z[1][g] * qsum[g][0];
      x[3] += s[1][g] * acc[g][3] + z[1][g] * qsum[g][1];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] *= scale_log2;
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
  float qsum[NT][H::G][2], m[NT][2], sum[NT][2];
  int sees[NT][2];  // the last key that the row's token sees
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int row = row0 + 8 * n + r, i = row / R;
    load_query<D>(q[n], i < rows.count ? a.q + (long)(rows.first + i) * a.q_stride + (long)(kvh * R + row % R) * D : nullptr, lane);
    query_sums<D>(qsum[n], q[n]);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      m[n][c] = MINUS_BIG, sum[n][c] = 0.f;
      sees[n][c] = min(end - 1, rows.before + (row0 + 8 * n + 2 * l + c) / R);
    }
  }
  for (int first = begin + STEP * warp; first < end; first += STEP * WARPS) {
    KeyTile<D> k;
    k.load(a, L, bt, kvh, first, end, lane);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float x[4];
      k.scores(x, q[n], qsum[n], a.scale_log2);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float x0 = first + r <= sees[n][c] ? x[c] : -INFINITY, x1 = first + r + 8 <= sees[n][c] ? x[c + 2] : -INFINITY;
        const float top = fmaxf(m[n][c], fmaxf(x0, x1));
        sum[n][c] = sum[n][c] * exp2f(m[n][c] - top) + exp2f(x0 - top) + exp2f(x1 - top);
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
        sum[n][c] = sum[n][c] * exp2f(m[n][c] - top) + os * exp2f(om - top);
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
    for (int w = 0; w < WARPS; ++w) den += joined[w][tid].y * exp2f(joined[w][tid].x - top);
    const long at = (long)(rows.first + row / R) * a.nq + kvh * R + row % R;
    if (a.slices > 1)
      a.part[at * a.slices + slice] = make_float2(top, den);
    else
      a.lse[at] = (top + log2f(den)) * LN_2;
  }
}

__global__ void mass_join_kernel(Mass a) {  // grid (blocks over observed rows, sequence)
  pdl_wait();
  pdl_launch_dependents();
  const Rows rows(a, blockIdx.y);
  const int u = blockIdx.x * blockDim.x + threadIdx.x;
  if (u >= rows.count * a.nq) return;
  const long at = (long)rows.first * a.nq + u;
  float top = MINUS_BIG, den = 0.f;
  for (int s = 0; s < a.slices; ++s) top = fmaxf(top, a.part[at * a.slices + s].x);
  for (int s = 0; s < a.slices; ++s) {
    const float2 y = a.part[at * a.slices + s];
    den += y.y * exp2f(y.x - top);
  }
  a.lse[at] = (top + log2f(den)) * LN_2;
}

// Column sums: grid (blocks of 64 MT keys, kv head, sequence); a warp keeps 16 MT keys in registers and goes through the rows.
template <int D, int MT> __global__ void __launch_bounds__(THREADS) mass_columns_kernel(Mass a) {
  using H = Head<D>;
  pdl_wait();
  pdl_launch_dependents();
  const int seq = blockIdx.z, kvh = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, l = lane & 3, R = a.nq / a.nkv;
  const Rows rows(a, seq);
  const int kv_len = rows.before + rows.count;
  const int first = (blockIdx.x * WARPS + warp) * STEP * MT;
  if (first >= kv_len || rows.count == 0) return;
  const Q4Page L(D, H::G, a.ps);
  const int* bt = a.block_table + (long)seq * a.max_pages;
  KeyTile<D> k[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) k[t].load(a, L, bt, kvh, first + STEP * t, kv_len, lane);
  float total[MT][2];
#pragma unroll
  for (int t = 0; t < MT; ++t) total[t][0] = total[t][1] = 0.f;
  // rows of tokens that see none of these keys are left out
  const int start = max(0, first - rows.before) * R;
  for (int row0 = start & ~7; row0 < rows.count * R; row0 += 8) {
    uint32_t q[H::WORDS][4];
    float qsum[H::G][2];
    {
      const int row = row0 + r, i = row / R;
      load_query<D>(q, i < rows.count ? a.q + (long)(rows.first + i) * a.q_stride + (long)(kvh * R + row % R) * D : nullptr, lane);
      query_sums<D>(qsum, q);
    }
    float lse2[2];
    int sees[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int row = row0 + 2 * l + c, i = row / R;
      const bool is = i < rows.count;
      lse2[c] = is ? a.lse[(long)(rows.first + i) * a.nq + kvh * R + row % R] * LOG2_E : 0.f;
      sees[c] = is ? rows.before + i : -1;
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      float x[4];
      k[t].scores(x, q, qsum, a.scale_log2);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = first + STEP * t + r + 8 * (e >> 1);
        total[t][e >> 1] += key <= sees[e & 1] ? exp2f(x[e] - lse2[e & 1]) : 0.f;
      }
    }
  }
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float y = total[t][half];
      y += __shfl_xor_sync(0xffffffffu, y, 1);
      y += __shfl_xor_sync(0xffffffffu, y, 2);
      const int key = first + STEP * t + r + 8 * half;
      if (l == 0 && key < kv_len) {
        const int page = bt[key / a.ps];
        if (page >= 0 && page < a.num_pages) a.mass[((long)page * a.nkv + kvh) * a.ps + key % a.ps] += y;
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
  if (rows.count) a.mass[((long)page * a.nkv + kvh) * a.ps + key % a.ps] += total;
}

template <int D, int NT, int MT> int launch_mass(const Mass& a, bool want_rows, int most_tokens, cudaStream_t stream) {
  const int rows = most_tokens * (a.nq / a.nkv);
  cudaError_t err = cudaSuccess;
  if (want_rows) {
    err = launch_pdl(mass_rows_kernel<D, NT>, dim3(a.slices, (rows + 8 * NT - 1) / (8 * NT), a.num_seqs * a.nkv), dim3(THREADS), 0, stream, a);
    if (err == cudaSuccess && a.slices > 1)
      err = launch_pdl(mass_join_kernel, dim3((most_tokens * a.nq + 127) / 128, a.num_seqs), dim3(128), 0, stream, a);
  }
  constexpr int KEYS = WARPS * STEP * MT;
  if (err == cudaSuccess)
    err = launch_pdl(mass_columns_kernel<D, MT>, dim3((a.max_len + KEYS - 1) / KEYS, a.nkv, a.num_seqs), dim3(THREADS), 0, stream, a);
  return err == cudaSuccess ? Q3_OK : Q3_ERR_LAUNCH;
}

}  // namespace

// `lse` holds the observed rows' log sums (have_lse) or is scratch for them; `part` [tokens][nq][slices] pairs of floats when slices > 1.
Q3_EXPORT int q3_attention_mass_4bit(int dtype, const void* q, int q_stride, const void* pages, int num_pages, const int* block_table,
                                     int max_pages, const int* kv_lens, const int* cu_seqlens, float* mass, float* lse, int have_lse,
                                     void* part, int slices, int num_seqs, int nq, int nkv, int D, int ps, float scale, int max_len,
                                     int observe, int most_tokens, cudaStream_t stream) {
  if (!q || !pages || !block_table || !kv_lens || !cu_seqlens || !mass || !lse || nq < 1 || nkv < 1 || nq % nkv || !q4_sizes_ok(D, ps) ||
      slices < 1 || (slices > 1 && !part) || observe < 1 || max_len > (long)max_pages * ps)
    return Q3_ERR_ARGUMENT;
  if (dtype != Q3_DTYPE_F32 && dtype != Q3_DTYPE_BF16) return Q3_ERR_ARGUMENT;
  if (num_seqs < 1 || most_tokens < 1 || max_len < 1) return Q3_OK;
  if (q_stride % 8 || (reinterpret_cast<uintptr_t>(q) & 15) || (reinterpret_cast<uintptr_t>(pages) & 15) ||
      (long)num_seqs * nkv > 65535 || nq > 65535)
    return Q3_ERR_UNSUPPORTED;
  Mass a{(const bf16*)q, q_stride, (const unsigned char*)pages, num_pages, block_table, kv_lens, cu_seqlens, max_pages, nq, nkv, ps,
         max_len, observe, slices, num_seqs, scale * LOG2_E, lse, (float2*)part, mass};
  if (dtype == Q3_DTYPE_BF16 && (D == 64 || D == 128 || D == 256)) {
    if ((long)most_tokens * (nq / nkv) > 65535L * 16) return Q3_ERR_UNSUPPORTED;
    if (D == 64) return launch_mass<64, 4, 2>(a, !have_lse, most_tokens, stream);
    if (D == 128) return launch_mass<128, 4, 2>(a, !have_lse, most_tokens, stream);
    return launch_mass<256, 2, 1>(a, !have_lse, most_tokens, stream);
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
                                       int splits, int max_len, const int* longest, cudaStream_t stream) {
  if (!q || !pages || !block_table || !kv_lens || !cu_seqlens || !out || nq < 1 || nkv < 1 || nq % nkv || ps < 1 || splits < 1 ||
      (splits > 1 && (!mid_o || !mid_lse)) || max_len > (long)max_pages * ps)
    return Q3_ERR_ARGUMENT;
  const int R = nq / nkv;
  if (R > 16 || q_stride % 8 || (reinterpret_cast<uintptr_t>(q) & 15) || (reinterpret_cast<uintptr_t>(pages) & 15) ||
      (reinterpret_cast<uintptr_t>(out) & 7) || num_seqs > 65535 || nkv > 65535)
    return Q3_ERR_UNSUPPORTED;
  if (num_seqs < 1) return Q3_OK;
  Decode a{(const bf16*)q, q_stride, (const unsigned char*)pages, num_pages, block_table, kv_lens, cu_seqlens, seq_list, max_pages,
           (bf16*)out, mid_o, mid_lse, lse, nq, nkv, ps, window, splits, max_len, scale * LOG2_E, longest};
  if (D == 64) return R <= 8 ? launch_decode<64, 1>(a, num_seqs, stream) : launch_decode<64, 2>(a, num_seqs, stream);
  if (D == 128) return R <= 8 ? launch_decode<128, 1>(a, num_seqs, stream) : launch_decode<128, 2>(a, num_seqs, stream);
  if (D == 256) return R <= 8 ? launch_decode<256, 1>(a, num_seqs, stream) : launch_decode<256, 2>(a, num_seqs, stream);
  return Q3_ERR_UNSUPPORTED;
}
