// Attention of portions of prompts whose sequences' keys and values were unpacked from a cache in 8 bits (csrc/cache_8bit.cu), on the 5th-generation tensor
// cores: heads of 64 to 256 (a multiple of 16; columns that a head lacks lie beyond the tensors' inner extent and arrive as zeros), any group of up to 128,
// optionally under a window, whose tokens may see the sequence's first ones as well.  The products, the softmax and their order are those of
// attention_prefill_tc.cu, whose head comment has the reasons and what was tried; what differs is how blocks get their work:
//
//   * Keys and values lie in tiles of 64 tokens, in a sequence's order, so a tile's place follows from the item alone, and 64 columns of it are one TMA box.
//   * An item is a sequence's 2 x 128 rows (A and B; as many as whole tokens give) for one kv head.  WIDE, heads of more than 128, whose results take half of
//     the tensor memory: one block of rows, with scores in two places by turns, so that the next product does not wait for the softmax.
//   * Blocks stay: one an SM takes item after item from a list that begins with the heaviest (csrc/cache_8bit.cu writes it), the next one when the keys of the
//     present one are all asked for.  Then the next item's queries, keys and first product come while the softmax ends the present one and writes its rows.
//   * Where items would leave SMs idle (a portion behind a long context), each one's tiles are cut into slices, items of their own; a second kernel joins
//     what they leave.
//
// What bounds it: 0.96 us a tile of both blocks (the softmax, as there: the tensor pipe is busy in 0.51 of the clocks, WIDE 0.58, the exponentials' in 0.41 and
// 0.24, and warps wait for tensor memory most), and what an item costs beside its tiles.  With a block of the launch for each item that
// was 6.5 us (1.1 between two blocks, 0.5 for the item, 2.8 until the first scores, 2 to 2.6 at the end), now the end's.  us, with the unpacking, 32 heads over
// 8 of 128, in blocks that stay and one for each item: 1,500 + 701 + 1,000 (behind 2,048) tokens and a single one 79, 87; 700 + 2,048 + 500 (behind 5,000) under
// a window of 1,024 59, 67 (straight over the codes 230); a prompt of 2,048 42, 47.  In slices and without: 64 tokens behind 4,000 28, 64; behind 16,000 52,
// 230.  WIDE, 16 heads over 2 of 256, and straight over the codes: a prompt of 2,048 40, 186; the first of the above 77, 387.
//
// Warps:  0 takes items and brings keys, 1 values, 2 queries;  4..7 and 8..11 softmax of block A and B, one thread per row;  12, 13 issue S = Q K^T,
// 14, 15 O += P V (WIDE: 4..7, 12 and 14).  An item passes through a ring of two places in shared memory.  What runs on from item to item are the rings' places
// and the numbers of scores and weights so far, whose last bits are the barriers' phases.  Tensor memory as there: per block S [0,64), P_0 and P_1 [64,128),
// O [128,256); WIDE: S_0 and S_1 [0,128), P_0 and P_1 [128,192), O [256,512).
// Every wait is bounded and, where a whole warp goes on behind it, of one mind; on expiry the block raises its abort flag and the error word, waits for its
// copies and products in flight, frees its tensor memory and returns.
#pragma once
#include <type_traits>

#include "async_tiles.cuh"
#include "prompt_slices.cuh"

namespace {

constexpr int BLOCK_M = 128, BLOCK_N = 64, THREADS = 512, TMEM_COLS = 512;
constexpr int PART_Q = BLOCK_M * 128;   // 64 columns of a block's queries: [128 rows][128 B]
constexpr int PART_KV = BLOCK_N * 128;  // 64 columns of a tile of keys or values
constexpr int STAGE_OUT = BLOCK_M * 128;  // 64 columns of a block's results
template <bool WIDE> struct Sizes {
  static constexpr int PARTS = WIDE ? 4 : 2, BLOCKS = WIDE ? 1 : 2, STAGES = WIDE ? 2 : 4;  // of 64 columns; of rows; of keys and values in flight
  static constexpr int Q_BYTES = PARTS * PART_Q, KV_BYTES = PARTS * PART_KV;
  static constexpr int SMEM = BLOCKS * Q_BYTES + 2 * STAGES * KV_BYTES + BLOCKS * STAGE_OUT + 1024;
  static constexpr int TMEM_BLOCK = 256, TMEM_P = WIDE ? 128 : 64, TMEM_O = WIDE ? 256 : 128;
  static constexpr int CONSUMERS = WIDE ? 8 : 14;  // warps that read an item
};

constexpr int MOST_STAGES = 4;
enum { Q_FULL, Q_EMPTY, K_FULL, K_EMPTY = K_FULL + MOST_STAGES, V_FULL = K_EMPTY + MOST_STAGES, V_EMPTY = V_FULL + MOST_STAGES,
       S_FULL = V_EMPTY + MOST_STAGES,  // [block] (WIDE: [place]) ..
       S_EMPTY = S_FULL + 2, P_FULL = S_EMPTY + 2, PV_FULL = P_FULL + 2, ITEM_FULL = PV_FULL + 2, ITEM_EMPTY = ITEM_FULL + 2, END = ITEM_EMPTY + 2,
       NUM_BARS = END + 4 };

struct Params {
  int4* items;  // [num_items][2], then a number that counts what blocks have taken beyond their first
  bf16* out;
  int num_items, nq, nkv, group, per, magic, head_dim, window, keep_first;  // per: tokens of a block; magic: 2^16 / group, rounded up
  float scale_log2;
  int* error_word;
  int splits;
  float *mid_o, *mid_ml;  // splits > 1: see PromptSlices
};

__device__ __forceinline__ float ex2(float x) {  // 2^x; below 2^-126 zero, which is what a weight that small is worth
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
// a row's accumulators in tensor memory times `corr`; rare, and out of line: branches are what the softmax warps stumble over
__device__ __noinline__ void rescale_rows(uint32_t o_addr, float corr, int cols) {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
  for (int c0 = 0; c0 < cols; c0 += 32) {
    uint32_t ov[32];
    tmem_load32(o_addr + c0, ov);
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int c = 0; c < 32; ++c) ov[c] = __float_as_uint(__uint_as_float(ov[c]) * corr);
    tmem_store32(o_addr + c0, ov);
  }
}
__device__ __forceinline__ void arrive_if(bool yes, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q mbarrier.arrive.shared::cta.b64 _, [%0];\n\t}"
      ::"r"(bar), "r"((uint32_t)yes)
      : "memory");
}

// An item, as all roles see it.  Its tokens are its sequence's tokens first .. ; tile j of its keys (of this slice, its tile j + j0) is tile `at(j)` of the sequence.
template <int BLOCKS> struct Item {
  int kvh, slice, tok0, q_len, base_pos, first, k_lo, p_last, firsts, skip, p_max[2], tiles[2], j0, num_tiles, place, kept, gap;
  __device__ __forceinline__ Item(const Params& p, const int4& what, const int4& where) {
    kvh = where.w & 0xffff, slice = where.w >> 16, tok0 = what.y, q_len = what.z, base_pos = what.w - what.z, first = BLOCKS * p.per * what.x;
    k_lo = p.window > 0 ? max(0, base_pos + first - p.window + 1) : 0;
    const int tile0 = k_lo / BLOCK_N;
    firsts = min((p.keep_first + BLOCK_N - 1) / BLOCK_N, tile0), skip = tile0 - firsts;
#pragma unroll
    for (int x = 0; x < 2; ++x) {  // B may not exist
      const int begin = first + x * p.per, end = min(q_len, begin + p.per);
      p_max[x] = x < BLOCKS && begin < q_len ? base_pos + end - 1 : -1;
      tiles[x] = p_max[x] >= 0 ? p_max[x] / BLOCK_N + 1 - skip : 0;
    }
    num_tiles = max(tiles[0], tiles[1]), p_last = max(p_max[0], p_max[1]), j0 = 0;
    if (p.splits > 1) {
      const int per = (num_tiles + p.splits - 1) / p.splits;
      j0 = slice * per;
      tiles[0] = max(0, min(tiles[0] - j0, per)), tiles[1] = max(0, min(tiles[1] - j0, per)), num_tiles = max(tiles[0], tiles[1]);
    }
    place = where.x, kept = where.y, gap = where.z - where.y;
  }
  __device__ __forceinline__ int tiles_of(int x) const { return x ? tiles[1] : tiles[0]; }  // (an index would put them into local memory)
  __device__ __forceinline__ int at(int j) const { return j + j0 + (j + j0 >= firsts ? skip : 0); }
  __device__ __forceinline__ int row(const Params& p, int j) const {  // of the unpacked tiles, as rows
    const int t = at(j);
    return ((place + t - (t < kept ? 0 : gap)) * p.nkv + kvh) * BLOCK_N;
  }
};

template <bool WIDE>
__global__ void __launch_bounds__(THREADS, 1) prompts_tiles_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                                                                   const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ Params p) {
  typedef Sizes<WIDE> Z;
  typedef Item<Z::BLOCKS> Work;
  constexpr int STAGES = Z::STAGES, Q_BYTES = Z::Q_BYTES, KV_BYTES = Z::KV_BYTES, TMEM_P = Z::TMEM_P, TMEM_O = Z::TMEM_O;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* q_s = base;                        // BLOCKS x [PARTS][128 rows][128 B]
  unsigned char* k_s = q_s + Z::BLOCKS * Q_BYTES;   // STAGES x [PARTS][64 rows][128 B]
  unsigned char* v_s = k_s + STAGES * KV_BYTES;
  unsigned char* out_s = v_s + STAGES * KV_BYTES;   // BLOCKS x [128 rows][128 B]
  __shared__ __align__(8) unsigned long long bars[NUM_BARS];
  __shared__ uint32_t tmem_base_s;
  __shared__ volatile int abort_flag;
  __shared__ int4 item_s[2][2];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t bar0 = smem_addr(&bars[0]);
  auto bar = [&](int i) { return bar0 + 8u * (uint32_t)i; };
  if (tid == 0) {
    abort_flag = 0;
    mbar_init(bar(Q_FULL), 1);
    mbar_init(bar(Q_EMPTY), Z::BLOCKS);  // the issuers of S
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(bar(K_FULL + i), 1);
      mbar_init(bar(K_EMPTY + i), Z::BLOCKS);  // the blocks' issuers
      mbar_init(bar(V_FULL + i), 1);
      mbar_init(bar(V_EMPTY + i), Z::BLOCKS);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(S_FULL + i), 1);
      mbar_init(bar(S_EMPTY + i), 4);  // a block's softmax warps
      mbar_init(bar(P_FULL + i), 4);
      mbar_init(bar(PV_FULL + i), 1);
      mbar_init(bar(ITEM_FULL + i), 1);
      mbar_init(bar(ITEM_EMPTY + i), Z::CONSUMERS);
    }
    for (int i = 0; i < 4; ++i) mbar_init(bar(END + i), 1);  // the issuers
    mbar_init_fence();
  }
  if (tid == 32)
    for (const CUtensorMap* map : {&tmap_q, &tmap_k, &tmap_v}) asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_base_s)), "r"(TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = tmem_base_s;
  pdl_wait();  // (the kernel that unpacks may have been at work on its last pages)

  const int parts = (p.head_dim + 63) / 64;
  int n = 0;  // items so far
  int4 what, where;
  // The next item, from its place in the ring; whole warps.  False: there is none, or somebody gave up.
  auto next_item = [&]() -> bool {
    const int slot = n & 1;
    if (!__all_sync(0xffffffffu, mbar_wait(bar(ITEM_FULL + slot), (n >> 1) & 1, &abort_flag))) return false;
    what = item_s[slot][0], where = item_s[slot][1];
    __syncwarp();
    arrive_if(lane == 0, bar(ITEM_EMPTY + slot));
    ++n;
    return what.x >= 0;
  };

  if (warp == 0) {  // ---- items, and their keys
    const int each = p.nkv * p.splits, units = p.num_items * each;  // item by item, the slices of each, the kv heads of each
    int unit = blockIdx.x, c = 0;
    bool ok = true;
    for (;; ++n) {
      what = make_int4(-1, 0, 0, 0), where = make_int4(0, 0, 0, 0);
      if (unit < units) {  // (an item that is none: the list's end)
        const int item = unit / each, rest = unit - item * each, slice = rest / p.nkv;
        what = p.items[2 * item], where = p.items[2 * item + 1];
        where.w = rest - slice * p.nkv + (slice << 16);
      }
      const int slot = n & 1;
      ok = __all_sync(0xffffffffu, mbar_wait(bar(ITEM_EMPTY + slot), ((n >> 1) & 1) ^ 1, &abort_flag));
      if (!ok) break;
      if (lane == 0) {
        item_s[slot][0] = what, item_s[slot][1] = where;
        mbar_arrive(bar(ITEM_FULL + slot));
      }
      __syncwarp();
      if (what.x < 0) break;
      const Work it(p, what, where);
      for (int j = 0; j < it.num_tiles; ++j, ++c) {
        const int st = c % STAGES;
        ok = __all_sync(0xffffffffu, mbar_wait(bar(K_EMPTY + st), ((c / STAGES) & 1) ^ 1, &abort_flag));
        if (!ok) break;
        if (lane == 0) {
          mbar_expect_tx(bar(K_FULL + st), parts * PART_KV);
          for (int h = 0; h < parts; ++h)
#ifdef Q3_TEST_WITHHOLD_A_BOX  // (a test build leaves the second part of the keys out: the stage never fills, a wait runs out)
            if (h != 1)
#endif
            tma_load_2d(smem_addr(k_s) + st * KV_BYTES + h * PART_KV, &tmap_k, bar(K_FULL + st), 64 * h, it.row(p, j));
        }
        __syncwarp();
      }
      if (!ok) break;
      int more = 0;
      if (lane == 0) more = atomicAdd(reinterpret_cast<int*>(p.items + 2 * p.num_items), 1);
      unit = gridDim.x + __shfl_sync(0xffffffffu, more, 0);
    }
    // the last boxes may still be in flight when others have given up
    if (lane == 0)
      for (int i = max(0, c - STAGES); i < c; ++i) mbar_wait_drain(bar(K_FULL + i % STAGES), (i / STAGES) & 1);
  } else if (warp == 1) {  // ---- values
    int c = 0;
    bool ok = true;
    while (ok && next_item()) {
      const Work it(p, what, where);
      for (int j = 0; j < it.num_tiles; ++j, ++c) {
        const int st = c % STAGES;
        ok = __all_sync(0xffffffffu, mbar_wait(bar(V_EMPTY + st), ((c / STAGES) & 1) ^ 1, &abort_flag));
        if (!ok) break;
        if (lane == 0) {
          mbar_expect_tx(bar(V_FULL + st), parts * PART_KV);
          for (int h = 0; h < parts; ++h) tma_load_2d(smem_addr(v_s) + st * KV_BYTES + h * PART_KV, &tmap_v, bar(V_FULL + st), 64 * h, it.row(p, j));
        }
        __syncwarp();
      }
    }
    if (lane == 0)
      for (int i = max(0, c - STAGES); i < c; ++i) mbar_wait_drain(bar(V_FULL + i % STAGES), (i / STAGES) & 1);
  } else if (warp == 2) {  // ---- queries
    int c = 0;
    while (next_item()) {
      const Work it(p, what, where);
      if (!__all_sync(0xffffffffu, mbar_wait(bar(Q_EMPTY), (c & 1) ^ 1, &abort_flag))) break;
      if (lane == 0) {
        const int blocks = it.tiles[1] ? 2 : it.tiles[0] ? 1 : 0;
        mbar_expect_tx(bar(Q_FULL), blocks * parts * p.per * p.group * 128);
        for (int x = 0; x < blocks; ++x)
          for (int h = 0; h < parts; ++h)
            tma_load_3d(smem_addr(q_s) + x * Q_BYTES + h * PART_Q, &tmap_q, bar(Q_FULL), 64 * h, it.kvh * p.group, it.tok0 + it.first + x * p.per);
      }
      __syncwarp();
      ++c;
    }
    if (lane == 0 && c > 0) mbar_wait_drain(bar(Q_FULL), (c - 1) & 1);
  } else if (warp > 11 && !(WIDE && (warp & 1))) {  // ---- issuers: warps 12 and 13 S of block A and B, warps 14 and 15 PV
    const int role = __shfl_sync(0xffffffffu, warp, 0), x = role & 1;
    const uint32_t tmem_x = __shfl_sync(0xffffffffu, tmem, 0) + x * Z::TMEM_BLOCK;
    const bool leader = elect_one();
    auto wait_all = [&](int b, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar(b), parity, &abort_flag)); };
    int st = 0, c = 0;  // c: this block's scores (or weights) so far
    uint32_t phase = 0;
    bool ok = true;
    while (ok && next_item()) {
      const Work it(p, what, where);
      const int mine = __shfl_sync(0xffffffffu, it.tiles_of(x), 0), all = __shfl_sync(0xffffffffu, it.num_tiles, 0);
      if (role < 14) {
        constexpr uint32_t idesc = umma_idesc(BLOCK_M, BLOCK_N, 0);  // S = Q K^T: N = 64 keys
        const uint32_t q_addr = smem_addr(q_s) + x * Q_BYTES;
        ok = wait_all(Q_FULL, (n - 1) & 1);
        if (ok && mine == 0) arrive_if(leader, bar(Q_EMPTY));
        for (int j = 0; j < all && ok; ++j) {
          // as soon as the softmax has the scores that lie in their place in its registers
          const int place = WIDE ? c & 1 : x, use = WIDE ? c >> 1 : c;
          ok = (j >= mine || use == 0 || wait_all(S_EMPTY + place, (use - 1) & 1)) && wait_all(K_FULL + st, phase);
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          if (leader) {
            if (j < mine) {
              const uint32_t k_addr = smem_addr(k_s) + st * KV_BYTES;
#pragma unroll
              for (int k = 0; k < 4 * Z::PARTS; ++k) {
                const uint32_t part = k >> 2, sub = (k & 3) * 2;  // 4 steps of 32 bytes per 64 columns
                if (16 * k < p.head_dim)
                  umma_bf16(tmem_x + (WIDE ? place * BLOCK_N : 0), umma_desc(q_addr + part * PART_Q) + sub, umma_desc(k_addr + part * PART_KV) + sub, idesc, k > 0 ? 1u : 0u);
              }
              umma_commit(bar(S_FULL + place));
              umma_commit(bar(K_EMPTY + st));
              if (j == mine - 1) umma_commit(bar(Q_EMPTY));  // the next item's queries may come
            } else {
              mbar_arrive(bar(K_EMPTY + st));
            }
          }
          __syncwarp();
          c += j < mine;
          if (++st == STAGES) st = 0, phase ^= 1;
        }
      } else {
        // N: the head's columns in whole parts, V with its rows as keys
        const uint32_t idesc = WIDE ? (parts == 3 ? umma_idesc(BLOCK_M, 192, 1) : umma_idesc(BLOCK_M, 256, 1))
                                    : (parts == 1 ? umma_idesc(BLOCK_M, 64, 1) : umma_idesc(BLOCK_M, 128, 1));
        for (int j = 0; j < all && ok; ++j) {
          ok = (j >= mine || wait_all(P_FULL + x, c & 1)) && wait_all(V_FULL + st, phase);  // the weights written, O at rest
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          if (leader) {
            if (j < mine) {
              const uint32_t v_addr = smem_addr(v_s) + st * KV_BYTES;
#pragma unroll
              for (int k = 0; k < BLOCK_N / 16; ++k)  // 16 keys: 8 columns of P, 2 KB down V's rows
                umma_bf16_tmem(tmem_x + TMEM_O, tmem_x + TMEM_P + (c & 1) * (BLOCK_N / 2) + 8 * k, umma_desc_mn_major(v_addr + k * 2048, PART_KV), idesc,
                               (j > 0 || k > 0) ? 1u : 0u);
              umma_commit(bar(PV_FULL + x));
              umma_commit(bar(V_EMPTY + st));
            } else {
              mbar_arrive(bar(V_EMPTY + st));
            }
          }
          __syncwarp();
          c += j < mine;
          if (++st == STAGES) st = 0, phase ^= 1;
        }
      }
    }
    if (elect_one()) {  // (the same lane again) nothing of this issuer's is in flight any more when the tensor memory is freed
      umma_commit(bar(END + role - 12));
      mbar_wait_drain(bar(END + role - 12), 0);
    }
    __syncwarp();
  } else if (warp > 3 && warp < (WIDE ? 8 : 12)) {  // ---- softmax: one thread per row; warps 4..7 block A, warps 8..11 block B
    const int x = (warp - 4) >> 2, quarter = warp & 3, r = quarter * 32 + lane;  // row of the tile = lane of tensor memory
    const int token = r * p.magic >> 16, head = r - token * p.group;
    const uint32_t lane_base = tmem + x * Z::TMEM_BLOCK + ((uint32_t)(quarter * 32) << 16), o_addr = lane_base + TMEM_O;
    const float scale_log2 = p.scale_log2;
    // O stays in tensor memory.  The reference point of the exponentials (m_ref) moves only when a row's maximum exceeds it by more than 2^8 after scaling;
    // then O and l are rescaled.  Weights may reach 2^8, which bfloat16 and float32 hold easily, and O / l is the same.
    const float slack = fminf(8.f / scale_log2, 1e38f);
    const float2 scale2 = make_float2(scale_log2, scale_log2);
    int c = 0, tiles_before = 0;  // this block's scores so far, and the tiles of all items before
    bool ok = true;
    while (ok && next_item()) {
      const Work it(p, what, where);
      const int tok = it.first + x * p.per + token;  // of the sequence's
      const bool row_ok = token < p.per && tok < it.q_len;
      const int pos = row_ok ? it.base_pos + tok : -1, lo = row_ok && p.window > 0 ? max(0, pos - p.window + 1) : 0;
      const int my_tiles = it.tiles_of(x), keep = p.keep_first;
      float m_ref = -INFINITY, l_run = 0.f;
      // One tile.  EDGE: some row of the block does not see all of its keys, or some of them lie outside of what the item reads; the others have no
      // branch but the rare one for a new reference point.
      auto step = [&](int j, auto edge) -> bool {
        constexpr bool EDGE = decltype(edge)::value;
        const int key0 = it.at(j) * BLOCK_N, buffer = (c + j) & 1, place = WIDE ? buffer : x;
        if (!mbar_wait_warp(bar(S_FULL + place), WIDE ? ((c + j) >> 1) & 1 : buffer, &abort_flag)) return false;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        uint32_t sa[32], sb[32];
        const uint32_t s_addr = lane_base + (WIDE ? buffer * BLOCK_N : 0);
        tmem_load32(s_addr, sa);
        tmem_load32(s_addr + 32, sb);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        arrive_if(lane == 0, bar(S_EMPTY + place));
        if constexpr (EDGE) {
          if (key0 + BLOCK_N - 1 > pos) {  // the tile crosses this row's diagonal
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              if (key0 + e > pos) sa[e] = 0xff800000u;  // -inf
              if (key0 + 32 + e > pos) sb[e] = 0xff800000u;
            }
          }
          if (key0 < lo) {  // keys before the window
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              if (key0 + e < lo && key0 + e >= keep) sa[e] = 0xff800000u;
              if (key0 + 32 + e < lo && key0 + 32 + e >= keep) sb[e] = 0xff800000u;
            }
          }
        }
        float mx;
        {  // eight independent running maxima: a single chain of 64 would expose its latency
          float part[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) part[e] = fmaxf(__uint_as_float(sa[e]), __uint_as_float(sb[e]));
#pragma unroll
          for (int e = 8; e < 32; ++e) part[e & 7] = fmaxf(part[e & 7], fmaxf(__uint_as_float(sa[e]), __uint_as_float(sb[e])));
          mx = fmaxf(fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])), fmaxf(fmaxf(part[4], part[5]), fmaxf(part[6], part[7])));
        }
        const float m_old = m_ref;
        m_ref = mx > m_ref + slack ? mx : m_ref;  // (also from -infinity)
        const bool moved = __any_sync(0xffffffffu, m_ref != m_old);
        const float m_use = m_ref == -INFINITY ? 0.f : m_ref;
        // weights, rounded to bfloat16 as the product will see them, into tensor memory; the scaling and the row sum run on pairs
        float2 sums[4] = {{0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}};
        uint32_t w[32];
        const float2 neg2 = make_float2(-m_use * scale_log2, -m_use * scale_log2);
#pragma unroll
        for (int ch = 0; ch < 8; ++ch) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int i = ch * 8 + 2 * e;
            const float2 s2 = make_float2(__uint_as_float(i < 32 ? sa[i & 31] : sb[i & 31]), __uint_as_float(i < 32 ? sa[(i + 1) & 31] : sb[(i + 1) & 31]));
            const float2 t2 = __ffma2_rn(s2, scale2, neg2);
            const float2 x2 = make_float2(ex2(t2.x), ex2(t2.y));
            sums[e] = __fadd2_rn(sums[e], x2);
            w[ch * 4 + e] = pack2(x2.x, x2.y);
          }
        }
        tmem_store32(lane_base + TMEM_P + buffer * (BLOCK_N / 2), w);
        {
          const float2 a = __fadd2_rn(sums[0], sums[1]), b = __fadd2_rn(sums[2], sums[3]), d = __fadd2_rn(a, b);
          const float corr = m_ref == m_old ? 1.f : exp2f((m_old - m_ref) * scale_log2);  // 0 from -infinity
          l_run = l_run * corr + (d.x + d.y);
        }
        // The product before must be finished before these weights are signalled: it keeps the barrier from running a phase ahead of the waiters, the
        // next weights go where the ones before were, and O must be at rest if it has to be rescaled.  (The last item's was waited for at its end.)
        if (!EDGE || j > 0) {
          if (!mbar_wait_warp(bar(PV_FULL + x), buffer ^ 1, &abort_flag)) return false;
          if (__builtin_expect(moved, 0)) rescale_rows(o_addr, m_ref == m_old ? 1.f : exp2f((m_old - m_ref) * scale_log2), 64 * Z::PARTS);
        }
        // Keys behind the item's last position, and those between the first tokens and its window, are nobody's, and their values may be what is no
        // number: zero before the product reads them (both blocks do, each before its own; keys between the blocks' last positions are real and only masked).
        if constexpr (EDGE) {
          if (key0 + BLOCK_N - 1 > it.p_last || key0 < it.k_lo) {
            const int tile = tiles_before + j, st = tile % STAGES;
            if (!mbar_wait_warp(bar(V_FULL + st), (tile / STAGES) & 1, &abort_flag)) return false;
            const int key = key0 + (r & 63);
            if (key > it.p_last || (key < it.k_lo && key >= keep)) {
#pragma unroll
              for (int part = 0; part < Z::PARTS; part += 2) {
                uint4* dst = reinterpret_cast<uint4*>(v_s + st * KV_BYTES + (part + (r >> 6)) * PART_KV + (r & 63) * 128);
#pragma unroll
                for (int ch = 0; ch < 8; ++ch) dst[ch] = make_uint4(0, 0, 0, 0);
              }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          }
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        arrive_if(lane == 0, bar(P_FULL + x));
        return true;
      };
      // tiles that every row of the block sees as a whole: from the last row's first key on, up to the first row's position
      int whole0 = 1, whole1 = 0;  // such tiles behind the first one
      if (my_tiles) {
        const int lo_last = p.window > 0 ? max(0, (x ? it.p_max[1] : it.p_max[0]) - p.window + 1) : 0;
        whole0 = max(1, (max(lo_last, it.k_lo) + BLOCK_N - 1) / BLOCK_N - it.skip - it.j0);
        whole1 = min(my_tiles, (it.base_pos + it.first + x * p.per + 1) / BLOCK_N - it.skip - it.j0);
      }
      for (int j = 0; j < my_tiles && ok; ++j) {
        if (j < whole0 || j >= whole1) {
          ok = step(j, std::true_type());
        } else {
          while (step(j, std::false_type()) && ++j < whole1) {}
          ok = j-- == whole1;
        }
      }
      c += my_tiles, tiles_before += it.num_tiles;
      if (ok && my_tiles) ok = mbar_wait_warp(bar(PV_FULL + x), (c - 1) & 1, &abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      const long at = (long)(it.tok0 + tok) * p.nq + it.kvh * p.group + head, at_slice = at * p.splits + it.slice;
      if (ok && p.splits > 1 && row_ok) {
        const bool seen = sees_tiles(it.j0, it.j0 + my_tiles, it.firsts, it.skip, BLOCK_N, pos, lo, keep);
        *reinterpret_cast<float2*>(p.mid_ml + 2 * at_slice) = make_float2(m_ref == -INFINITY ? MINUS_BIG : fmaxf(m_ref * scale_log2, -3e38f), seen ? l_run : NOTHING_SEEN);
      }
      if (!ok) continue;
      if (!my_tiles) {  // rows without a key: zero (slices are joined to that)
        if (p.splits == 1 && row_ok)
          for (int col = 0; col < p.head_dim; col += 8) *reinterpret_cast<uint4*>(p.out + at * p.head_dim + col) = make_uint4(0, 0, 0, 0);
        continue;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      // Out by way of shared memory, 128 bytes of a row at a time, so that a warp writes whole rows.
      unsigned char* mine = out_s + x * STAGE_OUT + quarter * 32 * 128;
      if (p.splits > 1) {  // as it is, for the kernel that joins the slices
        const unsigned long long dst = row_ok ? reinterpret_cast<unsigned long long>(p.mid_o + at_slice * p.head_dim) : 0;
#pragma unroll 1
        for (int c0 = 0; c0 < p.head_dim; c0 += 32) {
          uint32_t ov[32];
          tmem_load32(o_addr + c0, ov);
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
          for (int ch = 0; ch < 8; ++ch)
            *reinterpret_cast<uint4*>(mine + lane * 128 + 16 * (ch ^ (lane & 7))) = make_uint4(ov[4 * ch], ov[4 * ch + 1], ov[4 * ch + 2], ov[4 * ch + 3]);
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int row = 4 * i + (lane >> 3), piece = lane & 7;
            float* to = reinterpret_cast<float*>(__shfl_sync(0xffffffffu, dst, row));
            if (to && c0 + 4 * piece < p.head_dim) *reinterpret_cast<uint4*>(to + c0 + 4 * piece) = *reinterpret_cast<const uint4*>(mine + row * 128 + 16 * (piece ^ (row & 7)));
          }
          __syncwarp();
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        continue;
      }
      const float inv = 1.f / l_run;
      const uint32_t there = pos >= 0 ? 0xffffffffu : 0u;  // (a token in front of its sequence's first key: zero)
      const unsigned long long dst = row_ok ? reinterpret_cast<unsigned long long>(p.out + at * p.head_dim) : 0;
#pragma unroll 1
      for (int c0 = 0; c0 < p.head_dim; c0 += 64) {
        uint32_t ov[2][32];
        tmem_load32(o_addr + c0, ov[0]);
        tmem_load32(o_addr + c0 + 32, ov[1]);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
        for (int ch = 0; ch < 8; ++ch) {
          uint32_t y[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int i = 8 * (ch & 3) + 2 * e;
            y[e] = pack2(__uint_as_float(ov[ch >> 2][i]) * inv, __uint_as_float(ov[ch >> 2][i + 1]) * inv) & there;
          }
          *reinterpret_cast<uint4*>(mine + lane * 128 + 16 * (ch ^ (lane & 7))) = make_uint4(y[0], y[1], y[2], y[3]);
        }
        __syncwarp();
        const int piece = lane & 7;
        const bool there = c0 + 8 * piece < p.head_dim;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int row = 4 * i + (lane >> 3);
          bf16* to = reinterpret_cast<bf16*>(__shfl_sync(0xffffffffu, dst, row));
          if (to && there) *reinterpret_cast<uint4*>(to + c0 + 8 * piece) = *reinterpret_cast<const uint4*>(mine + row * 128 + 16 * (piece ^ (row & 7)));
        }
        __syncwarp();
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");  // (O read, before the next item's weights are signalled)
    }
  }

  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 12) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
  }
  if (tid == 0 && abort_flag && p.error_word) atomicExch(p.error_word, 2);
}

// Q as [tokens][heads][columns]: boxes of a block's tokens x group heads x 64 columns
bool q_map(CUtensorMap* map, const void* q, int cols, int nq, long num_tokens, long q_stride, int group) {
  Q3EncodeTiledFn fn = q3_encode_tiled();
  if (!fn) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)nq, (cuuint64_t)num_tokens};
  const cuuint64_t strides[2] = {(cuuint64_t)cols * 2, (cuuint64_t)q_stride * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)group, (cuuint32_t)(BLOCK_M / group)};
  const cuuint32_t es[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(q), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// q [num_tokens, *] bfloat16, head h at column h * head_dim.  k, v [tiles][nkv][64][head_dim].  `items` [num_items + 1][2]: the blocks' work in the order in
// which it is taken, as csrc/cache_8bit.cu writes it; the last one's first number is zero, and counts.  out [num_tokens, nq * head_dim]: the rows of the items.
// window > 0: a token sees the last `window` keys up to itself, and the sequence's first `keep_first`.  splits > 1: each item in so many slices, with
// mid_o and mid_ml (PromptSlices) as scratch and the sequences that the items are of.  error_word: set to 2 if a wait expired.
template <bool WIDE>
int launch_tiles(const void* q, int q_stride, int num_tokens, const void* k, const void* v, int tiles, void* items, int num_items, void* out,
                                    int nq, int nkv, int head_dim, float scale, int window, int keep_first, int splits, float* mid_o, float* mid_ml,
                                    const int* cu_seqlens, int num_seqs, int least, int* error_word, cudaStream_t stream) {
  if (num_items < 1 || tiles < 1 || num_tokens < 1) return Q3_OK;
  if (!q || !k || !v || !items || !out || nq < 1 || nkv < 1 || nq % nkv || window < 0 || keep_first < 0 || splits < 1 ||
      (splits > 1 && (!mid_o || !mid_ml || !cu_seqlens || num_seqs < 1 || least < 1)))
    return Q3_ERR_ARGUMENT;
  const int group = nq / nkv;
  if (head_dim < (WIDE ? 129 : 64) || head_dim > (WIDE ? 256 : 128) || head_dim % 16 || group > BLOCK_M || q_stride % 8 || (long)tiles * nkv * BLOCK_N > 0x7fffffffL ||
      nkv > 0xffff || splits > 0x7fff || (long)num_items * nkv * splits > 0x3fffffffL || (long)num_tokens * nq > 0x7fffffffL || (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out | (uintptr_t)items) & 15))
    return Q3_ERR_UNSUPPORTED;
  CUtensorMap tq, tk, tv;
  const long rows = (long)tiles * nkv * BLOCK_N;
  if (!q_map(&tq, q, head_dim, nq, num_tokens, q_stride, group) ||
      !q3_bf16_map(&tk, k, rows, head_dim, head_dim, BLOCK_N, CU_TENSOR_MAP_L2_PROMOTION_L2_128B) ||
      !q3_bf16_map(&tv, v, rows, head_dim, head_dim, BLOCK_N, CU_TENSOR_MAP_L2_PROMOTION_L2_128B))
    return Q3_ERR_LAUNCH;
  static int sms_of[Q3_MAX_DEVICES];
  const int dev = q3_current_device();
  if (!sms_of[dev]) {
    if (cudaFuncSetAttribute(prompts_tiles_kernel<WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, Sizes<WIDE>::SMEM) != cudaSuccess ||
        cudaDeviceGetAttribute(&sms_of[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
      return Q3_ERR_LAUNCH;
  }
  const Params p = {(int4*)items, (bf16*)out, num_items, nq, nkv, group, BLOCK_M / group, (65536 + group - 1) / group, head_dim, window, window > 0 ? keep_first : 0,
                    scale * LOG2_E, error_word, splits, mid_o, mid_ml};
  const int units = num_items * nkv * splits, blocks = units < sms_of[dev] ? units : sms_of[dev];
  cudaError_t err = launch_pdl(prompts_tiles_kernel<WIDE>, dim3(blocks), dim3(THREADS), Sizes<WIDE>::SMEM, stream, tq, tk, tv, p);
  if (err == cudaSuccess && splits > 1) err = merge_prompts({mid_o, mid_ml, (bf16*)out, cu_seqlens, num_seqs, least, num_tokens, nq, head_dim, splits}, stream);
  return err == cudaSuccess ? Q3_OK : Q3_ERR_LAUNCH;
}

}  // namespace
