// Attention of portions of prompts (and of single tokens that the decode kernel does not take) straight over a cache in 8 bits, in bfloat16: any head
// size that is a multiple of 16 up to 256, any group, page size and window, with or without the sequence's first tokens.  (Longer portions of
// heads of 64 and more go to the tcgen05 kernel, unpacked once: an n^2 product of their size is bound by the tensor cores.)
//
// Rows are the (token, head of the group) pairs of a sequence and kv head, token by token; a block takes 128 of them, 16 a warp, and goes through the
// keys in tiles of 64 (32 for heads of more than 128), which all warps share: a thread has its pieces of the next tile's codes on their way in
// registers while the tile before is worked on, turns them to bfloat16 times the page's scale -- exactly: 4 significant bits and a power of two --
// and puts them into the other of two buffers.  Products are mma.sync m16n8k16 with the queries in registers, scores and results in float32; weights
// are rounded to bfloat16 for the product with the values, as in the attention over wide pages.  Where the launch leaves SMs idle, the
// tiles are cut into slices, joined by a second kernel.
//
// What bounds it is mma.sync, which takes an SM's quarter some 27 cycles here for 16 x 8 x 16, and for few rows the chain of a tile.  us, a prompt of 2,048:
// 16 heads over 8 of 64 90 (tcgen05: 35), 32 over 8 of 128 203 (42), 20 over 4 of 80 110 (42), 40 over 2 of 128 213 (64), 16 over 2 of 256 186 (40); 64 tokens
// behind 4,000, 32 over 8 of 128: 37 (28); behind 16,000 91 (52: there the tensor pipe is busy in 0.39 of the clocks, instructions wait for one another).  Slices for more balance than idle SMs ask for, four blocks an SM: 84 for 89 with heads
// of 64, 230 for 192 with 256.
#include "eight_bit.cuh"
#include "mma_tiles.cuh"
#include "prompt_slices.cuh"

namespace {

constexpr int WARPS = 8, THREADS = 32 * WARPS, ROWS = 16 * WARPS;

__device__ __forceinline__ float exp2_fast(float x) {  // 2^x to 2 units in the last place; below 2^-126 zero
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct Prompts {
  const bf16* q;
  int q_stride;
  const unsigned char* pages;
  int num_pages;
  const int *block_table, *kv_lens, *cu_seqlens;
  int max_pages, num_seqs;
  bf16* out;
  float *mid_o, *mid_ml;  // splits > 1: see PromptSlices
  int splits, items, least, nq, nkv, D, ps, shift, window, keep_first, max_len;  // shift: log2 of the page size, or -1
  float scale_log2;
};

template <int KD> struct Sizes {  // KD: head size in steps of 16 channels, rounded up to one that has been compiled
  static constexpr int KEYS = KD <= 8 ? 64 : 32;                         // of a tile
  static constexpr int PITCH = 32 * KD + 16;                             // bytes of a row in shared memory: eight rows meet eight different banks
  static constexpr int BUFFER = 2 * KEYS * PITCH;                        // keys, then values
  static constexpr int SMEM = 2 * BUFFER;
  static constexpr int MINE = (KEYS * KD + THREADS - 1) / THREADS;       // pieces of a tile's keys (and as many of its values) that a thread brings
};

template <int KD> __global__ void __launch_bounds__(THREADS, KD <= 4 ? 2 : 1) prompts_8bit_kernel(Prompts a) {
  typedef Sizes<KD> Z;
  constexpr int KEYS = Z::KEYS, PITCH = Z::PITCH, MINE = Z::MINE;
  extern __shared__ __align__(128) unsigned char smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, kvh = blockIdx.y, G = a.nq / a.nkv, D = a.D;
  pdl_wait();
  pdl_launch_dependents();
  // the item's sequence and rows (late rows of long prompts, which have the most keys, first)
  int seq = -1, row0 = 0;
  for (int base = 0, item = a.items - 1 - (int)blockIdx.x; base < a.num_seqs && seq < 0; base += 32) {
    int n = 0;
    if (base + lane < a.num_seqs) {
      const int tokens = a.cu_seqlens[base + lane + 1] - a.cu_seqlens[base + lane];
      if (tokens >= a.least) n = (tokens * G + ROWS - 1) / ROWS;
    }
    int sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += y;
    }
    const uint32_t reach = __ballot_sync(0xffffffffu, sum > item);
    if (reach) {
      const int from = __ffs(reach) - 1;
      seq = base + from;
      row0 = (item - (__shfl_sync(0xffffffffu, sum, from) - __shfl_sync(0xffffffffu, n, from))) * ROWS;
    } else {
      item -= __shfl_sync(0xffffffffu, sum, 31);
    }
  }
  if (seq < 0) return;
  const int tok0 = a.cu_seqlens[seq], news = a.cu_seqlens[seq + 1] - tok0, kv_len = min(a.kv_lens[seq], a.max_len);
  const int rows = news * G, before = kv_len - news;  // (before < 0: rows without keys are zero)
  const int* bt = a.block_table + (long)seq * a.max_pages;
  // what the block's rows see: keys k_lo .. p_last, and those in front of keep
  const int p_last = before + (min(rows, row0 + ROWS) - 1) / G;
  const int k_lo = a.window > 0 ? max(0, before + row0 / G - a.window + 1) : 0, keep = a.window > 0 ? a.keep_first : 0;
  const int tile0 = k_lo / KEYS, firsts = min((keep + KEYS - 1) / KEYS, tile0), skip = tile0 - firsts;
  const int all = p_last >= 0 ? p_last / KEYS + 1 - skip : 0, per = (all + a.splits - 1) / a.splits;
  const int j0 = blockIdx.z * per, j1 = min(all, j0 + per);  // this slice's tiles, of those that count
  auto base_of = [&](int j) { return (j + (j >= firsts ? skip : 0)) * KEYS; };

  // ---- the next tiles, on their way: pieces of keys' and values' codes with their page's scales, and the pages of the tile behind them
  int page[MINE];
  uint4 kc[MINE], vc[MINE];
  float2 scale[MINE];
  const Q8Page L(D, a.ps);
  const int mask = q8_mask(D);
  auto find = [&](int j) {
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
      const int key = base_of(j) + (tid + THREADS * i) / KD;
      const bool seen = j < j1 && key <= p_last && (key >= k_lo || key < keep);
      page[i] = seen ? bt[a.shift >= 0 ? key >> a.shift : key / a.ps] : -1;
    }
  };
  auto fetch = [&](int j) {
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
      const int item = tid + THREADS * i, key = base_of(j) + item / KD, piece = item % KD;
      kc[i] = vc[i] = make_uint4(0, 0, 0, 0);
      scale[i] = make_float2(0.f, 0.f);
      if ((uint32_t)page[i] < (uint32_t)a.num_pages && item < KEYS * KD && 16 * piece < D) {
        const int row = a.shift >= 0 ? key & (a.ps - 1) : key - key / a.ps * a.ps;
        const unsigned char* rec = a.pages + ((long)page[i] * a.nkv + kvh) * L.record;
        const unsigned char* from = rec + (long)row * D + 16 * (piece ^ (row & mask));
        kc[i] = *reinterpret_cast<const uint4*>(from);
        vc[i] = *reinterpret_cast<const uint4*>(from + L.values);
        scale[i] = *reinterpret_cast<const float2*>(rec + L.scales);
      }
    }
  };
  auto widen = [](const uint4& w, float s, unsigned char* to) {
    const uint32_t word[4] = {w.x, w.y, w.z, w.w};
    uint32_t y[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float v[4];
      q8_floats(word[e], v);
      y[2 * e] = pack_bf16(v[0] * s, v[1] * s), y[2 * e + 1] = pack_bf16(v[2] * s, v[3] * s);
    }
    *reinterpret_cast<uint4*>(to) = make_uint4(y[0], y[1], y[2], y[3]);
    *reinterpret_cast<uint4*>(to + 16) = make_uint4(y[4], y[5], y[6], y[7]);
  };
  auto convert = [&](unsigned char* buffer) {
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
      const int item = tid + THREADS * i;
      if (item >= KEYS * KD) break;
      unsigned char* to = buffer + item / KD * PITCH + 32 * (item % KD);
      widen(kc[i], scale[i].x, to);
      widen(vc[i], scale[i].y, to + KEYS * PITCH);
    }
  };
  find(j0);
  fetch(j0);
  find(j0 + 1);
  // ---- the queries, through shared memory into operands
  for (int i = tid; i < ROWS * 2 * KD; i += THREADS) {
    const int r = i / (2 * KD), c = i - r * 2 * KD, row = row0 + r;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (row < rows && 8 * c < D) v = *reinterpret_cast<const uint4*>(a.q + (long)(tok0 + row / G) * a.q_stride + (long)(kvh * G + row % G) * D + 8 * c);
    *reinterpret_cast<uint4*>(smem + r * PITCH + 16 * c) = v;
  }
  __syncthreads();
  uint32_t q[KD][4];
#pragma unroll
  for (int k = 0; k < KD; ++k) ldmatrix_x4(q[k], smem_u32(smem + (16 * warp + (lane & 15)) * PITCH + 32 * k + 16 * (lane >> 4)));
  __syncthreads();
  convert(smem);
  fetch(j0 + 1);
  find(j0 + 2);
  __syncthreads();

  // this lane's rows: lane / 4 and + 8 of the warp's 16; the last key that each sees (-1: it is none) and the first of its window
  int pos[2], lo[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int row = row0 + 16 * warp + (lane >> 2) + 8 * h;
    pos[h] = row < rows ? before + row / G : -1;
    lo[h] = a.window > 0 ? max(0, pos[h] - a.window + 1) : 0;
  }
  const int w_first = row0 + 16 * warp, w_last = min(rows, w_first + 16) - 1;                       // the warp's rows
  const int pos_min = before + w_first / G, pos_max = w_first < rows ? before + w_last / G : -1;    // what all of them see, what any of them sees
  const int lo_min = a.window > 0 ? max(0, pos_min - a.window + 1) : 0, lo_max = a.window > 0 ? max(0, pos_max - a.window + 1) : 0;
  float o[2 * KD][4], m[2] = {MINUS_BIG, MINUS_BIG}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int c = 0; c < 2 * KD; ++c) o[c][0] = o[c][1] = o[c][2] = o[c][3] = 0.f;
  for (int j = j0; j < j1; ++j) {
    const unsigned char* ks = smem + ((j - j0) & 1) * Z::BUFFER;
    const unsigned char* vs = ks + KEYS * PITCH;
    const int key0 = base_of(j);
    if (key0 <= pos_max && (key0 + KEYS > lo_min || key0 < keep)) {
      float s[KEYS / 8][4];
#pragma unroll
      for (int n = 0; n < KEYS / 8; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
      for (int k = 0; k < KD; ++k)
#pragma unroll
        for (int n = 0; n < KEYS / 8; n += 2) {
          uint32_t b[4];
          ldmatrix_x4(b, smem_u32(ks + (8 * n + (lane & 7) + (lane >> 4 << 3)) * PITCH + 32 * k + 16 * (lane >> 3 & 1)));
          mma_bf16(s[n], q[k], b[0], b[1]);
          mma_bf16(s[n + 1], q[k], b[2], b[3]);
        }
      const bool whole = key0 + KEYS - 1 <= pos_min && (key0 >= lo_max || key0 + KEYS <= keep);  // (of one mind over the warp)
      float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int n = 0; n < KEYS / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[n][e] *= a.scale_log2;
          if (!whole) {
            const int key = key0 + 8 * n + 2 * (lane & 3) + (e & 1), h = e >> 1;
            if (key > pos[h] || (key < lo[h] && key >= keep)) s[n][e] = -INFINITY;
          }
          top[e >> 1] = fmaxf(top[e >> 1], s[n][e]);
        }
      float f[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
        top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
        // (the maximum moves only when it would be passed by a factor of 2^8: hardly ever after the first tiles)
        const float now = top[h] > m[h] + 8.f ? top[h] : m[h];
        f[h] = exp2_fast(m[h] - now);
        m[h] = now;
      }
      if (__any_sync(0xffffffffu, f[0] != 1.f || f[1] != 1.f)) {
        l[0] *= f[0], l[1] *= f[1];
#pragma unroll
        for (int c = 0; c < 2 * KD; ++c) o[c][0] *= f[0], o[c][1] *= f[0], o[c][2] *= f[1], o[c][3] *= f[1];
      }
#pragma unroll
      for (int n = 0; n < KEYS / 8; ++n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = exp2_fast(s[n][e] - m[e >> 1]);
        l[0] += s[n][0] + s[n][1];
        l[1] += s[n][2] + s[n][3];
      }
#pragma unroll
      for (int k = 0; k < KEYS / 16; ++k) {
        const uint32_t p[4] = {pack_bf16(s[2 * k][0], s[2 * k][1]), pack_bf16(s[2 * k][2], s[2 * k][3]), pack_bf16(s[2 * k + 1][0], s[2 * k + 1][1]),
                               pack_bf16(s[2 * k + 1][2], s[2 * k + 1][3])};
#pragma unroll
        for (int c = 0; c < 2 * KD; c += 2) {
          uint32_t b[4];
          ldmatrix_x4_trans(b, smem_u32(vs + (16 * k + (lane & 15)) * PITCH + 16 * (c + (lane >> 4))));
          mma_bf16(o[c], p, b[0], b[1]);
          mma_bf16(o[c + 1], p, b[2], b[3]);
        }
      }
    }
    if (j + 1 < j1) {
      convert(smem + ((j + 1 - j0) & 1) * Z::BUFFER);
      fetch(j + 2);
      find(j + 3);
      __syncthreads();
    }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    const int row = row0 + 16 * warp + (lane >> 2) + 8 * h;
    if (row >= rows) continue;
    const long at = (long)(tok0 + row / G) * a.nq + kvh * G + row % G;
    if (a.splits > 1) {
      float* to = a.mid_o + (at * a.splits + blockIdx.z) * D;
      const bool seen = sees_tiles(j0, j1, firsts, skip, KEYS, pos[h], lo[h], keep);
      if ((lane & 3) == 0) *reinterpret_cast<float2*>(a.mid_ml + 2 * (at * a.splits + blockIdx.z)) = make_float2(m[h], seen ? l[h] : NOTHING_SEEN);
      if (!seen) continue;
#pragma unroll
      for (int c = 0; c < 2 * KD; ++c)
        if (8 * c < D) *reinterpret_cast<float2*>(to + 8 * c + 2 * (lane & 3)) = make_float2(o[c][2 * h], o[c][2 * h + 1]);
    } else {
      bf16* to = a.out + at * D;
      const float inv = 1.f / l[h];
      const uint32_t there = pos[h] >= 0 ? 0xffffffffu : 0u;  // (a token without a key: zero)
#pragma unroll
      for (int c = 0; c < 2 * KD; ++c)
        if (8 * c < D) *reinterpret_cast<uint32_t*>(to + 8 * c + 2 * (lane & 3)) = pack_bf16(o[c][2 * h] * inv, o[c][2 * h + 1] * inv) & there;
    }
  }
}

template <int KD> int launch_prompts(const Prompts& a, int tokens, cudaStream_t stream) {
  static bool once[Q3_MAX_DEVICES];
  const int dev = q3_current_device();
  if (!once[dev]) {
    if (cudaFuncSetAttribute(prompts_8bit_kernel<KD>, cudaFuncAttributeMaxDynamicSharedMemorySize, Sizes<KD>::SMEM) != cudaSuccess) return Q3_ERR_LAUNCH;
    once[dev] = true;
  }
  cudaError_t err = launch_pdl(prompts_8bit_kernel<KD>, dim3(a.items, a.nkv, a.splits), dim3(THREADS), Sizes<KD>::SMEM, stream, a);
  if (err == cudaSuccess && a.splits > 1)
    err = merge_prompts({a.mid_o, a.mid_ml, a.out, a.cu_seqlens, a.num_seqs, a.least, tokens, a.nq, a.D, a.splits}, stream);
  return err == cudaSuccess ? Q3_OK : Q3_ERR_LAUNCH;
}

}  // namespace

// q [tokens, *]: head h at column h * D.  out [tokens, nq * D]: the rows of sequences that bring fewer than `least` tokens are left as they are.  `items`: sum
// over the others of ceil(tokens * (nq / nkv) / 128).  splits > 1: mid_o [tokens][nq][splits][D] and mid_ml [tokens][nq][splits][2] are scratch.
Q3_EXPORT int q3_prompts_attention_8bit(const void* q, int q_stride, const void* pages, int num_pages, const int* block_table, int max_pages,
                                        const int* kv_lens, const int* cu_seqlens, void* out, float* mid_o, float* mid_ml, int splits, int items,
                                        int least, int tokens, int num_seqs, int nq, int nkv, int D, int ps, float scale, int window, int keep_first,
                                        int max_len, cudaStream_t stream) {
  if (num_seqs < 1 || items < 1 || tokens < 1) return Q3_OK;
  if (!q || !pages || !block_table || !kv_lens || !cu_seqlens || !out || nq < 1 || nkv < 1 || nq % nkv || !q8_sizes_ok(D, ps) || splits < 1 || least < 1 ||
      (splits > 1 && (!mid_o || !mid_ml)) || window < 0 || keep_first < 0 || max_len > (long)max_pages * ps)
    return Q3_ERR_ARGUMENT;
  if (q_stride % 8 || (reinterpret_cast<uintptr_t>(q) & 15) || (reinterpret_cast<uintptr_t>(pages) & 15) || (reinterpret_cast<uintptr_t>(out) & 3) ||
      nkv > 65535 || splits > 65535 || (long)tokens * nq > 0x7fffffffL || (long)window + keep_first > 0x7ffffff0L)
    return Q3_ERR_UNSUPPORTED;
  int shift = 0;
  while ((1 << shift) < ps) ++shift;
  const Prompts a{(const bf16*)q, q_stride, (const unsigned char*)pages, num_pages, block_table, kv_lens, cu_seqlens, max_pages, num_seqs, (bf16*)out,
                  mid_o, mid_ml, splits, items, least, nq, nkv, D, ps, (1 << shift) == ps ? shift : -1, window, keep_first, max_len, scale * LOG2_E};
  const int steps = D / 16;
  if (steps <= 2) return launch_prompts<2>(a, tokens, stream);
  if (steps <= 4) return launch_prompts<4>(a, tokens, stream);
  if (steps <= 5) return launch_prompts<5>(a, tokens, stream);
  if (steps <= 6) return launch_prompts<6>(a, tokens, stream);
  if (steps <= 8) return launch_prompts<8>(a, tokens, stream);
  if (steps <= 12) return launch_prompts<12>(a, tokens, stream);
  return launch_prompts<16>(a, tokens, stream);
}
