// The cache in 8 bits (layout and rounding: eight_bit.cuh): what writes it and what reads it back.
//
// * store:  per-head q/k RMSNorm, rotation, and the write of keys and values in 8 bits.
// * unpack: a step's sequences as pages of bfloat16 or float32, one after the other, for the attention over prompts.
#include <type_traits>

#include "eight_bit.cuh"
#include "rotary.cuh"

#define Q3_ERR_POSITION 16

namespace {

constexpr int STORE_THREADS = 512;  // of a block, at most

struct Store {
  const float *q_w, *k_w, *cos_t, *sin_t;
  float eps;
  int rot_half, max_pos, pairing;
  const int *positions, *kv_lens, *cu_seqlens, *block_table;
  int max_pages, num_pages, num_seqs, num_tokens, ps;
  int units;    // pages that get tokens, at most; 0: none are written
  int q_blocks;  // blocks that a token's queries take
  unsigned char* pages;
  int* error_word;
};

// A unit of the write: one page of one sequence, and the rows r0 .. r1 - 1 of it that the step brings; a sequence's new tokens are the last of
// its kv_lens places.  Everything that shares a scale is in one block's hands.  Called by whole warps.
struct Unit {
  int r0, r1, token;    // token: of row 0 (as if it were new as well)
  unsigned char* rec;   // null: nothing to write
  // `single`: every sequence brings one token, unit u is sequence u's
  __device__ __forceinline__ Unit(const Store& a, bool single, int u, int nkv, int kvh, long record) : r0(0), r1(0), token(0), rec(nullptr) {
    const int lane = threadIdx.x & 31;
    int seq = -1, i = 0, first = 0, len = 0, news = 0, cu = 0;
    if (single) {
      seq = u, len = a.kv_lens[u], cu = a.cu_seqlens[u], news = a.cu_seqlens[u + 1] - cu;
      first = max(0, len - news), i = first / a.ps;
      if (news < 1 || len < 1) return;
    } else {
      for (int base = 0; base < a.num_seqs && seq < 0; base += 32) {
        int n = 0, l = 0, c = 0, w = 0;
        if (base + lane < a.num_seqs) {
          l = a.kv_lens[base + lane], c = a.cu_seqlens[base + lane], w = a.cu_seqlens[base + lane + 1] - c;
          if (w > 0 && l > 0) n = (l - 1) / a.ps - max(0, l - w) / a.ps + 1;
        }
        int sum = n;  // pages up to and with this lane's sequence
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, sum, o);
          if (lane >= o) sum += y;
        }
        const uint32_t reach = __ballot_sync(0xffffffffu, sum > u);
        if (reach) {
          const int from = __ffs(reach) - 1;
          seq = base + from;
          len = __shfl_sync(0xffffffffu, l, from), cu = __shfl_sync(0xffffffffu, c, from), news = __shfl_sync(0xffffffffu, w, from);
          first = max(0, len - news);
          i = first / a.ps + u - (__shfl_sync(0xffffffffu, sum, from) - __shfl_sync(0xffffffffu, n, from));
        } else {
          u -= __shfl_sync(0xffffffffu, sum, 31);
        }
      }
      if (seq < 0) return;
    }
    if (i >= a.max_pages) return;
    const int page = a.block_table[(long)seq * a.max_pages + i];
    if (page < 0 || page >= a.num_pages) return;
    const int begin = i * a.ps;
    r0 = max(first - begin, 0), r1 = min(len - begin, a.ps);
    token = cu + begin - (len - news);
    rec = a.pages + ((long)page * nkv + kvh) * record;
  }
};

// The step from the rows' largest number to the scale: rows in front of r0 were there before, and are cut to a scale that grows.  The exponent
// of the scale; `codes`: the keys' or values' of the record.  By the whole block; `red`: 32 words.
__device__ __forceinline__ int settle_scale(uint32_t most, int r0, int D, unsigned char* codes, float* scale, uint32_t* red) {
  const float held = r0 > 0 ? *scale : 0.f;
  most = __reduce_max_sync(0xffffffffu, most);
  if (blockDim.x > 32) {
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = most;
    __syncthreads();
    for (int w = 0; w < (blockDim.x >> 5); ++w) most = max(most, red[w]);
  }
  __syncwarp();
  int e = q8_exponent(most);
  if (r0 > 0) {
    const int old = q8_exponent_of(held);
    if (e > old) {
      const float shrink = e - old > 120 ? 0.f : q8_power(old - e);
      for (uint32_t at = 16 * threadIdx.x; at < (uint32_t)(r0 * D); at += 16 * blockDim.x) {  // (a page's codes may end just in front of 2^31)
        uint4 w = *reinterpret_cast<const uint4*>(codes + at);
        w.x = q8_rescaled(w.x, shrink), w.y = q8_rescaled(w.y, shrink), w.z = q8_rescaled(w.z, shrink), w.w = q8_rescaled(w.w, shrink);
        *reinterpret_cast<uint4*>(codes + at) = w;
      }
    } else {
      e = old;
    }
  }
  if (threadIdx.x == 0) *scale = q8_power(e);
  return e;
}

// Norm (w: the weights, or null) and rotation of one thread's share of a head (rotary.cuh); false: the position lies outside the tables.
// Called by whole warps.  For the order of operations see rotary.cuh; heads of 16, 32 and 64 add fused squares.
__device__ __forceinline__ bool norm_and_turn(float (&v0)[8], float (&v1)[8], const Store& a, const float* w, int p, int c, int D) {
  const int half = D / 2, tph = D / 16;
  if (w) {
    float ss;
    if (D >= 128) {
      float even = __fadd_rn(quad_of_squares(v0), quad_of_squares(v1)), odd = __fadd_rn(quad_of_squares(v0 + 4), quad_of_squares(v1 + 4));
#pragma unroll
      for (int o = tph >> 1; o > 0; o >>= 1) {
        even = __fadd_rn(even, __shfl_xor_sync(0xffffffffu, even, o));
        odd = __fadd_rn(odd, __shfl_xor_sync(0xffffffffu, odd, o));
      }
      ss = __fadd_rn(even, odd);
    } else {
      ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss += v0[e] * v0[e] + v1[e] * v1[e];
      for (int o = tph >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    }
    const float rstd = rsqrtf(ss / (float)D + a.eps);
    float wa[8], wb[8];
    load8(w + 8 * c, wa);
    load8(w + half + 8 * c, wb);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v0[e] = (v0[e] * rstd) * wa[e];
      v1[e] = (v1[e] * rstd) * wb[e];
    }
  }
  if (!a.cos_t) return true;
  if (p < 0 || p >= a.max_pos) return false;
  const Angles y = load_angles(a.cos_t + (long)p * half, a.sin_t + (long)p * half, c, half, a.pairing);
  if (!a.pairing) {
#pragma unroll
    for (int e = 0; e < 8; ++e) turn_rounded(v0[e], v1[e], y.cs[e], y.sn[e]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      turn_rounded(v0[2 * j], v0[2 * j + 1], y.cs[j], y.sn[j]);
      turn_rounded(v1[2 * j], v1[2 * j + 1], y.cs[4 + j], y.sn[4 + j]);
    }
  }
  return true;
}

// Head sizes 16, 32, 64, 128, 256 with the rotation over the whole head (or none): D / 16 threads per (token, head); thread c owns
// channels [8c, 8c + 8) and [D/2 + 8c, D/2 + 8c + 8).  Blocks of the write come first (unit, then key and value heads), each as many rows at a
// time as it has threads for; rows beyond that are made once more when the scale is known.  Then the queries' blocks.
// KNOWN: the head size where the compiler knows it, else 0.  SINGLE: every sequence brings one token.
// The floor is the bytes of the projection and of the queries.  What bounds it is latency, loads one behind the other (a position, its angles), and
// instructions: 3,258 tokens of 32 + 8 heads of 128 in bfloat16 take 21 us (3.5 TB/s), 14 of them the queries; 40 registers a thread, 48 warps an SM, are
// worth two spilled ones (with 56: 23 us, with 32: 26).  Every value rounded by itself, without the hardware's conversion: 27.  Several tokens in
// turn by a thread that keeps the weights and has the next one's values on their way, 80 registers: 27.
template <typename T, int KNOWN, bool SINGLE>
__global__ void __launch_bounds__(STORE_THREADS, SINGLE ? 2 : 3) store_8bit_vec_kernel(const T* qkv, int row_stride, T* q_out, int q_stride, int nq, int nkv, int size, Store a) {
  const int D = KNOWN ? KNOWN : size, tph = D / 16, tph_shift = 31 - __clz(tph), half = D / 2, mask = q8_mask(D);
  const int tid = threadIdx.x, c = tid & (tph - 1);
  __shared__ uint32_t red[32];
  pdl_wait();
  pdl_launch_dependents();
  const int write_blocks = a.units * 2 * nkv;
  if ((int)blockIdx.x >= write_blocks) {  // queries
    const int b = blockIdx.x - write_blocks, t = b / a.q_blocks;
    const int hi = ((b - t * a.q_blocks) * blockDim.x + tid) >> tph_shift;
    const bool live = hi < nq;
    float v0[8] = {}, v1[8] = {};
    const int p = a.positions[t];
    if (live) {
      const T* x = qkv + (long)t * row_stride + (long)hi * D;
      load8(x + 8 * c, v0);
      load8(x + half + 8 * c, v1);
    }
    const bool turned = norm_and_turn(v0, v1, a, a.q_w, p, c, D);
    if (!live) return;
    if (!turned) {
      if (a.error_word && c == 0) atomicExch(a.error_word, Q3_ERR_POSITION);
      return;
    }
    T* y = q_out + (long)t * q_stride + (long)hi * D;
    store8(y + 8 * c, v0);
    store8(y + half + 8 * c, v1);
    return;
  }
  const int u = blockIdx.x / (2 * nkv), hd = blockIdx.x - u * 2 * nkv, is_v = hd >= nkv, kvh = hd - is_v * nkv;
  const Q8Page L(D, a.ps);
  const Unit unit(a, SINGLE, u, nkv, kvh, L.record);
  if (!unit.rec) return;
  unsigned char* codes = unit.rec + (is_v ? L.values : 0);
  const int per = blockDim.x >> tph_shift, r_first = unit.r0 + (tid >> tph_shift);
  const T* x0 = qkv + (long)(nq + hd) * D;
  float v0[8], v1[8];
  bool live;
  auto make = [&](int row) {
    const int t = unit.token + row;
    live = row < unit.r1 && (tid >> tph_shift) < per && (uint32_t)t < (uint32_t)a.num_tokens;
#pragma unroll
    for (int e = 0; e < 8; ++e) v0[e] = v1[e] = 0.f;
    int p = 0;
    if (live) {
      const T* x = x0 + (long)t * row_stride;
      load8(x + 8 * c, v0);
      load8(x + half + 8 * c, v1);
      p = a.positions[t];
    }
    if (is_v) return;
    if (!norm_and_turn(v0, v1, a, a.k_w, p, c, D) && live) {
      if (a.error_word && c == 0) atomicExch(a.error_word, Q3_ERR_POSITION);
      live = false;
    }
  };
  uint32_t most = 0;
  const int passes = (unit.r1 - unit.r0 + per - 1) / per;
  for (int pass = 0; pass < passes; ++pass) {
    make(r_first + pass * per);
    if (live) most = max(most, max(q8_most(v0), q8_most(v1)));
  }
  const int e = settle_scale(most, unit.r0, D, codes, reinterpret_cast<float*>(unit.rec + L.scales) + is_v, red);
  const float down = q8_power(-e);
  for (int pass = 0; pass < passes; ++pass) {
    const int row = r_first + pass * per;
    if (passes > 1) make(row);
    if (!live) continue;
    unsigned char* to = codes + (long)row * D;
    *reinterpret_cast<uint2*>(to + q8_at(8 * c, row, mask)) = q8_words(v0, down);
    *reinterpret_cast<uint2*>(to + q8_at(half + 8 * c, row, mask)) = q8_words(v1, down);
  }
}

// Any other size, rotation or alignment: a warp per (token, head) of the queries, a block per (unit, head) of the write, its rows a warp each.
template <typename T>
__global__ void __launch_bounds__(STORE_THREADS) store_8bit_kernel(const T* qkv, int row_stride, T* q_out, int q_stride, int nq, int nkv, int D, Store a) {
  extern __shared__ float stage[];  // warps * 2 * D
  __shared__ uint32_t red[32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  float *xs = stage + warp * 2 * D, *ys = xs + D;
  // ys gets the head that x names; false: its position lies outside the tables
  auto make = [&](const T* x, const float* w, int p, bool turn) {
    float ss = 0.f;
    __syncwarp();
    for (int d = lane; d < D; d += 32) {
      const float v = to_f32(x[d]);
      xs[d] = v;
      ss += v * v;
    }
    const float rstd = w ? rsqrtf(warp_sum(ss) / (float)D + a.eps) : 1.f;
    __syncwarp();
    turn = turn && a.cos_t;
    if (turn && (p < 0 || p >= a.max_pos)) {
      if (a.error_word && lane == 0) atomicExch(a.error_word, Q3_ERR_POSITION);
      return false;
    }
    const float *cs = turn ? a.cos_t + (long)p * a.rot_half : nullptr, *sn = turn ? a.sin_t + (long)p * a.rot_half : nullptr;
    for (int d = lane; d < D; d += 32) {
      float y = w ? (xs[d] * rstd) * w[d] : xs[d];
      if (cs && d < 2 * a.rot_half) {
        const bool first = a.pairing ? (d & 1) == 0 : d < a.rot_half;
        const int i = a.pairing ? d >> 1 : (first ? d : d - a.rot_half);
        const int pd = a.pairing ? d ^ 1 : (first ? d + a.rot_half : d - a.rot_half);
        const float yp = w ? (xs[pd] * rstd) * w[pd] : xs[pd];
        y = first ? y * cs[i] - yp * sn[i] : y * cs[i] + yp * sn[i];
      }
      ys[d] = y;
    }
    __syncwarp();
    return true;
  };
  const int write_blocks = a.units * 2 * nkv;
  if ((int)blockIdx.x >= write_blocks) {
    const long item = (long)(blockIdx.x - write_blocks) * warps + warp;
    if (item >= (long)a.num_tokens * nq) return;
    const int t = (int)(item / nq), hi = (int)(item - (long)t * nq);
    if (!make(qkv + (long)t * row_stride + (long)hi * D, a.q_w, a.positions[t], true)) return;
    T* y = q_out + (long)t * q_stride + (long)hi * D;
    for (int d = lane; d < D; d += 32) y[d] = from_f32<T>(ys[d]);
    return;
  }
  const int u = blockIdx.x / (2 * nkv), hd = blockIdx.x - u * 2 * nkv, is_v = hd >= nkv, kvh = hd - is_v * nkv;
  const Q8Page L(D, a.ps);
  const Unit unit(a, false, u, nkv, kvh, L.record);
  if (!unit.rec) return;
  unsigned char* codes = unit.rec + (is_v ? L.values : 0);
  auto make_row = [&](int row) {
    const int t = unit.token + row;
    return (uint32_t)t < (uint32_t)a.num_tokens &&
           make(qkv + (long)t * row_stride + (long)(nq + hd) * D, is_v ? nullptr : a.k_w, a.positions[t], !is_v);
  };
  uint32_t most = 0;
  for (int row = unit.r0 + warp; row < unit.r1; row += warps)
    if (make_row(row))
      for (int d = lane; d < D; d += 32) most = max(most, q8_finite(q8_rounded(ys[d])));
  const int e = settle_scale(most, unit.r0, D, codes, reinterpret_cast<float*>(unit.rec + L.scales) + is_v, red);
  const float down = q8_power(-e);
  const int mask = q8_mask(D);
  for (int row = unit.r0 + warp; row < unit.r1; row += warps)
    if (make_row(row))
      for (int d = 4 * lane; d < D; d += 128) *reinterpret_cast<uint32_t*>(codes + (long)row * D + q8_at(d, row, mask)) = q8_word(ys + d, down);
}

// ---- back to wide pages -------------------------------------------------------------------------------------------------------------
// Two forms.  Without `cu_seqlens`, sequence z's page i goes to page z * width + i, rows behind its last token are zero, and whole pages behind
// it too.  With it, the attention over prompts reads the pages: only sequences that bring at least `least` tokens count, and of each only the
// pages that a new token sees (with a window those of the first `keep_first` tokens, and those from the first that the first new token's window
// reaches); they lie one after the other, `count` tiles of 64 tokens, in which rows behind a sequence's last token are left as they are.  Warps of their own
// write what that attention works through: `items`, of `item_tokens` tokens of a sequence each.
struct Unpack {
  const unsigned char* pages;
  int num_pages, nkv, ps;
  const int *block_table, *kv_lens, *cu_seqlens;
  int max_pages, num_seqs, max_len, least, window, keep_first, count, width;
  int item_tokens, num_items;
  int4* items;  // [num_items + 1][2], see write_item
};
constexpr int TILE = 64;  // tokens

// What sequence s brings: tokens (0: it does not count), length, and its tiles that are written: 0 .. kept - 1 and skip, skip + 1 ..
struct UnpackSequence {
  int tokens = 0, len = 0, kept = 0, skip = 0, tiles = 0;
  __device__ __forceinline__ UnpackSequence(const Unpack& a, int s) {
    if (s >= a.num_seqs) return;
    const int news = a.cu_seqlens[s + 1] - a.cu_seqlens[s];
    len = min(a.kv_lens[s], a.max_len);
    if (news < a.least) return;
    tokens = news;
    if (len <= 0) return;
    if (a.window > 0) skip = max(0, len - tokens - a.window + 1) / TILE;
    kept = min(skip, (a.keep_first + TILE - 1) / TILE);
    tiles = (len + TILE - 1) / TILE - skip + kept;
  }
};
__device__ __forceinline__ int warp_prefix(int n) {  // the sum up to and with this lane's
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, n, o);
    if ((threadIdx.x & 31) >= o) n += y;
  }
  return n;
}

// Item `w` of the attention, as {place in its sequence, the sequence's first token, its tokens, its length}, {its first tile that is written, kept, skip}; place
// -1: none.  The number behind the last item is zero: blocks of the attention count on it.  Items stand by how many keys they see, in units of a tile, the heaviest first, so that the last ones that are
// taken are short: 1,500, 701 and 1,000 (behind 2,048) tokens 79 us with their unpacking, in the order of the sequences 80, from the last 86; under a window
// 59 for 62 and 70.  An item's place follows from how many of each sequence see more, which is a division, as they grow evenly.  By a warp.
__device__ __forceinline__ void write_item(const Unpack& a, int w) {
  const int lane = threadIdx.x & 31, T = a.item_tokens;
  const int most = a.window > 0 ? a.window + a.keep_first + T : 0x7fffffff;  // keys that an item sees, roughly
  int seq = -1, i = 0, before = 0, tiles_before = 0;
  int4 what = make_int4(-1, 0, 0, 0), where = make_int4(0, 0, 0, 0);
  for (int base = 0, left = w; base < a.num_seqs && seq < 0; base += 32) {
    const UnpackSequence s(a, base + lane);
    const int n = (s.tokens + T - 1) / T, sum = warp_prefix(n), tile_sum = warp_prefix(s.tiles);
    const uint32_t reach = __ballot_sync(0xffffffffu, sum > left);
    if (reach) {
      const int from = __ffs(reach) - 1;
      seq = base + from;
      i = left - __shfl_sync(0xffffffffu, sum - n, from);
      what = make_int4(i, a.cu_seqlens[seq], __shfl_sync(0xffffffffu, s.tokens, from), __shfl_sync(0xffffffffu, s.len, from));
      where = make_int4(tiles_before + __shfl_sync(0xffffffffu, tile_sum - s.tiles, from), __shfl_sync(0xffffffffu, s.kept, from),
                        __shfl_sync(0xffffffffu, s.skip, from), 0);
    } else {
      left -= __shfl_sync(0xffffffffu, sum, 31);
      tiles_before += __shfl_sync(0xffffffffu, tile_sum, 31);
    }
  }
  int at = w;  // (places behind the last item say so)
  if (seq >= 0) {
    const int tiles = min(max(0, what.w - what.z) + (i + 1) * T, most) >> 6;
    for (int base = 0; base < a.num_seqs; base += 32) {
      const UnpackSequence s(a, base + lane);
      const int n = (s.tokens + T - 1) / T, first = max(0, s.len - s.tokens);
      auto items_of = [&](int t) {  // how many of this sequence's see at least t tiles: the last ones
        return t > most >> 6 ? 0 : n - min(n, max(0, (max(0, 64 * t - first) + T - 1) / T - 1));
      };
      const int more = items_of(tiles + 1);
      before += more + (base + lane < seq ? items_of(tiles) - more : 0) + (base + lane == seq ? n - more - 1 - i : 0);
    }
    at = __reduce_add_sync(0xffffffffu, before);
  }
  if (lane == 0 && at < a.num_items) a.items[2 * at] = what, a.items[2 * at + 1] = where;
  if (lane == 0 && w == 0) a.items[2 * a.num_items] = make_int4(0, 0, 0, 0);
}

__host__ __device__ __forceinline__ constexpr int unpack_rows(int D) { return 2048 / D; }  // of a page that a warp takes

// Page `p` of the output (of a launch whose second axis is the sequences), or with `cu_seqlens` tile `p`.  Called by whole warps.
struct UnpackPage {
  int seq, i;  // the sequence (-1: none) and its page (tile)
  __device__ __forceinline__ UnpackPage(const Unpack& a, int p) : seq(-1), i(0) {
    if (!a.cu_seqlens) {
      seq = blockIdx.y, i = p;
      return;
    }
    if (p >= a.count) return;
    const int lane = threadIdx.x & 31;
    for (int base = 0; base < a.num_seqs; base += 32) {
      const UnpackSequence s(a, base + lane);
      const int sum = warp_prefix(s.tiles);
      const uint32_t reach = __ballot_sync(0xffffffffu, sum > p);
      if (reach) {
        const int from = __ffs(reach) - 1;
        seq = base + from;
        const int kept = __shfl_sync(0xffffffffu, s.kept, from), skip = __shfl_sync(0xffffffffu, s.skip, from);
        i = p - __shfl_sync(0xffffffffu, sum - s.tiles, from);
        if (i >= kept) i += skip - kept;
        return;
      }
      p -= __shfl_sync(0xffffffffu, sum, 31);
    }
  }
  // where its bytes lie, and how many rows of it count
  __device__ __forceinline__ int rows(const Unpack& a, int* page) const {
    *page = i < a.max_pages ? a.block_table[(long)seq * a.max_pages + i] : -1;
    if (*page < 0 || *page >= a.num_pages) {
      *page = 0;
      return 0;
    }
    return min(max(min(a.kv_lens[seq], a.max_len) - i * a.ps, 0), a.ps);
  }
};

// What a lane writes at a time, 16 bytes: 8 values in bfloat16 (from 8 codes), 4 in float32.
__device__ __forceinline__ void unpack_codes(float* to, const uint32_t (&code)[1], float scale) {
  float v[4];
  q8_floats(code[0], v);
  *reinterpret_cast<float4*>(to) = make_float4(v[0] * scale, v[1] * scale, v[2] * scale, v[3] * scale);
}
__device__ __forceinline__ void unpack_codes(bf16* to, const uint32_t (&code)[2], float scale) {
  float lo[4], hi[4];
  q8_floats(code[0], lo);
  q8_floats(code[1], hi);
  const float v[8] = {lo[0] * scale, lo[1] * scale, lo[2] * scale, lo[3] * scale, hi[0] * scale, hi[1] * scale, hi[2] * scale, hi[3] * scale};
  store8(to, v);
}

// A warp per (page, kv head, keys or values, part of the rows: 2,048 channels), 16 bytes of the result a lane, so that what a warp writes at a time is one
// piece; eight loads a lane are under way before the first is used.  What bounds it is the bytes written: 5,306 tokens of 8 heads of 128, padded to
// 12,288, in 9.5 us.  (A warp for all of a page: 10.6, pages of 64 tokens 16; two pieces of 16 bytes side by side a lane, in float32: 33 us
// for 20.)  KNOWN: the head size where the compiler knows it, else 0.
template <typename T, int KNOWN> __global__ void __launch_bounds__(256) unpack_8bit_kernel(Unpack a, int size, int parts, T* __restrict__ k_out, T* __restrict__ v_out) {
  constexpr int AT_ONCE = 8, CHANNELS = 16 / sizeof(T);
  const int D = KNOWN ? KNOWN : size, words = D / CHANNELS, mask = q8_mask(D);
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  uint32_t item = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (item < a.num_items) {
    write_item(a, item);
    return;
  }
  item -= a.num_items;
  const uint32_t half = item >> 1, pair = parts == 1 ? half : half / parts;
  const int is_v = item & 1, part = (int)(half - pair * parts), kvh = (int)(pair % a.nkv), in_all = (int)(pair / a.nkv);
  const int per_tile = a.cu_seqlens ? TILE / a.ps : 1, p = in_all / per_tile, in_tile = in_all - p * per_tile;  // (the page size divides a tile)
  if (p >= (a.cu_seqlens ? a.count : a.width)) return;
  UnpackPage at_page(a, p);
  if (at_page.seq < 0) return;
  at_page.i = at_page.i * per_tile + in_tile;
  if (a.cu_seqlens && at_page.i * a.ps >= min(a.kv_lens[at_page.seq], a.max_len)) return;
  const int place = a.cu_seqlens ? p : blockIdx.y * a.width + p;
  int page;
  const int row0 = part * unpack_rows(D), rows = at_page.rows(a, &page) - row0;  // those that count, from the part's first on
  const Q8Page L(D, a.ps);
  const unsigned char* rec = a.pages + ((long)page * a.nkv + kvh) * L.record;
  const unsigned char* from = rec + (is_v ? L.values : 0) + (long)row0 * D;
  T* to = (is_v ? v_out : k_out) + (((long)place * a.nkv + kvh) * per_tile * a.ps + in_tile * a.ps + row0) * D;
  const float scale = rows > 0 ? reinterpret_cast<const float*>(rec + L.scales)[is_v] : 0.f;
  const int count = min(unpack_rows(D), a.ps - row0) * words, live = rows * words;
  for (int first = lane; first < count; first += 32 * AT_ONCE) {
    uint32_t code[AT_ONCE][CHANNELS / 4];
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      const int at = first + 32 * u;
#pragma unroll
      for (int e = 0; e < CHANNELS / 4; ++e) code[u][e] = 0;
      if (at < count && at < live) {
        if constexpr (CHANNELS == 8)
          *reinterpret_cast<uint2*>(code[u]) = *reinterpret_cast<const uint2*>(from + CHANNELS * at);
        else
          code[u][0] = *reinterpret_cast<const uint32_t*>(from + CHANNELS * at);
      }
    }
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      const int at = first + 32 * u, row = at / words;
      if (at < count) unpack_codes(to + (long)row * D + q8_at(CHANNELS * (at - row * words), row0 + row, mask), code[u], at < live ? scale : 0.f);
    }
  }
}

// Into tiles, whatever the pages' size: a warp per (quarter of a tile, kv head, keys or values), a lane of the first 16 looks a token up.
constexpr int QUARTER = TILE / 4;
template <typename T> __global__ void __launch_bounds__(256) unpack_8bit_other_kernel(Unpack a, int D, T* __restrict__ k_out, T* __restrict__ v_out) {
  constexpr int CHANNELS = 16 / sizeof(T);
  const int words = D / CHANNELS, mask = q8_mask(D);
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  uint32_t item = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (item < a.num_items) {
    write_item(a, item);
    return;
  }
  item -= a.num_items;
  const uint32_t half = item >> 1;
  const int is_v = item & 1, quarter = (int)(half / a.nkv), p = quarter / 4, kvh = (int)(half - (uint32_t)quarter * a.nkv);
  const UnpackPage at_page(a, p);
  if (at_page.seq < 0) return;
  const Q8Page L(D, a.ps);
  // where this lane's token lies, a multiple of 16, and below that how its pieces are ordered; 0: nowhere
  unsigned long long where = 0;
  float scale = 0.f;
  const int key = at_page.i * TILE + quarter % 4 * QUARTER + lane, in_page = key / a.ps;
  if (lane < QUARTER && key < min(a.kv_lens[at_page.seq], a.max_len) && in_page < a.max_pages) {
    const int page = a.block_table[(long)at_page.seq * a.max_pages + in_page], row = key - in_page * a.ps;
    if (page >= 0 && page < a.num_pages) {
      const unsigned char* rec = a.pages + ((long)page * a.nkv + kvh) * L.record;
      scale = reinterpret_cast<const float*>(rec + L.scales)[is_v];
      where = reinterpret_cast<unsigned long long>(rec + (is_v ? L.values : 0) + (long)row * D) | (uint32_t)(row & mask);
    }
  }
  T* to = (is_v ? v_out : k_out) + (((long)p * a.nkv + kvh) * TILE + quarter % 4 * QUARTER) * D;
#pragma unroll 4
  for (int at = lane; at < QUARTER * words; at += 32) {  // (a whole number of warps)
    const int row = at / words, channel = CHANNELS * (at - row * words);
    const unsigned long long from = __shfl_sync(0xffffffffu, where, row);
    const float s = __shfl_sync(0xffffffffu, scale, row);
    uint32_t code[CHANNELS / 4];
#pragma unroll
    for (int e = 0; e < CHANNELS / 4; ++e) code[e] = 0;
    if (from) {
      const unsigned char* c = reinterpret_cast<const unsigned char*>(from & ~15ull) + q8_at(channel, (int)from & 15, 15);
      if constexpr (CHANNELS == 8)
        *reinterpret_cast<uint2*>(code) = *reinterpret_cast<const uint2*>(c);
      else
        code[0] = *reinterpret_cast<const uint32_t*>(c);
    }
    unpack_codes(to + (long)row * D + channel, code, s);
  }
}

template <typename T> cudaError_t launch_unpack(const Unpack& a, int D, T* k_out, T* v_out, cudaStream_t stream) {
  if (a.cu_seqlens && TILE % a.ps)
    return launch_pdl(unpack_8bit_other_kernel<T>, dim3((unsigned)((8L * a.count * a.nkv + a.num_items + 7) / 8)), dim3(256), 0, stream, a, D, k_out, v_out);
  const int parts = (a.ps + unpack_rows(D) - 1) / unpack_rows(D);
  const long items = 2L * (a.cu_seqlens ? a.count * (TILE / a.ps) : a.width) * a.nkv * parts + a.num_items;
  const dim3 grid((unsigned)((items + 7) / 8), a.cu_seqlens ? 1 : a.num_seqs);
  if (D == 64) return launch_pdl(unpack_8bit_kernel<T, 64>, grid, dim3(256), 0, stream, a, D, parts, k_out, v_out);
  if (D == 128) return launch_pdl(unpack_8bit_kernel<T, 128>, grid, dim3(256), 0, stream, a, D, parts, k_out, v_out);
  if (D == 256) return launch_pdl(unpack_8bit_kernel<T, 256>, grid, dim3(256), 0, stream, a, D, parts, k_out, v_out);
  return launch_pdl(unpack_8bit_kernel<T, 0>, grid, dim3(256), 0, stream, a, D, parts, k_out, v_out);
}

inline bool q8_aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

// `units`: pages that get tokens, at most (0: the queries alone); `most_new`: tokens that a sequence brings, at most; `single`: every sequence
// brings one.
Q3_EXPORT int q3_store_8bit(int dtype, const void* qkv, int row_stride, void* q_out, int q_stride, int nq, int nkv, int D, const float* q_w,
                            const float* k_w, float eps, const float* cos_t, const float* sin_t, int rot_half, int max_pos,
                            const int* positions, const int* kv_lens, const int* cu_seqlens, const int* block_table, int max_pages,
                            int num_seqs, void* pages, int num_pages, int ps, int num_tokens, int units, int most_new, int single,
                            int pairing, int* error_word, cudaStream_t stream) {
  if (num_tokens < 1) return Q3_OK;  // (tensors of nothing have no address)
  if (!qkv || !q_out || !positions || nq < 1 || nkv < 1 || pairing < 0 || pairing > 1 || !q8_sizes_ok(D, ps) || units < 0) return Q3_ERR_ARGUMENT;
  if (cos_t && (max_pos < 1 || !sin_t || rot_half < 1 || 2 * rot_half > D)) return Q3_ERR_ARGUMENT;
  if (units > 0 && (!kv_lens || !cu_seqlens || !block_table || !pages || max_pages < 1 || num_seqs < 1 || most_new < 1 || (single && units != num_seqs)))
    return Q3_ERR_ARGUMENT;
  if (dtype != Q3_DTYPE_F32 && dtype != Q3_DTYPE_BF16) return Q3_ERR_ARGUMENT;
  if (units > 0 && !q8_aligned(pages)) return Q3_ERR_UNSUPPORTED;
  Store a{q_w, k_w, cos_t, sin_t, eps, rot_half, max_pos, pairing, positions, kv_lens, cu_seqlens, block_table,
          max_pages, num_pages, num_seqs, num_tokens, ps, units, 1, (unsigned char*)pages, error_word};
  const int tph = D / 16, rows = most_new < ps ? most_new : ps;
  const bool vec = (tph & (tph - 1)) == 0 && row_stride % 8 == 0 && q_stride % 8 == 0 && (!cos_t || 2 * rot_half == D) &&
                   q8_aligned(qkv) && q8_aligned(q_out) && q8_aligned(q_w) && q8_aligned(k_w) && q8_aligned(cos_t) && q8_aligned(sin_t);
  cudaError_t err;
  if (vec) {
    int threads = units > 0 ? (tph * rows + 31) / 32 * 32 : 128;
    threads = threads > STORE_THREADS ? STORE_THREADS : threads;
    a.q_blocks = (nq * tph + threads - 1) / threads;
    const long blocks = (long)units * 2 * nkv + (long)num_tokens * a.q_blocks;
    if (blocks > 0x7fffffffL) return Q3_ERR_UNSUPPORTED;
    auto launch = [&](auto known, auto alone) {
      constexpr int K = decltype(known)::value;
      constexpr bool S = decltype(alone)::value;
      err = dtype == Q3_DTYPE_F32 ? launch_pdl(store_8bit_vec_kernel<float, K, S>, dim3((unsigned)blocks), dim3(threads), 0, stream,
                                               (const float*)qkv, row_stride, (float*)q_out, q_stride, nq, nkv, D, a)
                                  : launch_pdl(store_8bit_vec_kernel<bf16, K, S>, dim3((unsigned)blocks), dim3(threads), 0, stream,
                                               (const bf16*)qkv, row_stride, (bf16*)q_out, q_stride, nq, nkv, D, a);
    };
    auto launch_size = [&](auto alone) {
      if (D == 64)
        launch(std::integral_constant<int, 64>(), alone);
      else if (D == 128)
        launch(std::integral_constant<int, 128>(), alone);
      else if (D == 256)
        launch(std::integral_constant<int, 256>(), alone);
      else
        launch(std::integral_constant<int, 0>(), alone);
    };
    if (single)
      launch_size(std::true_type());
    else
      launch_size(std::false_type());
    return err == cudaSuccess ? Q3_OK : Q3_ERR_LAUNCH;
  }
  // (a page's rows are its warps', one after the other: 475 tokens of 20 + 4 heads of 80 in pages of 64, with their unpacking 49 us with 4 warps, 20 with 16; single
  // tokens leave all but one idle)
  const int warps = units > 0 && rows > 4 ? STORE_THREADS / 32 : 4;
  const long blocks = (long)units * 2 * nkv + ((long)num_tokens * nq + warps - 1) / warps;
  if (blocks > 0x7fffffffL) return Q3_ERR_UNSUPPORTED;
  const size_t smem = (size_t)warps * 2 * D * sizeof(float);
  if (dtype == Q3_DTYPE_F32)
    store_8bit_kernel<float><<<(unsigned)blocks, warps * 32, smem, stream>>>((const float*)qkv, row_stride, (float*)q_out, q_stride, nq, nkv, D, a);
  else
    store_8bit_kernel<bf16><<<(unsigned)blocks, warps * 32, smem, stream>>>((const bf16*)qkv, row_stride, (bf16*)q_out, q_stride, nq, nkv, D, a);
  return q3_launch_status();
}

// `cu_seqlens` null: num_seqs * width pages are written, as large as the cache's; else `count` tiles of 64 tokens and `num_items` items (struct Unpack).
Q3_EXPORT int q3_unpack_8bit(int dtype, const void* pages, int num_pages, int nkv, int D, int ps, const int* block_table, int max_pages,
                             const int* kv_lens, int num_seqs, int max_len, const int* cu_seqlens, int least, int window, int keep_first,
                             int count, int width, void* k_out, void* v_out, int item_tokens, int num_items, void* items,
                             cudaStream_t stream) {
  if (num_seqs < 1 || (cu_seqlens ? count : width) < 1) return Q3_OK;
  if (!pages || !block_table || !kv_lens || !k_out || !v_out || nkv < 1 || max_pages < 1 || !q8_sizes_ok(D, ps)) return Q3_ERR_ARGUMENT;
  if (cu_seqlens ? !items || item_tokens < 1 || num_items < 0 || least < 1 || keep_first < 0 || window + (long)keep_first > 1 << 30 || !q8_aligned(items)
                 : num_items != 0)
    return Q3_ERR_ARGUMENT;
  if (dtype != Q3_DTYPE_F32 && dtype != Q3_DTYPE_BF16) return Q3_ERR_ARGUMENT;
  if ((!cu_seqlens && num_seqs > 65535) || !q8_aligned(pages) || !q8_aligned(k_out) || !q8_aligned(v_out)) return Q3_ERR_UNSUPPORTED;
  if ((long)(cu_seqlens ? (long)count * (TILE % ps ? 4 : TILE / ps) : width) * 2 * nkv * ((ps + unpack_rows(D) - 1) / unpack_rows(D)) + num_items > 0x7fffffffL) return Q3_ERR_UNSUPPORTED;
  const Unpack a{(const unsigned char*)pages, num_pages, nkv, ps, block_table, kv_lens, cu_seqlens, max_pages, num_seqs, max_len, least, window,
                 keep_first, count, width, item_tokens, num_items, (int4*)items};
  const cudaError_t err = dtype == Q3_DTYPE_F32 ? launch_unpack(a, D, (float*)k_out, (float*)v_out, stream)
                                                : launch_unpack(a, D, (bf16*)k_out, (bf16*)v_out, stream);
  return err == cudaSuccess ? Q3_OK : Q3_ERR_LAUNCH;
}
