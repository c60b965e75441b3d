// The cache in 4 bits (layout and rounding: four_bit.cuh): what writes it, what reads it back, and what drops tokens from it.
//
// * store:  per-head q/k RMSNorm, rotation, and the write of keys and values in 4 bits, as rope_kv.cu does it for wide pages: the same
//           float32 arithmetic in the same order, so queries have the same bits.
// * unpack: a step's sequences as pages of bfloat16 or float32, one after the other, for the attention over prompts.
// * evict:  see evict_select_kernel.
#include "four_bit.cuh"
#include "rotary.cuh"

#define Q3_ERR_POSITION 16

namespace {

struct Store {
  const float *q_w, *k_w, *cos_t, *sin_t;
  float eps;
  int rot_half, max_pos, pairing;
  const int *positions, *slots, *token_seq, *block_table;  // slots: a token's place in its sequence's cache (null: its position)
  int max_pages, num_pages, num_seqs, ps, write_kv;
  unsigned char* pages;
  float* mass;  // null, or [pages][kv_heads][ps]: zeroed for what is written
  int* places;  // null, or the same shape: gets the position
  int* error_word;
};

// Where a token's row of a kv head goes: the record's first byte and the row in it; false: nowhere.
__device__ __forceinline__ bool store_place(const Store& a, int t, int nkv, int kvh, long record, unsigned char** at, int* row, long* cell) {
  const int slot = a.slots ? a.slots[t] : a.positions[t];
  const int seq = a.token_seq[t];
  if (slot < 0 || slot / a.ps >= a.max_pages || seq < 0 || seq >= a.num_seqs) return false;
  const int page = a.block_table[(long)seq * a.max_pages + slot / a.ps];
  if (page < 0 || page >= a.num_pages) return false;
  *row = slot % a.ps;
  *at = a.pages + ((long)page * nkv + kvh) * record;
  *cell = ((long)page * nkv + kvh) * a.ps + *row;
  return true;
}

// Head sizes 16, 32, 64, 128, 256 with the rotation over the whole head (or none): D / 16 threads per (token, head); thread c owns
// channels [8c, 8c + 8) and [D/2 + 8c, D/2 + 8c + 8), which are one word of 4-bit numbers each.  Limited by the bytes of the projection
// and of the queries; the divisions of the rounding hide behind them.
template <typename T>
__global__ void store_4bit_vec_kernel(const T* qkv, int row_stride, T* q_out, int q_stride, int nq, int nkv, int D, int G, int tph_shift,
                                      Store a) {
  const int tph = 1 << tph_shift;
  const int heads = a.write_kv ? nq + 2 * nkv : nq;
  pdl_wait();
  pdl_launch_dependents();
  const int u = blockIdx.y * blockDim.x + threadIdx.x;
  const int t = blockIdx.x;
  const int hi_raw = u >> tph_shift;
  const int c = u & (tph - 1);
  const bool live = hi_raw < heads;
  const int hi = live ? hi_raw : 0;
  const int half = D / 2;
  const T* x = qkv + (long)t * row_stride + (long)hi * D;
  const int p = a.positions[t];
  float v0[8], v1[8];
  if (live) {
    load8(x + 8 * c, v0);
    load8(x + half + 8 * c, v1);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v0[e] = v1[e] = 0.f;
  }
  const bool is_v = hi >= nq + nkv, is_q = hi < nq;
  const float* w = is_q ? a.q_w : a.k_w;
  float ss = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) ss += v0[e] * v0[e] + v1[e] * v1[e];
  for (int o = tph >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  bool turned = true;
  if (!is_v) {
    if (w) {
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
    if (a.cos_t) {
      if (p < 0 || p >= a.max_pos) {
        if (live && a.error_word && c == 0) atomicExch(a.error_word, Q3_ERR_POSITION);
        turned = false;
      } else {
        rotate_chunks(v0, v1, a.cos_t + (long)p * half, a.sin_t + (long)p * half, c, half, a.pairing);
      }
    }
  }
  if (live && is_q) {
    if (turned) {
      T* y = q_out + (long)t * q_stride + (long)hi * D;
      store8(y + 8 * c, v0);
      store8(y + half + 8 * c, v1);
    }
  }
  // (all lanes take part in the reductions: heads of queries and keys may share a warp)
  float lo0 = v0[0], hi0 = v0[0], lo1 = v1[0], hi1 = v1[0], nan0 = 0.f, nan1 = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    lo0 = fminf(lo0, v0[e]), hi0 = fmaxf(hi0, v0[e]), nan0 += v0[e] * 0.f;
    lo1 = fminf(lo1, v1[e]), hi1 = fmaxf(hi1, v1[e]), nan1 += v1[e] * 0.f;
  }
  if (G == 1) {  // both words lie in the one group
    lo0 = lo1 = fminf(lo0, lo1), hi0 = hi1 = fmaxf(hi0, hi1), nan0 = nan1 = nan0 + nan1;
  }
  const int lanes = G == 1 ? tph : 8;  // of one group
  for (int o = lanes >> 1; o > 0; o >>= 1) {
    lo0 = fminf(lo0, __shfl_xor_sync(0xffffffffu, lo0, o));
    hi0 = fmaxf(hi0, __shfl_xor_sync(0xffffffffu, hi0, o));
    nan0 += __shfl_xor_sync(0xffffffffu, nan0, o);
    lo1 = fminf(lo1, __shfl_xor_sync(0xffffffffu, lo1, o));
    hi1 = fmaxf(hi1, __shfl_xor_sync(0xffffffffu, hi1, o));
    nan1 += __shfl_xor_sync(0xffffffffu, nan1, o);
  }
  if (!live || is_q || !turned) return;
  const int kvh = is_v ? hi - nq - nkv : hi - nq;
  const Q4Page L(D, G, a.ps);
  unsigned char* rec;
  int row;
  long cell;
  if (!store_place(a, t, nkv, kvh, L.record, &rec, &row, &cell)) return;
  const Q4Scale y0 = q4_scale(lo0, hi0, nan0), y1 = q4_scale(lo1, hi1, nan1);
  uint32_t* code = reinterpret_cast<uint32_t*>(rec + (is_v ? L.values : 0) + (long)row * L.half);
  uint32_t* par = reinterpret_cast<uint32_t*>(rec + (is_v ? L.vpar : L.kpar) + (long)row * L.par);
  // group and index in it of the two words
  const int g0 = G == 1 ? 0 : c >> 3, i0 = G == 1 ? c : c & 7;
  const int g1 = G == 1 ? 0 : G / 2 + (c >> 3), i1 = G == 1 ? tph + c : c & 7;
  code[i0 * G + g0] = q4_word(v0, y0);
  code[i1 * G + g1] = q4_word(v1, y1);
  if (i0 == 0) {
    par[g0] = y0.word;
    if (G > 1) par[g1] = y1.word;
  }
  if (!is_v && c == 0) {
    if (a.mass) a.mass[cell] = 0.f;
    if (a.places) a.places[cell] = p;
  }
}

// Any other size: one warp per (token, head).
template <typename T, int WARPS>
__global__ void store_4bit_kernel(const T* qkv, int row_stride, T* q_out, int q_stride, int nq, int nkv, int D, int G, int num_tokens,
                                  Store a) {
  extern __shared__ float stage[];  // WARPS * 2 * D
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int heads = a.write_kv ? nq + 2 * nkv : nq;
  const long item = (long)blockIdx.x * WARPS + warp;
  if (item >= (long)num_tokens * heads) return;
  const int t = (int)(item / heads);
  const int hi = (int)(item - (long)t * heads);
  const T* x = qkv + (long)t * row_stride + (long)hi * D;
  const int p = a.positions[t];
  const bool is_v = hi >= nq + nkv, is_q = hi < nq;
  if (a.cos_t && !is_v && (p < 0 || p >= a.max_pos)) {
    if (a.error_word && lane == 0) atomicExch(a.error_word, Q3_ERR_POSITION);
    return;
  }
  float* xs = stage + warp * 2 * D;
  float* ys = xs + D;
  float ss = 0.f;
  for (int d = lane; d < D; d += 32) {
    const float v = to_f32(x[d]);
    xs[d] = v;
    ss += v * v;
  }
  const float* w = is_v ? nullptr : is_q ? a.q_w : a.k_w;
  const float rstd = w ? rsqrtf(warp_sum(ss) / (float)D + a.eps) : 1.f;
  __syncwarp();
  const float* cs = a.cos_t && !is_v ? a.cos_t + (long)p * a.rot_half : nullptr;
  const float* sn = cs ? a.sin_t + (long)p * a.rot_half : nullptr;
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
  if (is_q) {
    T* y = q_out + (long)t * q_stride + (long)hi * D;
    for (int d = lane; d < D; d += 32) y[d] = from_f32<T>(ys[d]);
    return;
  }
  const int kvh = is_v ? hi - nq - nkv : hi - nq;
  const Q4Page L(D, G, a.ps);
  unsigned char* rec;
  int row;
  long cell;
  if (!store_place(a, t, nkv, kvh, L.record, &rec, &row, &cell)) return;
  uint32_t* code = reinterpret_cast<uint32_t*>(rec + (is_v ? L.values : 0) + (long)row * L.half);
  uint32_t* par = reinterpret_cast<uint32_t*>(rec + (is_v ? L.vpar : L.kpar) + (long)row * L.par);
  const int size = D / G;
  for (int g = 0; g < G; ++g) {
    float lo = INFINITY, high = -INFINITY, nan = 0.f;
    for (int d = lane; d < size; d += 32) {
      const float v = ys[g * size + d];
      lo = fminf(lo, v), high = fmaxf(high, v), nan += v * 0.f;
    }
    lo = -warp_max(-lo), high = warp_max(high), nan = warp_sum(nan);
    const Q4Scale y = q4_scale(lo, high, nan);
    if (lane < size / 8) {
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = ys[g * size + 8 * lane + e];
      code[lane * G + g] = q4_word(v, y);
    }
    if (lane == 0) par[g] = y.word;
  }
  if (!is_v && lane == 0) {
    if (a.mass) a.mass[cell] = 0.f;
    if (a.places) a.places[cell] = p;
  }
}

// ---- back to wide pages -------------------------------------------------------------------------------------------------------------
// Block: one page of one sequence and kv head.  out page index: sequence's row * width + its page; rows behind the sequence's last token
// are zero, and pages behind it too (fill) or left alone (not fill).  `cu_seqlens` (may be null): only sequences that bring more than
// one token count, in order; `table_out` [num_seqs][width] then gets where their pages went.
template <typename T>
__global__ void unpack_4bit_kernel(const unsigned char* __restrict__ pages, int num_pages, int nkv, int D, int G, int ps,
                                   const int* __restrict__ block_table, int max_pages, const int* __restrict__ kv_lens, int num_seqs,
                                   int max_len, const int* __restrict__ cu_seqlens, int width, int fill, T* __restrict__ k_out,
                                   T* __restrict__ v_out, int* __restrict__ table_out) {
  pdl_wait();
  pdl_launch_dependents();
  const int i = blockIdx.x, kvh = blockIdx.y;
  int seq = blockIdx.z;
  if (cu_seqlens) {  // the blockIdx.z-th of the sequences with more than one token
    int want = blockIdx.z, base = 0;
    seq = -1;
    for (; base < num_seqs; base += 32) {
      const int s = base + (threadIdx.x & 31);
      const bool is = s < num_seqs && cu_seqlens[s + 1] - cu_seqlens[s] > 1;
      const uint32_t found = __ballot_sync(0xffffffffu, is);
      if (want < __popc(found)) {
        seq = base + __fns(found, 0, want + 1);
        break;
      }
      want -= __popc(found);
    }
    if (seq < 0) return;
  }
  const int len = min(kv_lens[seq], max_len);
  const int place = blockIdx.z * width + i;
  if (table_out && kvh == 0 && threadIdx.x == 0) table_out[(long)seq * width + i] = place;
  int rows = min(max(len - i * ps, 0), ps);
  int page = -1;
  if (rows > 0 && i < max_pages) page = block_table[(long)seq * max_pages + i];
  if (page < 0 || page >= num_pages) rows = 0;
  if (rows == 0 && !fill) return;
  const Q4Page L(D, G, ps);
  const unsigned char* rec = pages + ((long)max(page, 0) * nkv + kvh) * L.record;
  const int words = D / 8, size_words = words / G;
  const long out_base = ((long)place * nkv + kvh) * ps * D;
  for (int u = threadIdx.x; u < 2 * ps * words; u += blockDim.x) {
    const int is_v = u >= ps * words;
    const int at = u - is_v * ps * words;
    const int row = at / words, w = at - row * words;  // word in the order of channels
    const int g = w / size_words, idx = w - g * size_words;
    float v[8];
    if (row < rows) {
      const uint32_t code = *reinterpret_cast<const uint32_t*>(rec + (is_v ? L.values : 0) + (long)row * L.half + 4 * (idx * G + g));
      const uint32_t par = *reinterpret_cast<const uint32_t*>(rec + (is_v ? L.vpar : L.kpar) + (long)row * L.par + 4 * g);
      const float s = q4_s(par), z = q4_z(par);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = z + (float)((code >> (4 * e)) & 15u) * s;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = 0.f;
    }
    store8((is_v ? v_out : k_out) + out_base + (long)at * 8, v);
  }
}

// ---- eviction -------------------------------------------------------------------------------------------------------------------------
// Per (layer, sequence, kv head) that holds more than `keep` tokens: which tokens stay, and who fills whose place.  Stay: positions below
// `first`, the last `recent` positions, and of the others those with the largest sums until `keep` are found (equal sums: the lower
// place; NaN counts as the largest).  The tokens that go leave holes among the first `keep` places, which the tokens that stay from
// behind `keep` fill, both in order: nothing that stays in front moves, and no token's source is another's goal, so the moves are
// independent of each other.
// One block: order-preserving keys in shared memory (or scratch when they are too many), the threshold by four passes of a histogram
// over 8 bits, then both lists by scans.  Limited by the latency of these passes (few blocks) or by reading sums and positions.
constexpr int EVICT_THREADS = 1024;

__device__ __forceinline__ int block_scan(int v, int* total, int* red) {  // exclusive sum over the block; red: 33 ints
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) red[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int s = lane < (int)(blockDim.x >> 5) ? red[lane] : 0;
    const int own = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += y;
    }
    red[lane] = s - own;
    if (lane == 31) red[32] = s;
  }
  __syncthreads();
  *total = red[32];
  return x - v + red[warp];
}

struct Evict {
  const int *block_table, *kv_lens;
  int max_pages, num_pages, num_seqs, nkv, ps, keep, first, recent, cap, max_len;
  float* mass;
  int* places;
  uint32_t* spill;  // null, or [pairs][max_len]: the keys when they do not fit shared memory
  int* lists;       // [pairs][1 + 2 cap]: how many, holes, movers
};

__global__ void __launch_bounds__(EVICT_THREADS, 1) evict_select_kernel(Evict a) {
  extern __shared__ uint32_t keys_s[];
  __shared__ int hist[256], red[33], s_newest, s_digit, s_left;
  pdl_wait();
  pdl_launch_dependents();
  const int kvh = blockIdx.x, seq = blockIdx.y, layer = blockIdx.z;
  const long pair = ((long)layer * a.num_seqs + seq) * a.nkv + kvh;
  int* list = a.lists + pair * (1 + 2 * (long)a.cap);
  const int n = min(a.kv_lens[seq], a.max_len), tid = threadIdx.x;
  if (n <= a.keep) {
    if (tid == 0) list[0] = 0;
    return;
  }
  uint32_t* keys = a.spill ? a.spill + pair * a.max_len : keys_s;
  const int* bt = a.block_table + (long)seq * a.max_pages;
  const long layer_cells = (long)layer * a.num_pages * a.nkv * a.ps;
  auto cell = [&](int slot) -> long {
    const int page = bt[slot / a.ps];
    return page < 0 || page >= a.num_pages ? -1 : layer_cells + ((long)page * a.nkv + kvh) * a.ps + slot % a.ps;
  };
  if (tid == 0) s_newest = -1;
  __syncthreads();
  int newest = -1;
  for (int i = tid; i < n; i += EVICT_THREADS) {
    const long c = cell(i);
    const int place = c < 0 ? -1 : a.places[c];
    newest = max(newest, place);
    const float m = c < 0 ? -INFINITY : a.mass[c] + 0.f;  // (minus zero is zero)
    uint32_t key = __float_as_uint(m);
    key = m != m ? 0xFFFFFFFEu : (key & 0x80000000u) ? ~key : key | 0x80000000u;
    keys[i] = c >= 0 && place < a.first ? 0xFFFFFFFFu : key;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) newest = max(newest, __shfl_xor_sync(0xffffffffu, newest, o));
  if ((tid & 31) == 0) atomicMax(&s_newest, newest);
  __syncthreads();
  newest = s_newest;
  for (int i = tid; i < n; i += EVICT_THREADS) {
    const long c = cell(i);
    if (c >= 0 && a.places[c] > newest - a.recent) keys[i] = 0xFFFFFFFFu;
  }
  // the keep-th largest key
  uint32_t prefix = 0, mask = 0;
  int left = a.keep;  // how many of those that share the prefix stay
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += EVICT_THREADS)
      if ((keys[i] & mask) == prefix) atomicAdd(&hist[(keys[i] >> shift) & 255], 1);
    __syncthreads();
    if (tid < 32) {  // from the largest digit down: lane l holds digits 255 - 8 l .. 248 - 8 l
      int own = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) own += hist[255 - 8 * tid - e];
      int sum = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, sum, o);
        if (tid >= o) sum += y;
      }
      int before = sum - own;
      if (before < left && left <= sum) {
        for (int e = 0; e < 8; ++e) {
          const int d = 255 - 8 * tid - e;
          if (before + hist[d] >= left) {
            s_digit = d;
            s_left = left - before;
            break;
          }
          before += hist[d];
        }
      }
    }
    __syncthreads();
    prefix |= (uint32_t)s_digit << shift;
    mask |= 255u << shift;
    left = s_left;
  }
  // holes in front, movers behind, in order; of the keys equal to the threshold the first `left` stay
  int ties = 0, holes = 0, movers = 0;
  for (int base = 0; base < n; base += EVICT_THREADS) {
    const int i = base + tid;
    const uint32_t key = i < n ? keys[i] : 0;
    const bool tie = i < n && key == prefix;
    int t_all, f_all;
    const int rank = ties + block_scan(tie, &t_all, red);
    const bool stays = i < n && (key > prefix || (tie && rank < left));
    const bool hole = i < n && i < a.keep && !stays, mover = i >= a.keep && stays;
    const int at = block_scan((hole ? 1 : 0) | (mover ? 1 << 16 : 0), &f_all, red);  // (at most 1024 of each)
    if (hole) list[1 + holes + (at & 0xFFFF)] = i;
    if (mover) list[1 + a.cap + movers + (at >> 16)] = i;
    ties += t_all;
    holes += f_all & 0xFFFF;
    movers += f_all >> 16;
  }
  if (tid == 0) list[0] = min(holes, movers);
}

// Moves rows: a group of 8 lanes per moved token; codes in pieces of 16 bytes, parameters in words.
__global__ void evict_move_kernel(Evict a, unsigned char* pages, int D, int G) {
  pdl_wait();
  pdl_launch_dependents();
  const int kvh = blockIdx.y % a.nkv, seq = blockIdx.y / a.nkv, layer = blockIdx.z;
  const long pair = ((long)layer * a.num_seqs + seq) * a.nkv + kvh;
  const int* list = a.lists + pair * (1 + 2 * (long)a.cap);
  const int count = list[0];
  const Q4Page L(D, G, a.ps);
  const int* bt = a.block_table + (long)seq * a.max_pages;
  const long layer_heads = (long)layer * a.num_pages * a.nkv;
  const int lane = threadIdx.x & 7, per_block = blockDim.x >> 3;
  const bool wide = L.half % 16 == 0;
  for (int m = blockIdx.x * per_block + (threadIdx.x >> 3); m < count; m += gridDim.x * per_block) {
    const int to = list[1 + m], from = list[1 + a.cap + m];
    const int tp = bt[to / a.ps], fp = bt[from / a.ps];
    if (tp < 0 || fp < 0 || tp >= a.num_pages || fp >= a.num_pages) continue;
    const long th = layer_heads + (long)tp * a.nkv + kvh, fh = layer_heads + (long)fp * a.nkv + kvh;
    const int tr = to % a.ps, fr = from % a.ps;
    unsigned char *dst = pages + th * L.record, *src = pages + fh * L.record;
    if (wide) {
      const int pieces = L.half / 16;
      for (int u = lane; u < 2 * pieces; u += 8) {
        const int is_v = u >= pieces;
        const long sec = is_v ? L.values : 0, off = 16 * (u - is_v * pieces);
        *reinterpret_cast<uint4*>(dst + sec + (long)tr * L.half + off) = *reinterpret_cast<const uint4*>(src + sec + (long)fr * L.half + off);
      }
    } else {
      const int words = L.half / 4;
      for (int u = lane; u < 2 * words; u += 8) {
        const int is_v = u >= words;
        const long sec = is_v ? L.values : 0, off = 4 * (u - is_v * words);
        *reinterpret_cast<uint32_t*>(dst + sec + (long)tr * L.half + off) =
            *reinterpret_cast<const uint32_t*>(src + sec + (long)fr * L.half + off);
      }
    }
    for (int u = lane; u < 2 * G; u += 8) {
      const int is_v = u >= G;
      const long sec = is_v ? L.vpar : L.kpar, off = 4 * (u - is_v * G);
      *reinterpret_cast<uint32_t*>(dst + sec + (long)tr * L.par + off) =
          *reinterpret_cast<const uint32_t*>(src + sec + (long)fr * L.par + off);
    }
    if (lane == 0) a.mass[th * a.ps + tr] = a.mass[fh * a.ps + fr];
    if (lane == 1) a.places[th * a.ps + tr] = a.places[fh * a.ps + fr];
  }
}

inline bool q4_aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

Q3_EXPORT int q3_store_4bit(int dtype, const void* qkv, int row_stride, void* q_out, int q_stride, int nq, int nkv, int D, const float* q_w,
                            const float* k_w, float eps, const float* cos_t, const float* sin_t, int rot_half, int max_pos,
                            const int* positions, const int* slots, const int* token_seq, const int* block_table, int max_pages,
                            int num_seqs, void* pages, int num_pages, int ps, int num_tokens, int write_kv, int pairing, float* mass,
                            int* places, int* error_word, cudaStream_t stream) {
  if (!qkv || !q_out || !positions || nq < 1 || nkv < 1 || pairing < 0 || pairing > 1 || !q4_sizes_ok(D, ps)) return Q3_ERR_ARGUMENT;
  if (cos_t && (max_pos < 1 || !sin_t || rot_half < 1 || 2 * rot_half > D)) return Q3_ERR_ARGUMENT;
  if (write_kv && (!token_seq || !block_table || !pages || max_pages < 1)) return Q3_ERR_ARGUMENT;
  if (dtype != Q3_DTYPE_F32 && dtype != Q3_DTYPE_BF16) return Q3_ERR_ARGUMENT;
  if (num_tokens == 0) return Q3_OK;
  Store a{q_w, k_w, cos_t, sin_t, eps, rot_half, max_pos, pairing, positions, slots, token_seq, block_table,
          max_pages, num_pages, num_seqs, ps, write_kv, (unsigned char*)pages, mass, places, error_word};
  const int G = q4_groups(D), tph = D / 16;
  const bool vec = (tph & (tph - 1)) == 0 && row_stride % 8 == 0 && q_stride % 8 == 0 && (!cos_t || 2 * rot_half == D) &&
                   q4_aligned(qkv) && q4_aligned(q_out) && q4_aligned(q_w) && q4_aligned(k_w) && q4_aligned(cos_t) && q4_aligned(sin_t);
  cudaError_t err;
  if (vec) {
    int shift = 0;
    while ((1 << shift) < tph) ++shift;
    const int threads = 128, per_token = (write_kv ? nq + 2 * nkv : nq) * tph;
    const dim3 grid((unsigned)num_tokens, (unsigned)((per_token + threads - 1) / threads));
    if (grid.y > 65535) return Q3_ERR_UNSUPPORTED;
    err = dtype == Q3_DTYPE_F32 ? launch_pdl(store_4bit_vec_kernel<float>, grid, dim3(threads), 0, stream, (const float*)qkv, row_stride,
                                             (float*)q_out, q_stride, nq, nkv, D, G, shift, a)
                                : launch_pdl(store_4bit_vec_kernel<bf16>, grid, dim3(threads), 0, stream, (const bf16*)qkv, row_stride,
                                             (bf16*)q_out, q_stride, nq, nkv, D, G, shift, a);
    return err == cudaSuccess ? Q3_OK : Q3_ERR_LAUNCH;
  }
  constexpr int WARPS = 4;
  const long items = (long)num_tokens * (write_kv ? nq + 2 * nkv : nq);
  if (items > 0x7fffffffL) return Q3_ERR_UNSUPPORTED;
  const unsigned blocks = (unsigned)((items + WARPS - 1) / WARPS);
  const size_t smem = (size_t)WARPS * 2 * D * sizeof(float);
  if (dtype == Q3_DTYPE_F32)
    store_4bit_kernel<float, WARPS><<<blocks, WARPS * 32, smem, stream>>>((const float*)qkv, row_stride, (float*)q_out, q_stride, nq, nkv,
                                                                          D, G, num_tokens, a);
  else
    store_4bit_kernel<bf16, WARPS><<<blocks, WARPS * 32, smem, stream>>>((const bf16*)qkv, row_stride, (bf16*)q_out, q_stride, nq, nkv, D,
                                                                         G, num_tokens, a);
  return q3_launch_status();
}

Q3_EXPORT int q3_unpack_4bit(int dtype, const void* pages, int num_pages, int nkv, int D, int ps, const int* block_table, int max_pages,
                             const int* kv_lens, int num_seqs, int max_len, const int* cu_seqlens, int count, int width, int fill,
                             void* k_out, void* v_out, int* table_out, cudaStream_t stream) {
  if (!pages || !block_table || !kv_lens || !k_out || !v_out || nkv < 1 || max_pages < 1 || !q4_sizes_ok(D, ps)) return Q3_ERR_ARGUMENT;
  if (dtype != Q3_DTYPE_F32 && dtype != Q3_DTYPE_BF16) return Q3_ERR_ARGUMENT;
  if (count < 1 || width < 1) return Q3_OK;
  if (nkv > 65535 || count > 65535) return Q3_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)width, (unsigned)nkv, (unsigned)count);
  const int G = q4_groups(D);
  const int threads = ps * D / 8 >= 256 ? 256 : 128;
  const cudaError_t err =
      dtype == Q3_DTYPE_F32
          ? launch_pdl(unpack_4bit_kernel<float>, grid, dim3(threads), 0, stream, (const unsigned char*)pages, num_pages, nkv, D, G, ps,
                       block_table, max_pages, kv_lens, num_seqs, max_len, cu_seqlens, width, fill, (float*)k_out, (float*)v_out, table_out)
          : launch_pdl(unpack_4bit_kernel<bf16>, grid, dim3(threads), 0, stream, (const unsigned char*)pages, num_pages, nkv, D, G, ps,
                       block_table, max_pages, kv_lens, num_seqs, max_len, cu_seqlens, width, fill, (bf16*)k_out, (bf16*)v_out, table_out);
  return err == cudaSuccess ? Q3_OK : Q3_ERR_LAUNCH;
}

// Keys that one block holds in shared memory; above, `spill` is needed.
#define Q3_EVICT_KEYS 49152

Q3_EXPORT int q3_evict_4bit_keys() { return Q3_EVICT_KEYS; }

Q3_EXPORT int q3_evict_4bit(void* pages, int num_layers, int num_pages, int nkv, int D, int ps, float* mass, int* places,
                            const int* block_table, int max_pages, const int* kv_lens, int num_seqs, int max_len, int keep, int first,
                            int recent, int cap, void* spill, int* lists, cudaStream_t stream) {
  if (!pages || !mass || !places || !block_table || !kv_lens || !lists || nkv < 1 || max_pages < 1 || !q4_sizes_ok(D, ps))
    return Q3_ERR_ARGUMENT;
  if (keep < 1 || first < 0 || recent < 0 || (long)first + recent > keep || cap < 1 || max_len > (long)max_pages * ps) return Q3_ERR_ARGUMENT;
  if (max_len > Q3_EVICT_KEYS && !spill) return Q3_ERR_ARGUMENT;
  if (num_seqs < 1 || num_layers < 1 || max_len <= keep) return Q3_OK;
  if (num_seqs > 65535 || num_layers > 65535 || (long)num_seqs * nkv > 65535) return Q3_ERR_UNSUPPORTED;
  Evict a{block_table, kv_lens, max_pages, num_pages, num_seqs, nkv, ps, keep, first, recent, cap, max_len, mass, places,
          max_len > Q3_EVICT_KEYS ? (uint32_t*)spill : nullptr, lists};
  static bool once[Q3_MAX_DEVICES];
  const int dev = q3_current_device();
  if (!once[dev]) {
    if (cudaFuncSetAttribute(evict_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 4 * Q3_EVICT_KEYS) != cudaSuccess)
      return Q3_ERR_LAUNCH;
    once[dev] = true;
  }
  const size_t smem = a.spill ? 0 : 4 * (size_t)max_len;
  cudaError_t err = launch_pdl(evict_select_kernel, dim3(nkv, num_seqs, num_layers), dim3(EVICT_THREADS), smem, stream, a);
  if (err != cudaSuccess) return Q3_ERR_LAUNCH;
  const int G = q4_groups(D);
  const long pairs = (long)num_seqs * nkv * num_layers;
  // 32 tokens a block at a time, about eight blocks an SM
  long chunks = (cap + 31) / 32, most = (148 * 8 + pairs - 1) / pairs;
  if (chunks > most) chunks = most;
  if (chunks < 1) chunks = 1;
  err = launch_pdl(evict_move_kernel, dim3((unsigned)chunks, (unsigned)(num_seqs * nkv), (unsigned)num_layers), dim3(256), 0, stream, a,
                   (unsigned char*)pages, D, G);
  return err == cudaSuccess ? Q3_OK : Q3_ERR_LAUNCH;
}
