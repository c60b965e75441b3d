// The cache in 4 bits (layout and rounding: four_bit.cuh): what writes it, what reads it back, and what drops tokens from it.
//
// * store:  per-head q/k RMSNorm, rotation, and the write of keys and values in 4 bits, as rope_kv.cu does it for wide pages.
// * unpack: a step's sequences as pages of bfloat16 or float32, one after the other, for the attention over prompts.
// * evict:  see evict_select_kernel.
#include <limits.h>

#include <type_traits>

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
// channels [8c, 8c + 8) and [D/2 + 8c, D/2 + 8c + 8), which are one word of 4-bit numbers each.  The floor is the bytes of the projection
// and of the queries; 3,258 tokens of 32 + 8 heads of 128 take 24 us, 2.9 TB/s.  What bounds it: schedulers issue in 0.7 of their clocks, and
// the rest waits for loads.  One side alone gives nothing: two numbers an instruction (24), angles asked for into L1 (25) or into registers
// ahead of the squares' sum (26), three heads a thread (41), blocks of 64 to 256 threads (24 to 28).
//
// A key near the border between two numbers falls on either side by float32's last bit.  So that it falls where element-wise float32
// operations put it that anybody can repeat, heads of 128 and 256 sum their squares in a stated order, four neighbours at a time and then
// by halves, and products and sums are rounded one by one (with fused products and another order 14 keys of 59 million fell elsewhere).
// Heads of 16, 32 and 64 add fused squares, as the general form below does.
__device__ __forceinline__ float quad_of_squares(const float* v) {
  return __fadd_rn(__fadd_rn(__fadd_rn(__fmul_rn(v[0], v[0]), __fmul_rn(v[1], v[1])), __fmul_rn(v[2], v[2])), __fmul_rn(v[3], v[3]));
}
__device__ __forceinline__ void turn_rounded(float& a, float& b, float cs, float sn) {
  const float x = a, y = b;
  a = __fsub_rn(__fmul_rn(x, cs), __fmul_rn(y, sn));
  b = __fadd_rn(__fmul_rn(y, cs), __fmul_rn(x, sn));
}
__device__ __forceinline__ float least_or_nan(float x, float y) {
  float z;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(z) : "f"(x), "f"(y));
  return z;
}
// KNOWN: the head size where the compiler knows it, else 0.
template <typename T, int KNOWN>
__global__ void store_4bit_vec_kernel(const T* qkv, int row_stride, T* q_out, int q_stride, int nq, int nkv, int size, Store a) {
  const int D = KNOWN ? KNOWN : size, G = q4_groups(D), tph = D / 16, tph_shift = 31 - __clz(tph);
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
  if (__all_sync(0xffffffffu, !live || is_q)) return;
  // (else all lanes take part in the reductions: heads of queries and keys may share a warp)
  float lo0 = v0[0], hi0 = v0[0], lo1 = v1[0], hi1 = v1[0];
#pragma unroll
  for (int e = 1; e < 8; ++e) {
    lo0 = least_or_nan(lo0, v0[e]), hi0 = fmaxf(hi0, v0[e]);
    lo1 = least_or_nan(lo1, v1[e]), hi1 = fmaxf(hi1, v1[e]);
  }
  if (G == 1) lo0 = least_or_nan(lo0, lo1), hi0 = fmaxf(hi0, hi1);  // both words lie in the one group
  const int lanes = G == 1 ? tph : 8;                               // of one group
#pragma unroll
  for (int o = lanes >> 1; o > 0; o >>= 1) {
    lo0 = least_or_nan(lo0, __shfl_xor_sync(0xffffffffu, lo0, o));
    hi0 = fmaxf(hi0, __shfl_xor_sync(0xffffffffu, hi0, o));
    if (G > 1) {
      lo1 = least_or_nan(lo1, __shfl_xor_sync(0xffffffffu, lo1, o));
      hi1 = fmaxf(hi1, __shfl_xor_sync(0xffffffffu, hi1, o));
    }
  }
  if (!live || is_q || !turned) return;
  const int kvh = is_v ? hi - nq - nkv : hi - nq;
  const Q4Page L(D, G, a.ps);
  unsigned char* rec;
  int row;
  long cell;
  if (!store_place(a, t, nkv, kvh, L.record, &rec, &row, &cell)) return;
  const Q4Scale y0 = q4_scale(lo0, hi0), y1 = G == 1 ? y0 : q4_scale(lo1, hi1);
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
    const Q4Scale y = q4_scale(lo + nan, high);
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
// Two forms.  Without `cu_seqlens`, sequence z's page i goes to page z * width + i, rows behind its last token are zero, and whole pages behind
// it too.  With it, the attention over prompts reads the pages: only sequences that bring at least `least` tokens count, and of each
// only the pages that its first new token's window reaches up to the last token's; they lie one after the other, `count` pages in all, and
// `table_out` [num_seqs][width] says where (entries that nobody asks for name a page of the same sequence, never none).
struct Unpack {
  const unsigned char* pages;
  int num_pages, nkv, ps;
  const int *block_table, *kv_lens, *cu_seqlens;
  int max_pages, num_seqs, max_len, least, window, count, width;
  int* table_out;
};

// Page `p` of the output (of a launch whose second axis is the sequences, without `cu_seqlens`).  Called by whole warps.
struct UnpackPage {
  int seq, i, first, last;  // the sequence (-1: none), its page, and the first and last of its pages that count
  __device__ __forceinline__ UnpackPage(const Unpack& a, int p) : seq(-1), i(0), first(0), last(a.width - 1) {
    if (!a.cu_seqlens) {
      seq = blockIdx.y, i = p;
      return;
    }
    if (p >= a.count) return;
    const int lane = threadIdx.x & 31;
    for (int base = 0; base < a.num_seqs; base += 32) {
      int skip = 0, n = 0;
      if (base + lane < a.num_seqs) {
        const int tokens = a.cu_seqlens[base + lane + 1] - a.cu_seqlens[base + lane], len = min(a.kv_lens[base + lane], a.max_len);
        if (tokens >= a.least && len > 0) {
          if (a.window > 0) skip = max(0, len - tokens - a.window + 1) / a.ps;
          n = (len + a.ps - 1) / a.ps - skip;
        }
      }
      int sum = n;  // pages up to and with this lane's sequence
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += y;
      }
      const uint32_t reach = __ballot_sync(0xffffffffu, sum > p);
      if (reach) {
        const int from = __ffs(reach) - 1;
        seq = base + from;
        first = __shfl_sync(0xffffffffu, skip, from);
        last = first + __shfl_sync(0xffffffffu, n, from) - 1;
        i = last - (__shfl_sync(0xffffffffu, sum, from) - 1 - p);
        return;
      }
      p -= __shfl_sync(0xffffffffu, sum, 31);
    }
  }
  // what the table says of this page, and of those in front of the first and behind the last; by one warp a page
  __device__ __forceinline__ void name(const Unpack& a, int p) const {
    if (!a.table_out) return;
    int* row = a.table_out + (long)seq * a.width;
    const int lane = threadIdx.x & 31;
    if (lane == 0 && i < a.width) row[i] = p;
    if (i == first)
      for (int j = lane; j < min(first, a.width); j += 32) row[j] = p;
    if (i == last)
      for (int j = last + 1 + lane; j < a.width; j += 32) row[j] = p;
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

// Head sizes 64, 128, 256: a warp per (page, kv head), 8 lanes a row.  Lane r of a row reads word r of every group and writes 8 channels of
// each, so that the 8 lanes' writes are one piece.  All of a page's loads (16 tokens: 8 of up to 16 bytes) are under way before the
// first is used: what bounds it is the bytes written, as long as enough warps have theirs under way.
template <typename T, int D> __global__ void __launch_bounds__(256) unpack_4bit_rows_kernel(Unpack a, T* __restrict__ k_out, T* __restrict__ v_out) {
  constexpr int G = D / 64, AT_ONCE = 8;
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, r = lane & 7;
  const long item = (long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int kvh = (int)(item % a.nkv), p = (int)(item / a.nkv);
  if (p >= (a.cu_seqlens ? a.count : a.width)) return;
  const UnpackPage at_page(a, p);
  if (at_page.seq < 0) return;
  const int place = a.cu_seqlens ? p : blockIdx.y * a.width + p;
  if (kvh == 0) at_page.name(a, place);
  int page;
  const int rows = at_page.rows(a, &page);
  const Q4Page L(D, G, a.ps);
  const unsigned char* rec = a.pages + ((long)page * a.nkv + kvh) * L.record;
  const long out_base = ((long)place * a.nkv + kvh) * a.ps * D;
  for (int first = lane >> 3; first < 2 * a.ps; first += 4 * AT_ONCE) {  // rows of keys, then of values
    uint32_t code[AT_ONCE][G], par[AT_ONCE][G];
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      const int at = first + 4 * u, is_v = at >= a.ps, row = at - is_v * a.ps;
#pragma unroll
      for (int g = 0; g < G; ++g) code[u][g] = par[u][g] = 0;
      if (at < 2 * a.ps && row < rows) {
        const unsigned char *c = rec + (is_v ? L.values : 0) + (long)row * (D / 2) + 4 * G * r, *p = rec + (is_v ? L.vpar : L.kpar) + (long)row * 4 * G;
        if constexpr (D == 64) code[u][0] = *reinterpret_cast<const uint32_t*>(c), par[u][0] = *reinterpret_cast<const uint32_t*>(p);
        if constexpr (D == 128)
          *reinterpret_cast<uint2*>(code[u]) = *reinterpret_cast<const uint2*>(c), *reinterpret_cast<uint2*>(par[u]) = *reinterpret_cast<const uint2*>(p);
        if constexpr (D == 256)
          *reinterpret_cast<uint4*>(code[u]) = *reinterpret_cast<const uint4*>(c), *reinterpret_cast<uint4*>(par[u]) = *reinterpret_cast<const uint4*>(p);
      }
    }
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      const int at = first + 4 * u, is_v = at >= a.ps, row = at - is_v * a.ps;
      if (at >= 2 * a.ps) break;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const float s = q4_s(par[u][g]), z = q4_z(par[u][g]);
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = z + (float)((code[u][g] >> (4 * e)) & 15u) * s;
        store8((is_v ? v_out : k_out) + out_base + (long)row * D + 64 * g + 8 * r, v);
      }
    }
  }
}

// Other sizes: a block per (page, kv head), a thread per word.
template <typename T> __global__ void unpack_4bit_kernel(Unpack a, int D, int G, T* __restrict__ k_out, T* __restrict__ v_out) {
  pdl_wait();
  pdl_launch_dependents();
  const int p = blockIdx.x / a.nkv, kvh = blockIdx.x % a.nkv;
  const UnpackPage at_page(a, p);
  if (at_page.seq < 0) return;
  const int place = a.cu_seqlens ? p : blockIdx.y * a.width + p;
  if (kvh == 0 && threadIdx.x < 32) at_page.name(a, place);
  int page;
  const int rows = at_page.rows(a, &page);
  const Q4Page L(D, G, a.ps);
  const unsigned char* rec = a.pages + ((long)page * a.nkv + kvh) * L.record;
  const int words = D / 8, size_words = words / G, ps = a.ps;
  const long out_base = ((long)place * a.nkv + kvh) * ps * D;
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

template <typename T> cudaError_t launch_unpack(const Unpack& a, int D, T* k_out, T* v_out, cudaStream_t stream) {
  const long items = (long)(a.cu_seqlens ? a.count : a.width) * a.nkv;
  const unsigned sequences = a.cu_seqlens ? 1 : a.num_seqs;
  if (D == 64 || D == 128 || D == 256) {
    const dim3 grid((unsigned)((items + 7) / 8), sequences);
    if (D == 64) return launch_pdl(unpack_4bit_rows_kernel<T, 64>, grid, dim3(256), 0, stream, a, k_out, v_out);
    if (D == 128) return launch_pdl(unpack_4bit_rows_kernel<T, 128>, grid, dim3(256), 0, stream, a, k_out, v_out);
    return launch_pdl(unpack_4bit_rows_kernel<T, 256>, grid, dim3(256), 0, stream, a, k_out, v_out);
  }
  return launch_pdl(unpack_4bit_kernel<T>, dim3((unsigned)items, sequences), dim3(a.ps * D / 8 >= 256 ? 256 : 128), 0, stream, a, D,
                    q4_groups(D), k_out, v_out);
}

// ---- eviction -------------------------------------------------------------------------------------------------------------------------
// Per (layer, sequence, kv head) that holds more than `keep` tokens: which tokens stay, and who fills whose place.  Stay: positions below
// `first`, the last `recent` positions, and of the others those with the largest sums until `keep` are found (equal sums: the lower
// place; NaN counts as the largest).  The tokens that go leave holes among the first `keep` places, which the tokens that stay from
// behind `keep` fill, both in order: nothing that stays in front moves, and no token's source is another's goal, so the moves are
// independent of each other.
// One block: order-preserving keys in shared memory (or scratch when they are too many), the threshold by three passes of a histogram over
// 11, 11 and 10 bits (with 8 bits the first pass meets a sum's exponent alone, and counters collide), then both lists in order: a thread
// owns neighbouring places, an odd number of them, so that threads read different banks.  What bounds it is the latency of these steps.
constexpr int EVICT_THREADS = 1024;
constexpr int EVICT_BINS = 2048;
constexpr int EVICT_KEYS = 49152;           // that one block holds in shared memory; more go through scratch
constexpr int EVICT_PLACES = 24576;         // up to here the positions fit beside them, and are read once
constexpr int EVICT_TOGETHER = 512;         // as many moves at most are made by the block that chose them: no second kernel

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
  int max_pages, num_pages, num_seqs, nkv, ps, ps_shift, keep, first, recent, cap, max_len;
  unsigned char* pages;
  int D, G, wide, fours;  // rows of codes in pieces of 16 bytes; sums and positions in fours
  float* mass;
  int* places;
  uint32_t* spill;  // null, or [pairs][max_len]: the keys when they do not fit shared memory
  int* lists;       // [pairs][1 + 2 cap]: how many, holes, movers
};

// Page and row of a place (pages of a power of two take no division).
struct EvictRow {
  int page, row;
  __device__ __forceinline__ EvictRow(const Evict& a, const int* bt, int slot) {
    const int i = a.ps_shift >= 0 ? slot >> a.ps_shift : slot / a.ps;
    row = slot - i * a.ps;
    page = bt[i];
    if ((uint32_t)page >= (uint32_t)a.num_pages) page = -1;
  }
};

// The rows of one (layer, sequence, kv head) that move: a group of 8 lanes takes four tokens at a time, so that their places, pages and
// bytes are looked up side by side.  Rows whose codes are whole pieces of 16 bytes go in those, others in words.
__device__ __forceinline__ void evict_move(const Evict& a, const int* list, int count, const int* bt, long layer_heads, int kvh, int group, int groups) {
  constexpr int AT_ONCE = 4;
  const Q4Page L(a.D, a.G, a.ps);
  const int lane = threadIdx.x & 7;
  for (int first = group * AT_ONCE; first < count; first += groups * AT_ONCE) {
    int to[AT_ONCE], from[AT_ONCE], tr[AT_ONCE], fr[AT_ONCE];
    long th[AT_ONCE], fh[AT_ONCE];
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      const bool is = first + u < count;
      to[u] = is ? list[1 + first + u] : -1;
      from[u] = is ? list[1 + a.cap + first + u] : -1;
    }
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      if (to[u] < 0) continue;
      const EvictRow t(a, bt, to[u]), f(a, bt, from[u]);
      tr[u] = t.row, fr[u] = f.row;
      th[u] = layer_heads + (long)t.page * a.nkv + kvh, fh[u] = layer_heads + (long)f.page * a.nkv + kvh;
      if (t.page < 0 || f.page < 0) to[u] = -1;
    }
    // parameters, sum and position: one word of each by lanes 0 .. 2 G + 1, the rest of them (more than three groups) below
    uint32_t word[AT_ONCE];
    uint4 piece[AT_ONCE];
    const int pieces = L.half / 16;  // of the key's codes, then as many of the value's
    auto word_at = [&](int v, long h, int row) -> uint32_t* {
      if (v >= 2 * a.G) return reinterpret_cast<uint32_t*>(v == 2 * a.G ? (void*)a.mass : (void*)a.places) + h * a.ps + row;
      const int is_v = v >= a.G;
      return reinterpret_cast<uint32_t*>(a.pages + h * L.record + (is_v ? L.vpar : L.kpar) + (long)row * L.par + 4 * (v - is_v * a.G));
    };
    auto piece_at = [&](int v, long h, int row) -> uint4* {
      const int is_v = v >= pieces;
      return reinterpret_cast<uint4*>(a.pages + h * L.record + (is_v ? L.values : 0) + (long)row * L.half + 16 * (v - is_v * pieces));
    };
    const bool first_piece = a.wide && lane < 2 * pieces, first_word = lane < 2 * a.G + 2;
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u)
      if (to[u] >= 0) {
        if (first_piece) piece[u] = *piece_at(lane, fh[u], fr[u]);
        if (first_word) word[u] = *word_at(lane, fh[u], fr[u]);
      }
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u)
      if (to[u] >= 0) {
        if (first_piece) *piece_at(lane, th[u], tr[u]) = piece[u];
        if (first_word) *word_at(lane, th[u], tr[u]) = word[u];
      }
    for (int u = 0; u < AT_ONCE; ++u) {  // what 8 lanes do not do at once
      if (to[u] < 0) continue;
      for (int v = lane + 8; v < 2 * a.G + 2; v += 8) *word_at(v, th[u], tr[u]) = *word_at(v, fh[u], fr[u]);
      if (a.wide) {
        for (int v = lane + 8; v < 2 * pieces; v += 8) *piece_at(v, th[u], tr[u]) = *piece_at(v, fh[u], fr[u]);
      } else {
        const int words = L.half / 4;
        for (int v = lane; v < 2 * words; v += 8) {
          const int is_v = v >= words;
          const long sec = (is_v ? L.values : 0) + 4 * (v - is_v * words);
          *reinterpret_cast<uint32_t*>(a.pages + th[u] * L.record + sec + (long)tr[u] * L.half) =
              *reinterpret_cast<const uint32_t*>(a.pages + fh[u] * L.record + sec + (long)fr[u] * L.half);
        }
      }
    }
  }
}

__global__ void __launch_bounds__(EVICT_THREADS, 1) evict_select_kernel(Evict a) {
  extern __shared__ uint32_t keys_s[];
  __shared__ int bins[EVICT_BINS], red[33], s_newest, s_digit, s_left;
  pdl_wait();
  pdl_launch_dependents();
  const int kvh = blockIdx.x, seq = blockIdx.y, layer = blockIdx.z;
  const long pair = ((long)layer * a.num_seqs + seq) * a.nkv + kvh;
  int* list = a.lists + pair * (1 + 2 * (long)a.cap);
  const int n = min(a.kv_lens[seq], a.max_len), tid = threadIdx.x, lane = tid & 31;
  constexpr int threads = EVICT_THREADS;
  if (n <= a.keep) {
    if (tid == 0) list[0] = 0;
    return;
  }
  uint32_t* keys = a.spill ? a.spill + pair * a.max_len : keys_s;
  int* place_s = reinterpret_cast<int*>(keys_s) + a.max_len;
  const bool kept_places = a.max_len <= EVICT_PLACES;
  const int* bt = a.block_table + (long)seq * a.max_pages;
  const long layer_heads = (long)layer * a.num_pages * a.nkv;
  if (tid == 0) s_newest = -1;
  for (int i = tid; i < EVICT_BINS; i += threads) bins[i] = 0;
  __syncthreads();
  int newest = -1;
  auto put = [&](int i, bool there, float sum, int place) {
    newest = max(newest, there ? place : -1);
    const float m = there ? sum + 0.f : -INFINITY;  // (minus zero is zero)
    uint32_t key = __float_as_uint(m);
    key = m != m ? 0xFFFFFFFEu : (key & 0x80000000u) ? ~key : key | 0x80000000u;
    keys[i] = there && place < a.first ? 0xFFFFFFFFu : key;
    if (kept_places) place_s[i] = there ? place : INT_MIN;
  };
  if (a.fours) {  // four neighbours lie in one page, at a multiple of 16 bytes
    for (int i = 4 * tid; i < n; i += 4 * threads) {
      const EvictRow at(a, bt, i);
      float4 m = make_float4(0.f, 0.f, 0.f, 0.f);
      int4 p = make_int4(0, 0, 0, 0);
      if (at.page >= 0) {
        const long c = (layer_heads + (long)at.page * a.nkv + kvh) * a.ps + at.row;
        m = *reinterpret_cast<const float4*>(a.mass + c);
        p = *reinterpret_cast<const int4*>(a.places + c);
      }
      put(i, at.page >= 0, m.x, p.x);
      if (i + 1 < n) put(i + 1, at.page >= 0, m.y, p.y);
      if (i + 2 < n) put(i + 2, at.page >= 0, m.z, p.z);
      if (i + 3 < n) put(i + 3, at.page >= 0, m.w, p.w);
    }
  } else {
    for (int i = tid; i < n; i += threads) {
      const EvictRow at(a, bt, i);
      const long c = (layer_heads + (long)at.page * a.nkv + kvh) * a.ps + at.row;
      put(i, at.page >= 0, at.page >= 0 ? a.mass[c] : 0.f, at.page >= 0 ? a.places[c] : 0);
    }
  }
  newest = __reduce_max_sync(0xffffffffu, newest);
  if (lane == 0) atomicMax(&s_newest, newest);
  __syncthreads();
  newest = s_newest;
  // the keep-th largest key; the first pass makes the newest positions' keys on its way
  uint32_t prefix = 0, mask = 0;
  int left = a.keep;  // how many of those that share the prefix stay
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
    for (int i = tid; i < n; i += threads) {
      uint32_t key = keys[i];
      if (pass == 0 && a.recent > 0) {
        int place;
        if (kept_places) {
          place = place_s[i];
        } else {
          const EvictRow at(a, bt, i);
          place = at.page < 0 ? INT_MIN : a.places[(layer_heads + (long)at.page * a.nkv + kvh) * a.ps + at.row];
        }
        if (place > newest - a.recent && place != INT_MIN) keys[i] = key = 0xFFFFFFFFu;
      }
      if ((key & mask) == prefix) atomicAdd(&bins[(key >> shift) & ((1 << bits) - 1)], 1);
    }
    __syncthreads();
    // from the largest digit down: thread t holds `per_bin` of them, the first EVICT_BINS - 1 - t * per_bin
    const int per_bin = EVICT_BINS / threads;
    int own = 0, all;
    for (int e = 0; e < per_bin; ++e) own += bins[EVICT_BINS - 1 - tid * per_bin - e];
    int before = block_scan(own, &all, red);
    if (before < left && left <= before + own) {
      for (int e = 0; e < per_bin; ++e) {
        const int d = EVICT_BINS - 1 - tid * per_bin - e;
        if (before + bins[d] >= left) {
          s_digit = d;
          s_left = left - before;
          break;
        }
        before += bins[d];
      }
    }
    __syncthreads();
    prefix |= (uint32_t)s_digit << shift;
    mask |= ((1u << bits) - 1) << shift;
    left = s_left;
    for (int i = tid; i < EVICT_BINS; i += threads) bins[i] = 0;
    __syncthreads();
  }
  // holes in front, movers behind, in order; of the keys equal to the threshold the first `left` stay
  const int per = ((n + threads - 1) / threads) | 1;
  const int begin = min(n, tid * per), end = min(n, begin + per);
  int ties = 0, all;
  for (int i = begin; i < end; ++i) ties += keys[i] == prefix;
  const int ties_before = block_scan(ties, &all, red);
  auto walk = [&](auto&& hole, auto&& mover) {
    int rank = ties_before;
    for (int i = begin; i < end; ++i) {
      const uint32_t key = keys[i];
      const bool stays = key > prefix || (key == prefix && rank < left);
      rank += key == prefix;
      if (i < a.keep && !stays) hole(i);
      if (i >= a.keep && stays) mover(i);
    }
  };
  int holes = 0, movers = 0, count;
  walk([&](int) { ++holes; }, [&](int) { ++movers; });
  // (there are as many of the one as of the other, so the movers' total is the holes')
  holes = block_scan(holes, &count, red);
  movers = block_scan(movers, &count, red);
  walk([&](int i) { list[1 + holes++] = i; }, [&](int i) { list[1 + a.cap + movers++] = i; });
  if (a.cap <= EVICT_TOGETHER) {
    __syncthreads();  // (orders the block's writes of the list, too)
    evict_move(a, list, count, bt, layer_heads, kvh, tid >> 3, threads >> 3);
  } else if (tid == 0) {
    list[0] = count;
  }
}

__global__ void __launch_bounds__(256) evict_move_kernel(Evict a) {
  pdl_wait();
  pdl_launch_dependents();
  const int kvh = blockIdx.y % a.nkv, seq = blockIdx.y / a.nkv, layer = blockIdx.z;
  const long pair = ((long)layer * a.num_seqs + seq) * a.nkv + kvh;
  const int* list = a.lists + pair * (1 + 2 * (long)a.cap);
  evict_move(a, list, list[0], a.block_table + (long)seq * a.max_pages, (long)layer * a.num_pages * a.nkv, kvh,
             blockIdx.x * (blockDim.x >> 3) + (threadIdx.x >> 3), gridDim.x * (blockDim.x >> 3));
}

inline bool q4_aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

Q3_EXPORT int q3_store_4bit(int dtype, const void* qkv, int row_stride, void* q_out, int q_stride, int nq, int nkv, int D, const float* q_w,
                            const float* k_w, float eps, const float* cos_t, const float* sin_t, int rot_half, int max_pos,
                            const int* positions, const int* slots, const int* token_seq, const int* block_table, int max_pages,
                            int num_seqs, void* pages, int num_pages, int ps, int num_tokens, int write_kv, int pairing, float* mass,
                            int* places, int* error_word, cudaStream_t stream) {
  if (num_tokens < 1) return Q3_OK;  // (tensors of nothing have no address)
  if (!qkv || !q_out || !positions || nq < 1 || nkv < 1 || pairing < 0 || pairing > 1 || !q4_sizes_ok(D, ps)) return Q3_ERR_ARGUMENT;
  if (cos_t && (max_pos < 1 || !sin_t || rot_half < 1 || 2 * rot_half > D)) return Q3_ERR_ARGUMENT;
  if (write_kv && (!token_seq || !block_table || !pages || max_pages < 1)) return Q3_ERR_ARGUMENT;
  if (dtype != Q3_DTYPE_F32 && dtype != Q3_DTYPE_BF16) return Q3_ERR_ARGUMENT;
  if (write_kv && !q4_aligned(pages)) return Q3_ERR_UNSUPPORTED;
  Store a{q_w, k_w, cos_t, sin_t, eps, rot_half, max_pos, pairing, positions, slots, token_seq, block_table,
          max_pages, num_pages, num_seqs, ps, write_kv, (unsigned char*)pages, mass, places, error_word};
  const int G = q4_groups(D), tph = D / 16;
  const bool vec = (tph & (tph - 1)) == 0 && row_stride % 8 == 0 && q_stride % 8 == 0 && (!cos_t || 2 * rot_half == D) &&
                   q4_aligned(qkv) && q4_aligned(q_out) && q4_aligned(q_w) && q4_aligned(k_w) && q4_aligned(cos_t) && q4_aligned(sin_t);
  cudaError_t err;
  if (vec) {
    const int threads = 128, per_token = (write_kv ? nq + 2 * nkv : nq) * tph;
    const dim3 grid((unsigned)num_tokens, (unsigned)((per_token + threads - 1) / threads));
    if (grid.y > 65535) return Q3_ERR_UNSUPPORTED;
    auto launch = [&](auto known) {
      constexpr int K = decltype(known)::value;
      err = dtype == Q3_DTYPE_F32 ? launch_pdl(store_4bit_vec_kernel<float, K>, grid, dim3(threads), 0, stream, (const float*)qkv, row_stride,
                                               (float*)q_out, q_stride, nq, nkv, D, a)
                                  : launch_pdl(store_4bit_vec_kernel<bf16, K>, grid, dim3(threads), 0, stream, (const bf16*)qkv, row_stride,
                                               (bf16*)q_out, q_stride, nq, nkv, D, a);
    };
    if (D == 64)
      launch(std::integral_constant<int, 64>());
    else if (D == 128)
      launch(std::integral_constant<int, 128>());
    else if (D == 256)
      launch(std::integral_constant<int, 256>());
    else
      launch(std::integral_constant<int, 0>());
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

// `cu_seqlens` null: num_seqs * width pages are written; else `count` pages (struct Unpack).
Q3_EXPORT int q3_unpack_4bit(int dtype, const void* pages, int num_pages, int nkv, int D, int ps, const int* block_table, int max_pages,
                             const int* kv_lens, int num_seqs, int max_len, const int* cu_seqlens, int least, int window, int count, int width,
                             void* k_out, void* v_out, int* table_out, cudaStream_t stream) {
  if (num_seqs < 1 || width < 1 || (cu_seqlens && count < 1)) return Q3_OK;
  if (!pages || !block_table || !kv_lens || !k_out || !v_out || nkv < 1 || max_pages < 1 || !q4_sizes_ok(D, ps)) return Q3_ERR_ARGUMENT;
  if (cu_seqlens && (!table_out || least < 1)) return Q3_ERR_ARGUMENT;
  if (dtype != Q3_DTYPE_F32 && dtype != Q3_DTYPE_BF16) return Q3_ERR_ARGUMENT;
  if ((!cu_seqlens && num_seqs > 65535) || !q4_aligned(pages) || !q4_aligned(k_out) || !q4_aligned(v_out)) return Q3_ERR_UNSUPPORTED;
  if ((long)(cu_seqlens ? count : width) * nkv > 0x7fffffffL) return Q3_ERR_UNSUPPORTED;
  const Unpack a{(const unsigned char*)pages, num_pages, nkv, ps, block_table, kv_lens, cu_seqlens, max_pages, num_seqs, max_len, least, window,
                 count, width, table_out};
  const cudaError_t err = dtype == Q3_DTYPE_F32 ? launch_unpack(a, D, (float*)k_out, (float*)v_out, stream)
                                                : launch_unpack(a, D, (bf16*)k_out, (bf16*)v_out, stream);
  return err == cudaSuccess ? Q3_OK : Q3_ERR_LAUNCH;
}

// `lists`: [layers * sequences * kv heads][1 + 2 cap] ints; `spill`: the same times max_len, for more than EVICT_KEYS tokens.
Q3_EXPORT int q3_evict_4bit(void* pages, int num_layers, int num_pages, int nkv, int D, int ps, float* mass, int* places,
                            const int* block_table, int max_pages, const int* kv_lens, int num_seqs, int max_len, int keep, int first,
                            int recent, int cap, void* spill, int* lists, cudaStream_t stream) {
  if (num_seqs < 1 || num_layers < 1 || max_len <= keep) return Q3_OK;
  if (!pages || !mass || !places || !block_table || !kv_lens || !lists || nkv < 1 || max_pages < 1 || !q4_sizes_ok(D, ps))
    return Q3_ERR_ARGUMENT;
  if (keep < 1 || first < 0 || recent < 0 || (long)first + recent > keep || cap < 1 || max_len > (long)max_pages * ps) return Q3_ERR_ARGUMENT;
  if (max_len > EVICT_KEYS && !spill) return Q3_ERR_ARGUMENT;
  if (cap < (keep < max_len - keep ? keep : max_len - keep)) return Q3_ERR_ARGUMENT;
  if (num_seqs > 65535 || num_layers > 65535 || (long)num_seqs * nkv > 65535 || !q4_aligned(pages)) return Q3_ERR_UNSUPPORTED;
  int shift = 0;
  while ((1 << shift) < ps) ++shift;
  Evict a{block_table, kv_lens, max_pages, num_pages, num_seqs, nkv, ps, (1 << shift) == ps ? shift : -1, keep, first, recent, cap, max_len,
          (unsigned char*)pages, D, q4_groups(D), (D / 2) % 16 == 0, ps % 4 == 0 && q4_aligned(mass) && q4_aligned(places), mass, places, max_len > EVICT_KEYS ? (uint32_t*)spill : nullptr, lists};
  static bool once[Q3_MAX_DEVICES];
  const int dev = q3_current_device();
  if (!once[dev]) {
    if (cudaFuncSetAttribute(evict_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 4 * EVICT_KEYS) != cudaSuccess)
      return Q3_ERR_LAUNCH;
    once[dev] = true;
  }
  const size_t smem = a.spill ? 0 : (max_len <= EVICT_PLACES ? 8 : 4) * (size_t)max_len;
  cudaError_t err = launch_pdl(evict_select_kernel, dim3(nkv, num_seqs, num_layers), dim3(EVICT_THREADS), smem, stream, a);
  if (err != cudaSuccess) return Q3_ERR_LAUNCH;
  if (cap <= EVICT_TOGETHER) return Q3_OK;
  // 128 tokens a block at a time, about eight blocks an SM
  const long pairs = (long)num_seqs * nkv * num_layers;
  long chunks = (cap + 127) / 128, most = (148 * 8 + pairs - 1) / pairs;
  if (chunks > most) chunks = most;
  err = launch_pdl(evict_move_kernel, dim3((unsigned)chunks, (unsigned)(num_seqs * nkv), (unsigned)num_layers), dim3(256), 0, stream, a);
  return err == cudaSuccess ? Q3_OK : Q3_ERR_LAUNCH;
}
