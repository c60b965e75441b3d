// Prompts over unpacked tiles, heads of 64 to 128: prompts_tiles.cuh.  (Apart from heads of more: both forms in one library, and this one is 4 % slower.)
#include "prompts_tiles.cuh"

Q3_EXPORT int q3_prompts_tiles_8bit(const void* q, int q_stride, int num_tokens, const void* k, const void* v, int tiles, void* items, int num_items, void* out,
                                    int nq, int nkv, int head_dim, float scale, int window, int keep_first, int splits, float* mid_o, float* mid_ml,
                                    const int* cu_seqlens, int num_seqs, int least, int* error_word, cudaStream_t stream) {
  return launch_tiles<false>(q, q_stride, num_tokens, k, v, tiles, items, num_items, out, nq, nkv, head_dim, scale, window, keep_first, splits, mid_o, mid_ml,
                             cu_seqlens, num_seqs, least, error_word, stream);
}
