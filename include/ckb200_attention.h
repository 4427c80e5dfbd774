/* Paged attention library (lib/attention/libkernel.so) on B200 (sm_100a). Conventions as in ckb200_softmax.h. */
#ifndef CKB200_ATTENTION_H
#define CKB200_ATTENTION_H

#include <cuda_runtime.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Bytes of device workspace that ckb_attention_paged_launch needs for these sizes (the lengths themselves do not
 * matter), or -1 where it would reject them. */
long long ckb_attention_workspace(long long batch, int tokens, int q_heads, int kv_heads, int head_dim, int block_size,
                                  long long table_width, long long shared_prefix);

/* Attention of `tokens` new tokens of each of `batch` sequences over the paged cache that ckb_rope_kv_cache_launch
 * writes: q is a [batch, tokens, q_heads, head_dim] view (q_strides, host memory: its batch, token and head strides in
 * elements, multiples of 8; contiguous last dim), key_cache / value_cache [num_blocks, block_size, kv_heads, head_dim],
 * all of dtype 1 (bf16) or 2 (fp16) and 16-byte aligned; tables int64 [batch, table_width] the blocks of each sequence
 * in order (a block id outside the cache reads as zeros); lens int64 [batch] the tokens of each sequence, its new ones
 * included (clamped to [0, table_width * block_size]). Token t of sequence b sees the positions below lens[b] - tokens
 * + t + 1; out [batch, tokens, q_heads, head_dim] (contiguous) = softmax(scale * q . k) v over them, zeros where there
 * are none. q head h reads kv head h / (q_heads / kv_heads). shared_prefix: a multiple of block_size; the first
 * shared_prefix tokens are the same blocks for the whole batch and are read once for all, through the row of tables of
 * the first sequence all of whose new tokens see them (shorter ones, padded rows among them, through their own row: a
 * row's entries behind its length are not looked at).
 * head_dim a multiple of 8, at most 256; batch at most 4096. work: the workspace (16-byte aligned, contents do not
 * matter before and after). No counterpart in the reference. */
int ckb_attention_paged_launch(const void* q, const void* key_cache, const void* value_cache, const void* tables,
                               const void* lens, void* out, void* work, long long work_bytes,
                               const long long* q_strides, long long batch, int tokens, int q_heads, int kv_heads,
                               int head_dim, long long num_blocks, int block_size, long long table_width,
                               long long shared_prefix, float scale, int dtype, cudaStream_t stream);

/* Bounded-wait status of the kernels since the last reset: 0 fine, 1 a wait for a copy gave up after 2 s (that launch's
 * output is void), negative a cudaError_t from reading it. Synchronises the device. */
int ckb_attention_status(int reset);

#ifdef __cplusplus
}
#endif
#endif
