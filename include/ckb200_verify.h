/* Draft verification library (lib/verify/libkernel.so) on B200 (sm_100a). Conventions as in ckb200_softmax.h. */
#ifndef CKB200_VERIFY_H
#define CKB200_VERIFY_H

#include <cuda_runtime.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Speculative sampling from given random numbers, one cluster of CTAs per sequence. For each of `batch` sequences with
 * n = counts[b] (int64, clamped to [0, drafts]; counts null: drafts) drafted tokens (int64 [batch, drafts]), target
 * probabilities [batch, drafts + 1, vocab] and draft probabilities [batch, drafts, vocab] of dtype 0 (fp32) or 1 (bf16)
 * (draft null: all of a row's mass is on its drafted token), and uniforms fp32 [batch, drafts + 1] in [0, 1):
 *   token i is accepted when uniforms[i] * q_i(token) < p_i(token) and it lies in [0, vocab);
 *   after the first refusal at a the next token is drawn from max(p_a - q_a, 0) (all zero: from p_a), with all n
 *   accepted from p_n: the first column whose running sum exceeds uniforms[drafts] times the whole sum (64-bit sums).
 * out int64 [batch, drafts + 1]: the accepted tokens, the drawn one (-1 where its row has no mass), then -1; accepted
 * int64 [batch]. Probabilities that are NaN or negative count as 0. Strides (batch and row, in elements) with a
 * contiguous last dim; the other tensors are contiguous. vocab <= 2^30, drafts < 2^20. Needs no workspace. No counterpart in the reference. */
int ckb_verify_launch(const void* target, const void* draft, const void* tokens, const void* counts,
                      const float* uniforms, void* out, void* accepted, long long target_batch, long long target_row,
                      long long draft_batch, long long draft_row, long long batch, int drafts, int vocab, int dtype,
                      cudaStream_t stream);

#ifdef __cplusplus
}
#endif
#endif
