/*
 * C ABI of log probabilities over rows of logits, in the same library and with
 * the same conventions as nvm_moe.h: device pointers, work on `stream`, no
 * host synchronisation, no device allocation (callers pass outputs and the
 * workspace), NVM_OK or a negative NVM_ERR_* status (message in
 * nvm_last_error()).
 */
#ifndef NVM_LOGPROBS_H
#define NVM_LOGPROBS_H

#include "nvm_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Types of logits (the codes of nvm_kv_dtype). */
enum nvm_logits_dtype { NVM_LOGITS_F16 = 0, NVM_LOGITS_BF16 = 1, NVM_LOGITS_F32 = 2 };

enum { NVM_MAX_TOP_LOGPROBS = 64 };

/*
 * Of each of N rows of V logits (rows ld values apart, of `dtype`), with p =
 * softmax(row):
 *   logprobs      [N] float32: log p of token tokens[n]; 0 for a token outside
 *                 [0, V), which so adds nothing to a sum over a sequence
 *   entropy       [N] float32: -sum p log p (a probability of zero adds zero)
 *   top_ids,
 *   top_logprobs  [N, top_k] int64 and float32: the top_k largest logits in
 *                 descending order, equal ones by ascending id, and their log p
 * tokens [N] int64; top_k from 0 (both top outputs may then be NULL) to the
 * smaller of V and NVM_MAX_TOP_LOGPROBS.  Sums are float32 of few terms and
 * float64 beyond, rounded to float32 once; the largest logit's term is exactly 1
 * and summed in float64, so that results next to zero (a token that is all but
 * certain) are no less exact than others.  A row with a NaN or +infinity, or
 * of -infinities only, has NaN log probabilities (but for tokens outside) and
 * entropy; among the largest logits a NaN is the first.  V below 2^31 - 64, N below
 * 2^24.  Rows are read in aligned pieces of 16 bytes, so up to 15 bytes around one
 * are, too.
 * Workspace: nvm_token_logprobs_workspace_size, on the device that the call
 * runs on (zero bytes if no row is split; workspace may then be NULL).
 */
int nvm_token_logprobs_workspace_size(int64_t N, int64_t V, int dtype, int top_k, size_t *bytes);
int nvm_token_logprobs(const void *logits, int64_t N, int64_t V, int64_t ld, int dtype,
                       const int64_t *tokens, int top_k, float *logprobs, float *entropy,
                       int64_t *top_ids, float *top_logprobs, void *workspace,
                       size_t workspace_bytes, nvm_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* NVM_LOGPROBS_H */
