/*
 * ie_logprobs.h — C ABI of log probabilities: of given tokens, with their
 * ranks, the rows' entropies and the top alternatives.  Conventions as
 * ie_amd.h.  The reference has the softmax of its sampler only
 * (src/sampler.cu:28-36, over the k selected logits on the host).
 */
#ifndef IE_LOGPROBS_H
#define IE_LOGPROBS_H

#include "ie_amd.h"
#include "ie_engine.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Most alternatives per row, and the widest row. */
#define IE_LOGPROBS_TOP_MAX 128
#define IE_LOGPROBS_N_MAX (1 << 19)

/* Bytes of workspace that a call of this size needs (0: it needs none). */
size_t ie_token_logprobs_workspace_bytes(int rows, int n, int k);

/* For each row r of logits [rows, n] fp32, rows row_stride >= n floats apart
 * (columns n and on are not read), with p = softmax(logits[r, 0:n]):
 *   logprobs[r] = log p[targets[r]], ranks[r] = 1 + the number of tokens ahead
 *     of it (a larger logit, or an equal one at a lower index); a target of -1
 *     asks for none and gets 0 and 0 (as do all rows where targets is NULL),
 *     any other outside [0, n) NaN and 0;
 *   entropy[r] = -sum p log p (natural logarithm, 0 log 0 = 0);
 *   top_logprobs / top_idx [rows, k]: the k largest by value descending, equal
 *     values by index ascending (+0 and -0 are equal), as ie_topk's; 0 <= k <=
 *     min(n, IE_LOGPROBS_TOP_MAX).
 * logprobs, ranks and entropy may each be NULL.  A logit of -inf has
 * probability 0 (log probability -inf, as has one below fp32's range); a row
 * of nothing else has log probabilities -inf and entropy 0.  A row that holds
 * NaN or +inf has NaN log probabilities and entropy, and its ranks and indices
 * say nothing (the indices lie in [0, n)).  n <= IE_LOGPROBS_N_MAX.  Sums are
 * fp32 over a fixed order: a repeated call repeats its bits.  A workspace
 * serves one call at a time: calls that may run at once (on two streams, from
 * two replayed graphs) take one each. */
int ie_token_logprobs(int rows, const float* logits, int row_stride, int n, const int* targets,
                      int k, float* logprobs, int* ranks, float* entropy, float* top_logprobs,
                      int* top_idx, float* workspace, size_t workspace_bytes, ie_stream_t stream);

/* Scores tokens with the engine (GPT2Engine::score): prefill of tokens [batch,
 * prompt_len] (host) at the current position; entry [b, t] of the host arrays
 * [batch, prompt_len] is the log probability of tokens[b, t + 1] after the ones
 * before it, its rank, and the entropy and the k most likely tokens [batch,
 * prompt_len, k] of that prediction.  The last entry of a sequence has no token
 * to score (0 and rank 0).  Any array may be NULL. */
int ie_engine_score(ie_engine* e, int batch, int prompt_len, const int* tokens, int k,
                    float* logprobs, int* ranks, float* entropy, float* top_logprobs, int* top_idx);

#ifdef __cplusplus
}
#endif
#endif
