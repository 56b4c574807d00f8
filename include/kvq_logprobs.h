/*
 * kvq_logprobs.h -- C ABI of the log probabilities of given tokens, with the entropy and the likeliest
 * tokens of each row of logits.
 *
 * The rules of kvq.h hold: plain device pointers, nothing allocates or synchronises, the work goes
 * to `stream`, KVQ_OK or a KVQ_ERR_* code with kvq_last_error().  The reference takes an argmax of its
 * logits and no more (src/engine/generate_loop.py).
 */
#ifndef KVQ_LOGPROBS_H_
#define KVQ_LOGPROBS_H_

#include "kvq.h"

#ifdef __cplusplus
extern "C" {
#endif

#define KVQ_LOGITS_F16 0
#define KVQ_LOGITS_BF16 1
#define KVQ_LOGITS_F32 2

#define KVQ_LOGPROBS_MAX_TOP 32

/* With p = softmax(inv_temperature * logits[i, :vocab]):  logprobs[i] = log p[tokens[i]] (NaN for a token outside
 * [0, vocab)), entropy[i] = -sum p log p, and the `top` tokens of the largest logits, the lower token first among
 * equal ones, NaN below all, with their log p.  A row whose softmax is none (a NaN, a +Inf, nothing but -Inf) has
 * NaN for its values. */
typedef struct kvq_token_logprobs_params {
  const void* logits;         /* [rows, vocab] of logits_type, vocab contiguous, aligned to its elements */
  int64_t row_stride;         /* elements */
  const void* tokens;         /* [rows] int32 or int64; NULL: logprobs is not written */
  float* logprobs;            /* fp32 [rows] */
  float* entropy;             /* fp32 [rows] */
  float* top_logprobs;        /* fp32 [rows, top] */
  int64_t* top_tokens;        /* int64 [rows, top] */
  void* workspace;            /* kvq_token_logprobs_workspace_bytes(), any contents, 16-byte aligned */
  int64_t workspace_bytes;
  int64_t rows;
  int32_t vocab;
  int32_t top;                /* at most vocab and KVQ_LOGPROBS_MAX_TOP */
  int32_t logits_type;
  int32_t tokens64;           /* tokens are int64 */
  float inv_temperature;      /* 1e-30 to 1e30 */
  int32_t reserved;           /* 0 */
} kvq_token_logprobs_params;
int kvq_token_logprobs(const kvq_token_logprobs_params* p, kvq_stream_t stream);
int64_t kvq_token_logprobs_workspace_bytes(const kvq_token_logprobs_params* p);

#ifdef __cplusplus
}
#endif
#endif /* KVQ_LOGPROBS_H_ */
