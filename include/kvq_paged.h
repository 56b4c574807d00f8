/*
 * kvq_paged.h -- C ABI of the paged cache: append, one-token attention, windowed prompt
 * attention and eviction.
 *
 * A layer's cache is a pool of pages.  A page holds page_size token slots of every KV head; token
 * t of row b lies in page table[b][t / page_size] at slot t % page_size.  Rows of a batch have
 * lengths of their own, and a page may serve several rows as long as nothing writes to it.
 *
 * The rules of kvq.h hold: plain device pointers, nothing allocates or synchronises, the work goes
 * to `stream`, KVQ_OK or a KVQ_ERR_* code with kvq_last_error().  Lengths, positions and page
 * numbers are device memory that the host does not read: lengths are clamped to the table's
 * columns, and a page number outside [0, num_pages) stands for a page that is not there (its
 * tokens are left out of the attention, nothing is written to it, and a row that has one is not
 * evicted).  Pages that are written (append, eviction) need memory of their own: a stride of 0 between
 * them, or between heads, is refused.  No counterpart in the reference, whose caches are dense.
 */
#ifndef KVQ_PAGED_H_
#define KVQ_PAGED_H_

#include "kvq.h"

#ifdef __cplusplus
extern "C" {
#endif

/* element types of activations and of pages that hold them as they are */
#define KVQ_PAGED_F16 0
#define KVQ_PAGED_BF16 1
/* pages of int8 codes with an fp16 scale per (token, group): value = code * scale */
#define KVQ_PAGED_INT8 2

/* One layer's pages and the rows' page tables.  K and V rows are 128 values, contiguous; strides
 * are in bytes, multiples of 16, as are the base addresses. */
typedef struct kvq_paged_cache {
  void* k;
  void* v;
  int64_t k_stride_p, k_stride_h, k_stride_t; /* bytes between pages, heads, tokens */
  int64_t v_stride_p, v_stride_h, v_stride_t;
  void* k_scale;              /* INT8: fp16 [num_pages, heads, page_size, 128 / group_size], the last */
  void* v_scale;              /* two dimensions dense, 16-byte aligned pages; else NULL */
  int64_t ks_stride_p, ks_stride_h, vs_stride_p, vs_stride_h; /* bytes, multiples of 16 */
  const int32_t* table;       /* device int32 [batch, max_pages] */
  int64_t table_stride;       /* elements between rows */
  int32_t num_pages, max_pages;
  int32_t page_size;          /* 16, 32, 64, 128 or 256 */
  int32_t format;             /* KVQ_PAGED_* */
  int32_t group_size;         /* INT8: 32, 64 or 128 */
  int32_t batch, kv_heads;
  int32_t reserved;           /* 0 */
} kvq_paged_cache;

/* Appends k, v [B, heads, seq_new, 128] (16-bit elements of type x_type, strides in elements): token i
 * of row b goes to slot write_pos[b] + i for i < new_lens[b] (NULL: seq_new); slots at or past
 * max_pages * page_size are not written.  INT8: scale = fp16(min(max(absmax, 1e-5) / 127, 65504)),
 * code = clamp(rne(fp16(x / scale)), -127, 127), as INT8KVCache at percentile 100
 * (src/quant/int8_basic.py:18-108); a group with a NaN or Inf gets the scale NaN and codes 0. */
typedef struct kvq_paged_append_params {
  kvq_paged_cache cache;
  const void* k;
  const void* v;
  int64_t k_stride_b, k_stride_h, k_stride_s, v_stride_b, v_stride_h, v_stride_s;
  const int32_t* write_pos;
  const int32_t* new_lens;
  int32_t seq_new;
  int32_t x_type;             /* KVQ_PAGED_F16 or _BF16; the pages' own type unless they are INT8 */
} kvq_paged_append_params;
int kvq_paged_append(const kvq_paged_append_params* p, kvq_stream_t stream);

/* Attention of one query token a row: with n = context_lens[b], query head h sees token t of its KV
 * head where t < n and (window <= 0 or t >= n - window or t < sinks);
 *   out[b,h] = softmax_t(sm_scale * inv_tau[h] * q[b,h] . k_t) @ v_t,   0 where it sees nothing.
 * weights (fp32 [B, kv_heads, >= max_pages * page_size] or NULL): weights[b,g,t] += the sum of the
 * softmax over the query heads of KV head g. */
typedef struct kvq_paged_decode_params {
  kvq_paged_cache cache;
  const void* q;              /* [B, q_heads, 128] of q_type, strides in elements, multiples of 8 */
  int64_t q_stride_b, q_stride_h;
  void* out;                  /* [B, q_heads, 128] of q_type, dense */
  const int32_t* context_lens;
  const float* inv_tau;       /* fp32 [q_heads] or NULL */
  float* weights;
  int64_t w_stride_b, w_stride_h; /* elements */
  void* workspace;            /* kvq_paged_decode_workspace_bytes(), any contents, 16-byte aligned */
  int64_t workspace_bytes;
  float sm_scale;
  int32_t window, sinks;
  int32_t q_heads;            /* a multiple of kv_heads, at most 16 times */
  int32_t q_type;
  int32_t reserved;           /* 0 */
} kvq_paged_decode_params;
int kvq_paged_decode(const kvq_paged_decode_params* p, kvq_stream_t stream);
int64_t kvq_paged_decode_workspace_bytes(const kvq_paged_decode_params* p);

/* Attention of a prompt, or of a chunk of one: query i of row b, i < q_lens[b] (NULL: seq_q), stands at
 * position m = kv_lens[b] - q_lens[b] + i (kv_lens NULL: seq_kv) and sees key j where j <= m and (window
 * <= 0 or j > m - window or j < sinks).  Queries that see nothing, and those at or past q_lens[b], are 0. */
typedef struct kvq_prefill_params {
  const void* q;              /* [B, q_heads, seq_q, 128], strides in elements, multiples of 8 */
  const void* k;              /* [B, kv_heads, seq_kv, 128] */
  const void* v;
  int64_t q_stride_b, q_stride_h, q_stride_s;
  int64_t k_stride_b, k_stride_h, k_stride_s;
  int64_t v_stride_b, v_stride_h, v_stride_s;
  void* out;                  /* [B, q_heads, seq_q, 128] */
  int64_t o_stride_b, o_stride_h, o_stride_s;
  const int32_t* q_lens;
  const int32_t* kv_lens;
  const float* inv_tau;       /* fp32 [q_heads] or NULL */
  void* workspace;            /* kvq_prefill_workspace_bytes(), any contents, 16-byte aligned */
  int64_t workspace_bytes;
  float sm_scale;
  int32_t batch, q_heads, kv_heads, seq_q, seq_kv;
  int32_t window, sinks;
  int32_t type;               /* KVQ_PAGED_F16 or _BF16, of q, k, v and out */
  int32_t reserved;           /* 0 */
} kvq_prefill_params;
int kvq_prefill_attn(const kvq_prefill_params* p, kvq_stream_t stream);
int64_t kvq_prefill_workspace_bytes(const kvq_prefill_params* p);

/* Cuts every row of more than `budget` tokens down to `budget`, per KV head: the first `sinks`, the last
 * `recent` and, of the others, those of the largest weight (NaN counts as the lowest, equal weights go to
 * the lower token).  Kept tokens move, in order, to slots 0 .. budget - 1; slots behind are left as they
 * were.  new_lens [B], kept [B, kv_heads, budget] (old token of each slot, -1 behind the row's last) and
 * new_weights [B, kv_heads, w_tokens] dense (0 behind the row's last) are written.  Rows of at most
 * budget tokens, and rows with a page that is not there, keep their tokens; no page may serve two rows, or
 * two places of one.  budget and w_tokens are at most 2^30. */
typedef struct kvq_paged_evict_params {
  kvq_paged_cache cache;
  const int32_t* context_lens;
  const float* weights;       /* fp32 [B, kv_heads, w_tokens], tokens contiguous */
  int64_t w_stride_b, w_stride_h; /* elements */
  int32_t* new_lens;
  int32_t* kept;
  float* new_weights;
  int32_t w_tokens;           /* at least max_pages * page_size */
  int32_t budget, sinks, recent; /* sinks + recent <= budget */
} kvq_paged_evict_params;
int kvq_paged_evict(const kvq_paged_evict_params* p, kvq_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* KVQ_PAGED_H_ */
