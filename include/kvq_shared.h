/*
 * kvq_shared.h -- C ABI of what several answers from one prompt need on the paged cache of
 * kvq_paged.h: copies of pages (a fork's last page, a pool's compaction) and one-token attention of
 * rows that share their first tokens.
 *
 * The rules of kvq.h hold: plain device pointers, nothing allocates or synchronises, the work goes
 * to `stream`, KVQ_OK or a KVQ_ERR_* code with kvq_last_error().  Lengths and page numbers are device
 * memory that the host does not read; a page number outside its pool stands for a page that is not
 * there.  No counterpart in the reference, whose caches are dense and have one owner a row.
 */
#ifndef KVQ_SHARED_H_
#define KVQ_SHARED_H_

#include "kvq_paged.h"

#ifdef __cplusplus
extern "C" {
#endif

/* One tensor of pages [num_pages, heads, page_size, row]: rows of row_bytes (a power of two, 2 to
 * 1024), contiguous; strides in bytes.  Rows of less than 16 bytes are dense over the tokens; the base and
 * the other strides are multiples of 16. */
typedef struct kvq_page_pool {
  void* base;
  int64_t stride_p, stride_h, stride_t;
  int32_t row_bytes;
  int32_t reserved;           /* 0 */
} kvq_page_pool;

/* Of every pool, to[dst[i]][:, :lens[i]] = from[src[i]][:, :lens[i]] for i < pairs (lens NULL: whole pages;
 * clamped to [0, page_size]); the slots behind are left as they were.  Pairs with a page that is not there
 * are left out.  No page may be written twice, or written and read by two pairs. */
typedef struct kvq_copy_pages_params {
  const kvq_page_pool* from;  /* host memory, n_pools of each */
  const kvq_page_pool* to;
  const int32_t* src;         /* device int32 [pairs] */
  const int32_t* dst;
  const int32_t* lens;
  int32_t n_pools, pairs;
  int32_t page_size, heads;   /* page_size 16, 32, 64, 128 or 256 */
  int32_t from_pages, to_pages;
} kvq_copy_pages_params;
int kvq_copy_pages(const kvq_copy_pages_params* p, kvq_stream_t stream);

/* How rows that share their first tokens are worked on.  Rows of a batch stand in groups, one behind the
 * other: group g has sizes[g] >= 1 rows, whose first lens[g] tokens are those of the group's first row.
 * kvq_shared_plan() (host work only) fills `info` and, where `words` is given, info->words int32 of it (as many as
 * `capacity` holds): the plan, for device memory.  It holds for any pages and contexts. */
typedef struct kvq_shared_plan_info {
  int32_t rows, units, slots, words;
} kvq_shared_plan_info;
int kvq_shared_plan(const int32_t* sizes, const int32_t* lens, int32_t groups, int32_t q_heads, int32_t kv_heads,
                    kvq_shared_plan_info* info, int32_t* words, int64_t capacity);

/* Attention of one query token a row.  With n = context_lens[b],
 *   out[b,h] = softmax_t(sm_scale * inv_tau[h] * q[b,h] . k_t) @ v_t  over t < n,   0 where it sees nothing,
 * token t < lens[g] read through the table of the first row of b's group, the others through b's own. */
typedef struct kvq_shared_decode_params {
  kvq_paged_cache cache;
  const void* q;              /* [B, q_heads, 128] of q_type, strides in elements, multiples of 8 */
  int64_t q_stride_b, q_stride_h;
  void* out;                  /* [B, q_heads, 128] of q_type, dense */
  const int32_t* context_lens;
  const float* inv_tau;       /* fp32 [q_heads] or NULL */
  const int32_t* plan_words;  /* device memory, of the same q_heads and kv_heads */
  void* workspace;            /* kvq_shared_decode_workspace_bytes(), any contents, 16-byte aligned */
  int64_t workspace_bytes;
  kvq_shared_plan_info plan;
  float sm_scale;
  int32_t q_heads;            /* a multiple of kv_heads, at most 128 times */
  int32_t q_type;
  int32_t reserved;           /* 0 */
} kvq_shared_decode_params;
int kvq_shared_decode(const kvq_shared_decode_params* p, kvq_stream_t stream);
int64_t kvq_shared_decode_workspace_bytes(const kvq_shared_decode_params* p);

#ifdef __cplusplus
}
#endif
#endif /* KVQ_SHARED_H_ */
