/*
 * qwen_b200_paged.h - C ABI of the operators on paged KV pools: attention for
 * a batch whose sequences share their first pages, and copying, forking,
 * compacting and freeing pages.  No upstream counterpart: upstream keeps one
 * contiguous cache of one sequence (Model/Qwen06B_architecture.py:233-237).
 * All calls are asynchronous on `stream` (a cudaStream_t), neither allocate
 * device memory nor synchronise, can be captured into a CUDA graph, and return
 * 0 or a nonzero code with a message from qwen_b200_last_error()
 * (include/qwen_b200.h); arguments are checked before the first launch, so
 * after a refusal nothing has been launched (code 20, a launch that failed,
 * may come after others).
 */
#ifndef QWEN_B200_PAGED_H
#define QWEN_B200_PAGED_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ------------------------------------------------------------------ pages
 * K and V pools of one geometry: [num_pages][inner][page_tokens][token_bytes]
 * each (inner = layers x kv heads of a page), contiguous, 16-byte aligned, in
 * memory of their own, token_bytes a multiple of 16 (the element type does not
 * matter). */
typedef struct QwenPagePools {
  void *k_pool, *v_pool;
  int num_pages, inner, page_tokens, token_bytes;
} QwenPagePools;

/* A device page table int32 [num_seqs][max_pages], rows `pitch` entries
 * apart: the page holding positions [page_tokens i, page_tokens (i + 1)) of a
 * sequence, or -1. */
typedef struct QwenPageTable {
  int *entries;
  int num_seqs, max_pages;
  long long pitch;
} QwenPageTable;

/* The lists below are HOST arrays of n entries, read before the call returns
 * (they travel as kernel parameters: a captured graph holds their values).
 * They are checked in full; what only the device knows (the pages that a
 * table row names) is range-checked there: such an entry is skipped (fork: -1 in
 * the child's row, or a tail that is not copied) and recorded for
 * qwen_b200_paged_status().
 *
 * copy: the first tokens[i] tokens (NULL: all) of page src[i] into page
 * dst[i], K and V.  Destinations are distinct and no destination is a source;
 * a source may repeat.
 * fork: sequence children[i] becomes a copy of the first lengths[i] positions
 * of sequence parents[i]: its table row takes the parent's full pages
 * (shared), the tokens of the last, partly filled page (lengths[i] %
 * page_tokens of them) are copied into page new_pages[i], and the rest of the
 * row is -1.  new_pages[i] is ignored when lengths[i] is a multiple of the
 * page.  Children are distinct and none of them is a parent; the used new
 * pages are distinct, and no table row that stays may hold one.
 * compact: every page src[i] moves to dst[i] (copied whole) and every entry
 * src[i] of the table becomes dst[i].  Sources are distinct, destinations are
 * distinct and none is a source; no table row may hold a destination.
 * free: the table rows of the sequences become -1 (the same one may be named
 * twice). */
int qwen_b200_pages_copy(const QwenPagePools *pools, const int *src, const int *dst, const int *tokens,
                         int n, void *stream);
int qwen_b200_pages_fork(const QwenPagePools *pools, const QwenPageTable *table, const int *parents,
                         const int *children, const int *lengths, const int *new_pages, int n,
                         void *stream);
int qwen_b200_pages_compact(const QwenPagePools *pools, const QwenPageTable *table, const int *src,
                            const int *dst, int n, void *stream);
int qwen_b200_pages_free(const QwenPageTable *table, const int *seqs, int n, void *stream);

/* Synchronises the current device; 0 if no page operator has recorded an
 * error there since the last call, else 3 (a table entry outside the pool),
 * and clears the record. */
int qwen_b200_paged_status(uint64_t *detail);

/* ------------------------------------------- shared-prefix attention
 * One token per row: row r is a query of sequence seq_ids[r] that sees the
 * positions 0 .. lengths[r] - 1 (+ length_bias) of that sequence's pages:
 *   out[r, h] = sum_t softmax_t(scale q[r, h] . k_t) v_t,
 * k and v of kv head h / (heads / kv_heads); lse[r, h] = log sum_t exp(scale
 * q . k_t).  Scores, softmax statistics and sums are fp32.  The weights are
 * rounded to the input type for their product with v (bf16: half a step each;
 * fp16: half a step, or 2^-32 of the row's largest weight where that is more),
 * the result once more at the end; lse counts the weights unrounded.  A row that sees nothing gives 0 and -inf.  The rows come in
 * groups: consecutive rows whose sequences hold the same tokens in their
 * first prefix_lens[g] positions.  Those are read and multiplied once for the
 * whole group, through the pages of its first row that is as long as the
 * prefix.  A row shorter than its group's prefix runs on its own pages alone.
 *
 * Plan of a batch's groups (host arrays; sum of group_rows = rows): fills
 * `words` (host, int32) and returns how many it wrote, which the caller
 * copies to 16-byte aligned device memory; with words NULL only returns the
 * number.  0: bad arguments (qwen_b200_last_error).  max_length: about the
 * longest row (it weighs the prefix work against the rows' own).  ctas: CTAs
 * that share the prefix work at most (the device's SM count).  The first
 * QWEN_PREFIX_HEADER words are also the host's view of the plan. */
#define QWEN_PREFIX_HEADER 16
int qwen_b200_prefix_plan(int groups, const int *group_rows, const int *prefix_lens, int heads,
                          int kv_heads, int dim, int max_length, int ctas, int *words,
                          int capacity);

typedef struct QwenPrefixAttention {
  const void *q;            /* [rows, heads, dim], last dimension contiguous */
  void *out;                /* the same shape and type; q itself, or memory of its own */
  float *lse;               /* [rows, heads] contiguous, or NULL */
  const void *k_pool, *v_pool; /* [num_pages, kv_heads, page_tokens, dim], strides below */
  const int *page_table, *seq_ids, *lengths; /* device */
  const int *plan_header;   /* host: the first words of the plan */
  void *plan;               /* device: the whole plan */
  void *workspace;          /* 16-byte aligned; one call at a time uses it */
  long long workspace_bytes;
  long long q_row_stride, q_head_stride, out_row_stride, out_head_stride;   /* elements */
  long long page_stride, head_stride, token_stride;                         /* elements, of both pools */
  long long table_pitch;
  int rows, heads, kv_heads, dim;  /* dim 64 or 128 */
  int dtype;                /* of q, out and the pools: 0 fp16, 1 bf16 */
  int num_pages, page_tokens; /* page_tokens a multiple of 16 */
  int num_seqs, max_pages;
  int max_length;           /* about the longest row: chooses how far one row is split */
  int length_bias;          /* added to every lengths[r] (1: lengths are positions) */
  float scale;              /* > 0 */
} QwenPrefixAttention;

long long qwen_b200_prefix_workspace(const int *plan_header, int dim, int max_length);
int qwen_b200_prefix_attention(const QwenPrefixAttention *a, void *stream);
/* Synchronises the current device; 0, or the code that a launch with this
 * device plan has recorded since the last call (1: a bounded wait gave up,
 * 3: a sequence, length or page outside the tables, skipped), and clears the
 * record.  Until a 1 has been read here, the rows that share a prefix give NaN. */
int qwen_b200_prefix_status(const int *plan_header, void *plan, uint64_t *detail);

#ifdef __cplusplus
}
#endif
#endif /* QWEN_B200_PAGED_H */
