/*
 * fa_kv.h — C ABI of the paged 8-bit KV cache for MI355X (gfx950): what a serving step does around attention.
 *
 *   fa_kv_plan_launch    block table, slot map, positions and prefix sums of a step, from the requests' lengths
 *   fa_kv_write_launch   new keys and values into 8-bit pages, one scale for each (block of tokens, kv head)
 *   fa_kv_attn_launch    attention over such a cache: single tokens, a few speculative ones, prompt chunks, packed batches
 *
 * Exported by libfa_kv.so.  The rules are those of fa_fwd.h: plain C, all pointers are device pointers, no allocation, no
 * synchronisation, no exception crosses; work is enqueued on the caller's stream; FA_OK or a negative code, nothing is
 * enqueued on an error.  The *_validate functions make the host checks alone and touch no GPU.  Strides between pages and those
 * of scales are below 2^31, strides between a page's rows below 2^24.  What stands on the device
 * (lengths, tables, slots) cannot be refused: each call says what a bad value does; none reads or writes out of bounds.
 * No counterpart in the reference, whose attention ops take whole tensors of 16-bit values.
 */
#ifndef FA_KV_H_
#define FA_KV_H_

#include "fa_fwd.h"

#ifdef __cplusplus
extern "C" {
#endif

#define FA_KV_ABI_VERSION 1

/* How a cache holds its values: value = stored x scale of its (page, block of tokens, kv head). */
#define FA_KV_E4M3 0 /* OCP e4m3 (finite and NaN, no infinities; largest 448) */
#define FA_KV_INT8 1 /* two's complement */

#define FA_KV_MAX_BATCH 8192 /* requests of one fa_kv_plan_launch */

/*
 * Plan of a step.  Request b holds cached[b] tokens and gets new_tokens[b] more (values below 0 count as 0); the pages it
 * holds are the first ceil(cached / page_size) entries of its row of block_table.  The new tokens of all requests stand
 * packed, one request after the other, in arrays of max_tokens rows.
 *   cu_seqlens[b]   rows before request b, at most max_tokens
 *   admitted[b]     1 where the request's tokens and pages fit: its last row is below max_tokens, cached + new <= table_pages *
 *                   page_size, and it needs no page, or the pages that it and the fitting requests before it need are there
 *   block_table     entries of the pages an admitted request gets: the i-th page that the fitting requests need, in order, is
 *                   free_pages[free_count - 1 - i]; other entries stay as they were
 *   seqused[b]      cached + new where admitted, else cached
 *   positions[t]    position of row t in its request, at most 2^31 - 1; 0 behind the last row
 *   slots[t]        page x page_size + offset of row t; -1 where its request is not admitted, where the page is negative and
 *                   behind the last row
 *   free_left       free_count less the pages given out: the first free_left entries of free_pages are still free
 * A free_count beyond free_capacity counts as free_capacity, one below 0 as 0.  Outputs overlap neither the inputs nor the
 * table nor one another: a step's seqused becomes the next one's cached by changing places, not by being the same array.
 */
typedef struct fa_kv_plan_params {
  const int32_t* cached;     /* [batch] */
  const int32_t* new_tokens; /* [batch] */
  int32_t* block_table;      /* [batch][block_table_stride], written in place */
  const int32_t* free_pages; /* [free_capacity]; may be NULL when that is 0 */
  const int32_t* free_count; /* [1] */
  int32_t* cu_seqlens;       /* [batch + 1] */
  int32_t* seqused;          /* [batch] */
  int32_t* positions;        /* [max_tokens] */
  int64_t* slots;            /* [max_tokens] */
  uint8_t* admitted;         /* [batch] */
  int32_t* free_left;        /* [1] */
  int64_t block_table_stride; /* elements */
  int32_t batch;             /* 0 ... FA_KV_MAX_BATCH */
  int32_t table_pages;       /* entries of a row, at most block_table_stride */
  int32_t page_size;         /* > 0; table_pages * page_size < 2^31 */
  int32_t max_tokens;        /* >= 0 */
  int32_t free_capacity;     /* >= 0 */
  int32_t reserved;          /* must be 0 */
} fa_kv_plan_params;

FA_API int fa_kv_plan_validate(const fa_kv_plan_params* p);
FA_API int fa_kv_plan_launch(const fa_kv_plan_params* p, void* stream);

/*
 * Write rows into the cache.  Row t of key / value ([tokens][heads][head_dim], elements of `dtype`) goes to slot slots[t];
 * a slot below 0 or beyond the pool leaves its row out.  The rows of one call that go to one block of scale_block tokens
 * stand next to each other in the call and no slot is given twice, as fa_kv_plan_launch lays them out (other orders leave
 * the contents of such a block undefined, and nothing else).  The same goes for one pool given for keys and values alike.  For
 * each block and head that rows go to:
 *   needed = e4m3: 2^e, the smallest e >= -100 with 448 x 2^e >= the rows' largest finite magnitude (2^-100 without one)
 *            int8: max(largest finite magnitude x fp32(1 / 127), 2^-100)
 *   scale  = max(old scale, needed); needed alone where a row goes to the block's first slot: the block starts anew then,
 *            whatever a recycled page held
 *   the rows are stored as round(x * fp32(1 / scale)), to nearest even, infinities as the largest magnitude, NaN as NaN (int8: 0)
 *   where the scale grew, the block's other rows are rounded again, stored x fp32(old / scale): with the powers of two of e4m3
 *   that changes values only where they leave the normal range
 */
typedef struct fa_kv_write_params {
  const void* key;   /* 16-byte aligned, as are all rows */
  const void* value;
  void* key_pages;   /* [num_pages][page_size][heads][head_dim] bytes, 16-byte aligned, as are all rows */
  void* value_pages;
  float* key_scales; /* [num_pages][page_size / scale_block][heads] */
  float* value_scales;
  const int64_t* slots; /* [tokens] */
  int64_t key_stride_t, key_stride_h; /* elements */
  int64_t value_stride_t, value_stride_h;
  int64_t kp_stride_p, kp_stride_s, kp_stride_h; /* bytes */
  int64_t vp_stride_p, vp_stride_s, vp_stride_h;
  int64_t ks_stride_p, ks_stride_b, ks_stride_h; /* elements */
  int64_t vs_stride_p, vs_stride_b, vs_stride_h;
  int32_t tokens;      /* >= 0 */
  int32_t heads;       /* > 0 */
  int32_t head_dim;    /* multiple of 16, 16 ... 256 */
  int32_t num_pages;   /* > 0; num_pages * page_size < 2^31 */
  int32_t page_size;   /* multiple of scale_block */
  int32_t scale_block; /* multiple of 32 */
  int32_t dtype;       /* FA_DTYPE_* */
  int32_t format;      /* FA_KV_* */
} fa_kv_write_params;

FA_API int fa_kv_write_validate(const fa_kv_write_params* p);
FA_API int fa_kv_write_launch(const fa_kv_write_params* p, void* stream);

/*
 * Attention:  out = softmax(scale Q K^T + mask) V  with K and V read from the cache, as fa_fwd_launch computes it over a paged
 * 16-bit cache.  Products are formed from the stored values, exact in `dtype`; a block's scales multiply scores and
 * probabilities in fp32, so they enter unrounded.  Scales are finite and not negative.
 *   dense  (cu_seqlens_q NULL): sequence b has seqlen_q query rows at q + b q_stride_b
 *   packed: sequence b owns rows [cu[b], cu[b + 1]) (clipped to total_q rows); seqlen_q is the longest; rows beyond it are left
 *           as they were, and so are those behind the last sequence; q_stride_b, o_stride_b and lse_stride_b are ignored
 * Keys of sequence b: the first seqused_k[b] (clipped to 0 ... table_pages * page_size); key r lives in page
 * block_table[b][r / page_size].  A table entry outside 0 ... num_pages - 1 hides its keys.  is_causal: query row i of Lq
 * sees key j <= Lk - Lq + i.  Rows that see no key get out = 0, lse = +inf.
 * K and V of keys that a row does not see, beyond a sequence's end or behind the causal mask, have no part in it, whatever
 * bytes stand there.  A NaN (e4m3) in a key of K makes the rows that see it NaN, one in V their outputs, in that element at least
 * and not their lse.
 */
typedef struct fa_kv_attn_params {
  const void* q;         /* dtype elements; base and rows 16-byte aligned */
  const void* key_pages; /* [num_pages][page_size][heads_k][head_dim] bytes; base and rows 16-byte aligned */
  const void* value_pages;
  const float* key_scales; /* [num_pages][page_size / scale_block][heads_k] */
  const float* value_scales;
  void* out;
  float* lse;
  const int32_t* block_table;  /* [batch][block_table_stride] */
  const int32_t* seqused_k;    /* [batch] */
  const int32_t* cu_seqlens_q; /* [batch + 1] or NULL */
  int64_t q_stride_b, q_stride_s, q_stride_h; /* elements */
  int64_t kp_stride_p, kp_stride_s, kp_stride_h; /* bytes */
  int64_t vp_stride_p, vp_stride_s, vp_stride_h;
  int64_t ks_stride_p, ks_stride_b, ks_stride_h; /* elements */
  int64_t vs_stride_p, vs_stride_b, vs_stride_h;
  int64_t o_stride_b, o_stride_s, o_stride_h;
  int64_t lse_stride_b, lse_stride_h, lse_stride_s;
  int64_t block_table_stride; /* elements */
  int32_t batch, heads_q, heads_k;
  int32_t seqlen_q;    /* >= 0; packed: the longest sequence's */
  int32_t total_q;     /* packed: rows of q and out */
  int32_t head_dim;    /* multiple of 16, 16 ... 256 */
  int32_t num_pages;   /* > 0 */
  int32_t table_pages; /* entries of a table row that may be used, at most block_table_stride */
  int32_t page_size;   /* multiple of scale_block, at most 2^20; table_pages * page_size <= 2^29 */
  int32_t scale_block; /* multiple of 32 */
  float scale;
  int32_t dtype;       /* FA_DTYPE_* */
  int32_t format;      /* FA_KV_* */
  int32_t is_causal;   /* 0 / 1 */
  int32_t num_splits;  /* slices of the key range: 0 = choose, else 1 ... FA_MAX_SPLITS */
  int32_t reserved;    /* must be 0 */
} fa_kv_attn_params;

FA_API int fa_kv_attn_validate(const fa_kv_attn_params* p);
/* Device scratch of the call: partial results of key slices; 0 where there are none or `p` is invalid. */
FA_API size_t fa_kv_attn_workspace_bytes(const fa_kv_attn_params* p);
/* The workspace (16-byte aligned) must stay alive until the enqueued work has run; nothing in it needs clearing. */
FA_API int fa_kv_attn_launch(const fa_kv_attn_params* p, void* workspace, size_t workspace_bytes, void* stream);

FA_API int fa_kv_version(void);
FA_API const char* fa_kv_error_string(int rc);

#ifdef __cplusplus
}
#endif
#endif /* FA_KV_H_ */
