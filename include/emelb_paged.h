/*
 * emelb_paged.h — many requests that share one key / value cache: pages on the device, rows kept in 4 bits, attention
 * over them, and attention of packed prompts.
 *
 * No counterpart in the reference, whose generator keeps one sequence's cache in f16
 * (src/emel/text/generator/detail.hpp:3010-3048).  A serving step goes through these calls in order:
 *
 *   emelb_kv_plan       page tables, slots and running sums of the step from the requests' lengths
 *   emelb_kv_store      the step's keys and values into their slots
 *   emelb_kv_attend     the newest tokens of each request over its pages (decoding)
 *   emelb_attend_packed whole prompts of different lengths, packed behind one another, over 16-bit keys and values;
 *                       what earlier steps left in the pages comes back through emelb_kv_load
 *
 * Conventions
 *  - As in emelb.h: an error bitmask, work enqueued on the context's stream, no allocation, no host wait, calls may be
 *    recorded between emelb_graph_begin and emelb_graph_end.
 *  - Every pointer of a request is memory of the context's GPU; a host pointer or another GPU's memory is refused with
 *    EMELB_INVALID_REQUEST.  emelb_*_can_run checks what can be told without a GPU; the calls check the same first.
 *  - Lengths, tables and slots are read by the kernels.  Values that are out of range are skipped, never followed, and
 *    make the next emelb_sync return EMELB_INVALID_REQUEST.
 *  - Strides count elements.  The head_dim values of a row are contiguous.
 *  - No result overlaps an input, but for emelb_kv_plan's in-place step; a request where one does is refused.
 */
#ifndef EMELB_PAGED_H
#define EMELB_PAGED_H

#include "emelb.h"

#ifdef __cplusplus
extern "C" {
#endif

/* most requests of one call of emelb_kv_plan or emelb_kv_attend */
#define EMELB_KV_MAX_REQUESTS 8192

/* ---- the cache: `pages` pages of page_tokens tokens for every key / value head.
 * A row of a head is kept in groups of 32 values.  With m the group's value of largest magnitude (the first of equal
 * ones): d = m / -8 rounded to f16 and kept within the finite range, q = floor(x / d + 8.5) within 0 .. 15 in exact
 * arithmetic (8 where d is 0), and the value kept is (q - 8) * d: 18 bytes for 32 values, ggml's Q4_0 but for the
 * quotient, which is taken by the scale that is kept.  A NaN counts as 0.
 *
 * Bytes of a page: kv_heads x page_tokens / 16 tiles of 16 tokens, 18 * head_dim bytes each: quants of the keys, of the
 * values, scales of the keys, of the values.  Inside a tile the order is the one in which emelb_kv_attend's lanes read
 * (kv_tile.cuh); emelb_kv_load gives plain rows.  Slot s of the cache is token s % page_tokens of page s / page_tokens.
 * head_dim 32, 64, 96 or 128; page_tokens 16, 32, 64, 128 or 256, else EMELB_UNSUPPORTED_OP. */
typedef struct emelb_kv_pages {
  void* data; /* 16-byte aligned, pages * emelb_kv_page_bytes() */
  int32_t pages, page_tokens, kv_heads, head_dim;
} emelb_kv_pages;
/* bytes of one page; 0 for sizes that the cache does not take */
EMELB_API uint64_t emelb_kv_page_bytes(int32_t head_dim, int32_t kv_heads, int32_t page_tokens);

/* ---- page tables and slot maps of one step.
 * fresh[b] tokens join the cached[b] of request b; fresh[b] = -1: the request has ended.  The ended requests' pages go on
 * top of the stack free_pages (free_count entries before) in request and table order; then each request in order takes
 * the pages it lacks from the top and appends them to its row of `table`.  The first request for which they do not suffice
 * gets nothing in this step, nor does any after it that lacks a page: its slots are -1 and its length stays cached[b].  Its
 * rows count in query_begin all the same: attention computes them, against the last of its cached tokens, and a slot of -1 is the
 * sign to drop the result.
 * A page belongs to one request: one that stands in two rows of the table is given back twice.  A page number out of range is
 * reported each time it is given back or taken, but passed on as it stands; slots in it are -1, and other calls skip it.
 *
 *   lengths[b]      tokens of the request behind the step (0 when ended)
 *   query_begin[b]  first packed row of the request's fresh tokens; [requests] = all of them (waiting requests included)
 *   key_begin[b]    running sum of lengths; [requests] = all of them
 *   slots[i], positions[i]  slot and position of packed row i; -1 and 0 from query_begin[requests] to token_capacity
 *   free_left       entries of the stack behind the step; what lies above them is left as it was
 *   shortage        pages that were wanting
 *
 * `lengths` may be `cached` and free_left may be free_count: then the step is made in place and a captured call can be
 * replayed step after step.  No other two of the arrays may overlap. */
typedef struct emelb_kv_plan_request {
  const int32_t* cached;  /* [requests] */
  const int32_t* fresh;   /* [requests] */
  int32_t* table;         /* [requests][table_stride], the first table_width of each row used */
  int32_t* free_pages;    /* [pages] */
  const int32_t* free_count;
  int32_t* free_left;
  int32_t* lengths;       /* [requests] */
  int32_t* query_begin;   /* [requests + 1] */
  int32_t* key_begin;     /* [requests + 1] */
  int64_t* slots;         /* [token_capacity] */
  int32_t* positions;     /* [token_capacity] */
  int32_t* shortage;
  int64_t table_stride;
  int32_t requests, table_width, pages, page_tokens, token_capacity;
} emelb_kv_plan_request;
EMELB_API uint32_t emelb_kv_plan_can_run(const emelb_kv_plan_request* request);
EMELB_API uint32_t emelb_kv_plan(emelb_ctx* ctx, const emelb_kv_plan_request* request);

/* ---- keys and values of `tokens` packed rows into their slots; rows with a negative slot are skipped.  type EMELB_F32,
 * EMELB_F16 or EMELB_BF16.  The slots of one call are distinct (which of two rows a slot named twice holds is not
 * specified, nor whether it holds one of them whole).  tokens at most 2^31 - 16. */
typedef struct emelb_kv_store_request {
  emelb_kv_pages cache;
  const void* k;          /* [tokens][kv_heads][head_dim] by strides */
  const void* v;
  const int64_t* slots;   /* [tokens] */
  int64_t k_token_stride, k_head_stride, v_token_stride, v_head_stride;
  int32_t tokens;
  uint8_t type;
} emelb_kv_store_request;
EMELB_API uint32_t emelb_kv_store_can_run(const emelb_kv_store_request* request);
EMELB_API uint32_t emelb_kv_store(emelb_ctx* ctx, const emelb_kv_store_request* request);

/* ---- rows back out of the pages, as the values kept (rounded once to `type`): token first[b] + i of request b, up to
 * lengths[b], to row row_begin[b] + i.  Other rows are left as they were, and tokens whose row would be `rows` or more are left out
 * (row_begin may say so without being out of range).  first null: 0. */
typedef struct emelb_kv_load_request {
  emelb_kv_pages cache;
  void* k;                /* [rows][kv_heads][head_dim] by strides */
  void* v;
  const int32_t* table;   /* [requests][table_stride] */
  const int32_t* first;   /* [requests] or null */
  const int32_t* lengths; /* [requests] */
  const int32_t* row_begin; /* [requests + 1], ascending; request b owns rows row_begin[b] .. row_begin[b + 1] - 1 */
  int64_t table_stride, k_token_stride, k_head_stride, v_token_stride, v_head_stride;
  int32_t requests, table_width, rows;
  uint8_t type;
} emelb_kv_load_request;
EMELB_API uint32_t emelb_kv_load_can_run(const emelb_kv_load_request* request);
EMELB_API uint32_t emelb_kv_load(emelb_ctx* ctx, const emelb_kv_load_request* request);

/* ---- attention over the pages.  Request b brings query rows query_begin[b] .. query_begin[b + 1] - 1 (null: row b
 * alone); the last of them is its newest token, so that row i of n sees positions 0 .. lengths[b] - n + i, and none where
 * that is negative (the result is 0).  out = softmax(scale * q k^T) v per head; query heads h * heads / kv_heads .. share
 * key / value head h.  What is rounded: a query row of a head goes in as f16 numbers times a power of two of its own (f32 ones as
 * the sum of two, 22 bits).  Its product with 32 dims of a key is an f32 sum that holds quants above a base: 18 bits of what such
 * products may come to are kept, of f32 queries 22.  A weight times a value's scale is rounded to f16 (bf16 results: the weight
 * before, too; f32 results: to the sum of two).  With S the largest value scale of the head, or 1 where that is larger, and the largest
 * weight of a row as 1, fewer bits are left of weights below 2^-25 S (16-bit results) and of such products below 2^-25 S (f32
 * results: 2^-14 S).  Statistics and sums are f32.
 * Rows of no request are left as they were.  max_queries bounds the rows of a request (more of them are an error that
 * emelb_sync reports, and are not computed); it is fast for few rows, longer chunks belong to emelb_attend_packed.  Lengths
 * of more than 2^31 - 64 are out of range, and so is a call as a whole whose requests' tokens / 32 times kv_heads times rows of a
 * key / value head / 8, each rounded up, come to more than 2^40 or without the tokens to 2^30: nothing of it is computed.
 * heads / kv_heads at most 64; type EMELB_F32, EMELB_F16 or EMELB_BF16 of q and out. */
typedef struct emelb_kv_attend_request {
  emelb_kv_pages cache;
  const void* q;          /* [queries][heads][head_dim] by strides */
  void* out;              /* the same shape */
  const int32_t* table;   /* [requests][table_stride] */
  const int32_t* lengths; /* [requests] */
  const int32_t* query_begin; /* [requests + 1] or null */
  int64_t table_stride, q_token_stride, q_head_stride, out_token_stride, out_head_stride;
  int32_t requests, table_width, heads, queries, max_queries;
  float scale;            /* positive, below 2^127 */
  uint8_t type;
} emelb_kv_attend_request;
EMELB_API uint32_t emelb_kv_attend_can_run(const emelb_kv_attend_request* request);
EMELB_API uint32_t emelb_kv_attend(emelb_ctx* ctx, const emelb_kv_attend_request* request);

/* ---- attention of packed prompts.  Request b: query rows query_begin[b] .. query_begin[b + 1] - 1, key and value rows
 * key_begin[b] .. key_begin[b + 1] - 1.  causal != 0: row i of n sees keys 0 .. keys - n + i of its request, and none
 * where that is negative; else all of them.  A row that sees nothing is 0; rows of no request are left as they were; keys
 * and values that a row does not see have no influence on it, whatever they hold.  A value that is not finite reaches the
 * rows that see it in its head and dim alone.  max_queries bounds the rows of a request (more of them are an error that
 * emelb_sync reports, and are not computed).
 * type EMELB_F16 or EMELB_BF16 of all four tensors; head_dim a multiple of 8 up to 128; heads / kv_heads at most 128; keys at most 2^25; every
 * row 16-byte aligned (base, strides), strides of q, k and v below 2^39, else EMELB_UNSUPPORTED_OP.  Scores, statistics and sums
 * are f32, softmax weights are rounded to `type` for the second product (f16 ones with fewer bits below 2^-21 of a row's largest). */
typedef struct emelb_attend_packed_request {
  const void* q;          /* [queries][heads][head_dim] by strides */
  const void* k;          /* [keys][kv_heads][head_dim] */
  const void* v;
  void* out;              /* [queries][heads][head_dim] */
  const int32_t* query_begin; /* [requests + 1], ascending */
  const int32_t* key_begin;   /* [requests + 1], ascending */
  int64_t q_token_stride, q_head_stride, k_token_stride, k_head_stride, v_token_stride, v_head_stride, out_token_stride,
      out_head_stride;
  int32_t requests, heads, kv_heads, head_dim, queries, keys, max_queries;
  int32_t causal;
  float scale;            /* positive, below 2^127 */
  uint8_t type;
} emelb_attend_packed_request;
EMELB_API uint32_t emelb_attend_packed_can_run(const emelb_attend_packed_request* request);
EMELB_API uint32_t emelb_attend_packed(emelb_ctx* ctx, const emelb_attend_packed_request* request);

#ifdef __cplusplus
}
#endif
#endif /* EMELB_PAGED_H */
