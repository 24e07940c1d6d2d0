/*
 * bonsai_pages.h - C ABI of what goes around the pages of a 4-bit cache (bonsai_paged.h) that many requests use: page tables on the device
 * (growing, giving back, forking, compacting, copying pages), attention of requests that have a long prefix in common, and attention
 * over the pages that a cheap score chooses for each query. Contexts, pools, rows, errors, streams and bp_paged_status are those of
 * bonsai_paged.h. The reference has no counterpart.
 */
#ifndef BONSAI_PAGES_H
#define BONSAI_PAGES_H

#include "bonsai_paged.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Page tables, all device int32: row r has kv_len[r] tokens in the pages table[r * table_stride + i], i = 0 .. ceil(kv_len / page_tokens) - 1
 * (entries behind these mean nothing, and the calls may overwrite them; whoever shortens a row by hand has to take the pages behind it
 * from refs, too); refs[p] is how often page p is held, by rows and by whoever
 * else adds to it; a page with refs 0 is free. n_rows <= 16384. A row may be any sequence: a request, a prefix of several, a kept one.
 * The calls below run on the device alone, in the stream's order; what they refuse there they leave as it was, and
 * bp_paged_status reports it (rows, pages or lengths out of range, no free page left, a row that has no room). The results do not depend on how the
 * device goes about them. */
typedef struct bp_page_tables {
  void *table, *kv_len, *refs;
  uint32_t n_rows, row_pages, table_stride, n_pages, page_tokens;
} bp_page_tables;

/* Every row r gets n_new[r] (device int32, >= 0) further tokens: kv_len[r] += n_new[r]; pages that it needs for them are the
 * lowest free ones, in the order of the rows. For what is done with the tokens: q_start[n_rows + 1] (device int32) = sums of n_new, and of
 * token t of row r, at q_start[r] + t: positions (device int32 [n_out]) = its place in the row, slots (device int64 [n_out])
 * = page * page_tokens + place in the page. Places from q_start[n_rows] on become -1 in both: padding, as for bp_rope and
 * bp_kv4_append. A row that is refused (no room, no pages) keeps its length, and its tokens become padding too. */
int bp_pages_grow(bp_paged_ctx* ctx, void* stream, const bp_page_tables* tables, const void* n_new, void* q_start, void* positions, void* slots, uint32_t n_out);
/* The rows rows[0 .. n - 1] (device int32; negative: none) give their pages back: refs - 1 for each, kv_len 0. Entries that are no pages, and counts that are 0 already, are passed over. */
int bp_pages_release(bp_paged_ctx* ctx, void* stream, const bp_page_tables* tables, const void* rows, uint32_t n);
/* Row children[i] (which must be empty) becomes what row parents[i] is (device int32 [n] both; a negative one of either: no pair). Full pages are
 * shared; a last page that is not full is to be copied, into the lowest free pages in the order of the pairs: src[i], dst[i] (device
 * int32 [n]) say from where to where, -1 where there is nothing to copy. A row is a child once in a call, and not a parent too. n <= 16384. */
int bp_pages_fork(bp_paged_ctx* ctx, void* stream, const bp_page_tables* tables, const void* parents, const void* children, uint32_t n, void* src, void* dst);
/* Moves pages to the front: the i-th highest used page goes to the i-th lowest free one as long as that lies below it, for i < most. Tables and refs
 * follow; src[i], dst[i] (device int32 [most]) are what is to be copied, -1 behind the last. Afterwards nothing but the moved pages'
 * places has changed, and no source is a destination. (Holders of pages outside of the tables' rows have to follow src and dst themselves.) */
int bp_pages_compact(bp_paged_ctx* ctx, void* stream, const bp_page_tables* tables, void* src, void* dst, uint32_t most);

/* Arrays of n_pages pages of page_bytes bytes each (a multiple of 4, 4-byte aligned; 16 is faster): the pools of a model's layers, their summaries. */
typedef struct bp_page_array {
  void* data;
  uint64_t page_bytes;
} bp_page_array;
/* Page src[i] of every array (host array of n_arrays) goes to page dst[i] (device int32 [n]; a negative one of either: nothing). A destination is there once and is no source. */
int bp_pages_copy(bp_paged_ctx* ctx, void* stream, const bp_page_array* arrays, uint32_t n_arrays, uint32_t n_pages, const void* src, const void* dst, uint32_t n);

/* bp_kv4_attention for requests behind prefixes that several of them have in common. Prefix g (prefix_len[g] keys in the pages
 * prefix_table[g * prefix_stride + i]) is that of the requests prefix_start[g] .. prefix_start[g + 1] - 1 (device int32 [n_prefix + 1], ascending);
 * requests before prefix_start[0] and from prefix_start[n_prefix] on have none. Every query of a request sees all keys of its
 * prefix, and of the request's own ones (kv_len[r], in page_table) those that it would see in bp_kv4_attention; so the outputs are those of
 * bp_kv4_attention over prefix and own keys in one row of pages, where a request has no fewer own keys than queries. A query that sees no key
 * gives zeros. What has fewer than 32 bits is what has fewer in bp_kv4_attention (queries, and the weights that multiply values); results of either part are joined in 32.
 * How the SMs are shared between prefixes and requests goes by max_prefix and max_kv: close ones are worth it. max_prefix: no prefix has more keys. work: device memory for 32-bit results of either part, 16-byte aligned, of
 * bp_kv4_shared_work(total_q, n_head, head_dim) floats; it may serve one call after the other. */
typedef struct bp_kv4_shared {
  bp_rows q, out;
  const void *q_start, *kv_len, *page_table, *prefix_start, *prefix_len, *prefix_table;
  void* work;
  uint32_t n_req, n_head, total_q, max_q, max_kv, table_stride, n_prefix, max_prefix, prefix_stride;
  float scale;
} bp_kv4_shared;
uint64_t bp_kv4_shared_work(uint32_t total_q, uint32_t n_head, uint32_t head_dim);
int bp_kv4_attention_shared(bp_paged_ctx* ctx, void* stream, uint32_t dtype, const bp_kv4_pool* pool, const bp_kv4_shared* args);

/* What is kept of the keys of each page p and KV head h of a pool, in 8 bits: scales f32 [n_pages][n_kv_head], codes int8
 * [n_pages][n_kv_head][2][head_dim]; codes[0] * scale is the smallest such number that is no smaller than any of the keys in that dim,
 * codes[1] * scale the same of the negated keys. With e the exponent of the largest of them, limited to -24 .. 16, scale is 2^(e - 6), or twice
 * that where 127 * 2^(e - 6) is less; codes are limited to +-127. Keys that are no numbers are passed over (a dim that has no others counts as 0). */
typedef struct bp_block_summary {
  void *codes, *scales; /* 16-byte and 4-byte aligned */
} bp_block_summary;
/* The summaries of pages[0 .. n - 1] (device int32; negative: none), of their first n_tok[i] tokens (device int32, > 0; null: all). A page is there once. */
int bp_kv4_summarise(bp_paged_ctx* ctx, void* stream, const bp_kv4_pool* pool, const bp_block_summary* summary, const void* pages, const void* n_tok, uint32_t n);

/* Chooses at most `chosen` pages for every token and KV head. A token that sees n keys (of its request, as in bp_kv4_attention without a
 * window) sees ceil(n / page_tokens) pages. The first `first` and the last `last` of them are always chosen (last >= 1, first + last <= chosen); of the others, which have to be
 * full and to have a summary, those with the highest scores, of equal ones the earlier. The score is no less than the sum of q . k over the
 * group's query heads for any key k of the page, but for its roundings to 8 bits:
 *   P_d, M_d = sum over the group's query heads, in their order and in binary32, of max(q_d, 0), max(-q_d, 0)
 *   p_d, m_d = min(rint(P_d / u), 255), min(rint(M_d / u), 255), u = 2^(e - 7) with e the exponent of the largest of all P_d, M_d (e >= -100)
 *   score = scale * sum over d of p_d codes[0][d] + m_d codes[1][d]      (the sum is a whole number below 2^24: nothing rounds)
 * pages [total_q][n_kv_head][chosen] (device int32): the chosen pages in the order of the keys, -1 behind them; keys [total_q] (device
 * int32): the number of keys in them, the same for every head; -1 and no pages for rows that are no request's. Queries that are no numbers count as 0.
 * ceil(max_kv / page_tokens) <= 49152. */
typedef struct bp_kv4_choice {
  bp_rows q;
  const void *q_start, *kv_len, *page_table;
  void *pages, *keys;
  uint32_t n_req, n_head, total_q, max_q, max_kv, table_stride, chosen, first, last;
} bp_kv4_choice;
int bp_kv4_select(bp_paged_ctx* ctx, void* stream, uint32_t dtype, const bp_kv4_pool* pool, const bp_block_summary* summary, const bp_kv4_choice* args);
/* Attention of every token over pages of its own for each KV head: pages and keys as bp_kv4_select writes them. Zeros where
 * keys is 0; rows with negative keys are left as they were. Fewer bits: as in bp_kv4_attention. total_q <= 65535. */
typedef struct bp_kv4_chosen {
  bp_rows q, out;
  const void *pages, *keys;
  uint32_t n_head, total_q, chosen;
  float scale;
} bp_kv4_chosen;
int bp_kv4_attention_selected(bp_paged_ctx* ctx, void* stream, uint32_t dtype, const bp_kv4_pool* pool, const bp_kv4_chosen* args);

#ifdef __cplusplus
}
#endif
#endif /* BONSAI_PAGES_H */
