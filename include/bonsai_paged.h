/*
 * bonsai_paged.h - C ABI of the operators that serve many requests at once from ONE paged KV cache held in 4 bits:
 * rotary positions, append, read-back and attention. Same conventions as bonsai_attn.h (status codes, an opaque owner of
 * the scratch memory, device pointers, asynchronous on the caller's stream, no CPU path), but the cache, the RoPE table and
 * every activation belong to the caller. The reference has no counterpart: it holds one sequence per model in 8 bits.
 *
 * Activations are 16-bit rows [token][head][head_dim] (BP_DTYPE_F16 or BP_DTYPE_BF16); a row of head_dim values is dense,
 * tokens and heads lie `tok_stride` and `head_stride` ELEMENTS apart (a view into a fused projection's output). All sums,
 * norms and softmax statistics are binary32.
 *
 * The cache of one layer is a pool of pages [n_pages][n_kv_head][page_tokens * head_dim * 5 / 4 bytes], 16-byte aligned.
 * A token's slot is page * page_tokens + place in the page. A page of a head holds, in this order,
 *   K codes [page_tokens][head_dim / 2 bytes], K d [page_tokens][blocks] f16, K m [page_tokens][blocks] f16, then the
 *   same three of V; a block is 32 consecutive dims and a value is m + d * q with a whole q of 0 .. 15.
 * A row of K codes has 4 chunks c of one little-endian 32-bit word per block b: bits 4 j .. 4 j + 3 are dim
 * 32 b + 8 c + 2 j, bits 16 + 4 j .. the dim behind it (j = 0 .. 3). A row of V codes has 8 chunks c of 16 bits per block
 * b: bits 4 i .. are dim 32 b + 4 c + i; where a row has 64 bytes (head_dim 128), tokens with bit 1 of their place set
 * have the two halves of the row changed over. (The orders are those in which the attention kernels' lanes want them.)
 * Quantisation of a block, in binary32 without contraction: values are limited to +-64512; with u = the power of two that
 * is the distance of neighbouring f16 numbers at max |x| * 65 / 64 (at least 2^-24), m = rint(min / u) u,
 * d = rint((max - min) * (1 / 15) / u) u, q = clamp(rint((x - m) * (1 / d)), 0, 15), 0 where d = 0. So every value of a
 * block is an f16 number: dequantisation does not round. A NaN makes its whole block NaN.
 */
#ifndef BONSAI_PAGED_H
#define BONSAI_PAGED_H

#include "bonsai_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { BP_DTYPE_F16 = 0, BP_DTYPE_BF16 = 1 };
enum { BP_ROPE_HALF = 0, BP_ROPE_INTERLEAVED = 1 };

/* Owner of the scratch memory of these calls on one device: not thread-safe, and calls on one context must not overlap on
 * different streams. One serves any number of pools, layers and shapes. `*out` is set even on failure (message); destroy
 * it either way. */
typedef struct bp_paged_ctx bp_paged_ctx;
int bp_paged_create(int32_t device, bp_paged_ctx** out);
void bp_paged_destroy(bp_paged_ctx* ctx);
/* Waits for `stream`, then: BP_OK; BP_ERR_CONTEXT_OVERFLOW once if a token's position lay behind the table, its slot behind
 * the pool, a page id outside the pool, or a request had more keys than its row of the page table holds or max_kv says, more
 * queries than max_q says or some outside the rows of q (they were left out or cut, nothing outside the caller's buffers was
 * touched); or the latched BP_ERR_TIMEOUT / BP_ERR_DEVICE_LOST. */
int bp_paged_status(bp_paged_ctx* ctx, void* stream);
const char* bp_paged_last_error(const bp_paged_ctx* ctx);

/* Rotary table: device f32 [n_pos][rot_dim / 2][2] = (cos, sin), of the first rot_dim dims of a head (even, >= 2).
 * layout BP_ROPE_HALF: dim i is turned with dim i + rot_dim / 2; BP_ROPE_INTERLEAVED: dim 2 i with dim 2 i + 1. */
typedef struct bp_rope_table {
  const void* cos_sin;
  uint32_t n_pos, rot_dim, layout;
} bp_rope_table;
/* What a table is made from: theta_i = freq_base^(-2 i / rot_dim), scaled for long contexts.
 * BP_ROPE_SCALE_NONE; LINEAR: theta_i / factor; NTK: freq_base * factor^(rot_dim / (rot_dim - 2)) instead of freq_base;
 * YARN: between the two of NONE and LINEAR by how often dim pair i turns within orig_ctx positions: more than beta_fast
 * times keeps theta_i, fewer than beta_slow times divides it, in between a linear ramp over the pair's index; cos and sin
 * are multiplied by 0.1 ln(factor) + 1 (factor > 1). */
enum { BP_ROPE_SCALE_NONE = 0, BP_ROPE_SCALE_LINEAR = 1, BP_ROPE_SCALE_NTK = 2, BP_ROPE_SCALE_YARN = 3 };
typedef struct bp_rope_config {
  uint32_t n_pos, rot_dim, scaling;
  float freq_base, factor, beta_fast, beta_slow;
  uint32_t orig_ctx;
} bp_rope_config;
/* Fills a table on the device, in binary64, rounded once. */
int bp_rope_fill(bp_paged_ctx* ctx, void* stream, const bp_rope_config* cfg, void* table_out);

/* x rows -> out rows (the same memory, or memory that does not overlap): an RMS norm over the head first if w_norm (activation
 * type, [head_dim]) is given, then the rotation by positions[token] (device int32). inverse != 0 is its transpose, by minus
 * the angle and with the same factor: the gradient with respect to x (not with w_norm). With a table of cos^2 + sin^2 = 1 it
 * undoes the rotation; a BP_ROPE_SCALE_YARN table's factor it applies once more. head_dim even, <= 256; n_tok * n_head
 * <= 2^28. Tokens with a negative position are padding: their rows are not written. */
typedef struct bp_rows {
  void* data;
  int64_t tok_stride, head_stride;
} bp_rows;
int bp_rope(bp_paged_ctx* ctx, void* stream, uint32_t dtype, const bp_rows* x, const bp_rows* out, uint32_t n_tok, uint32_t n_head,
            uint32_t head_dim, const void* positions, const bp_rope_table* table, const void* w_norm, float eps, uint32_t inverse);

typedef struct bp_kv4_pool {
  void* data;
  uint32_t n_pages, page_tokens, n_kv_head, head_dim; /* page_tokens 16, 32 or 64; head_dim 64 or 128 */
} bp_kv4_pool;
/* Bytes of a pool (0 if its shape is not one that the calls accept). */
uint64_t bp_kv4_pool_bytes(const bp_kv4_pool* pool);
/* k, v rows -> the pool, at slots[token] (device int64; negative: padding, nothing is written). K is normalised first if
 * w_k_norm is given and rotated by positions[token] if table is; the squares of a row are summed as a binary tree over
 * neighbouring dims, 1 / sqrt is correctly rounded, nothing is contracted: a cache does not depend on the batch. With a table,
 * tokens with a negative position are padding too. A slot may occur once in a call (the bytes
 * of one that occurs twice are of both tokens). */
int bp_kv4_append(bp_paged_ctx* ctx, void* stream, uint32_t dtype, const bp_kv4_pool* pool, const bp_rows* k, const bp_rows* v,
                  uint32_t n_tok, const void* positions, const void* slots, const bp_rope_table* table, const void* w_k_norm, float eps);
/* The pool's rows at slots[token] -> k, v rows (negative slots: not written). */
int bp_kv4_read(bp_paged_ctx* ctx, void* stream, uint32_t dtype, const bp_kv4_pool* pool, const void* slots, uint32_t n_tok,
                const bp_rows* k, const bp_rows* v);

/* Attention of several requests. q, out: rows of n_head heads, the requests' queries one behind the other: request r has
 * rows [q_start[r], q_start[r + 1]) (device int32 [n_req + 1], no entry below the one before it) and kv_len[r] keys (device
 * int32), in the pages page_table[r * table_stride + i] (device int32), i = 0 .. ceil(kv_len / page_tokens) - 1. Its last query
 * sees all its keys, the one before all but the last, and so on; with window > 0 each sees the last `window` of those. A query
 * that sees none gives zeros; one that sees a value that is no number gives none in that value's block of dims. out may be q
 * itself. total_q = rows of q; max_q, max_kv: no request has more queries or keys (they only size the launches; more keys
 * than max_kv or than table_stride pages are not looked at). scale multiplies q.k.
 * Scores, maxima and sums are binary32. Two things have fewer bits: queries become f16 numbers times a power of two per row
 * (both types keep all their bits down to 2^-18 of a row's largest element), and the exponentials that weigh the values are
 * rounded to f16 once (2^-11 of each; they are summed before). */
typedef struct bp_kv4_attn {
  bp_rows q, out;
  const void *q_start, *kv_len, *page_table;
  uint32_t n_req, n_head, total_q, max_q, max_kv, table_stride, window;
  float scale;
} bp_kv4_attn;
int bp_kv4_attention(bp_paged_ctx* ctx, void* stream, uint32_t dtype, const bp_kv4_pool* pool, const bp_kv4_attn* args);

#ifdef __cplusplus
}
#endif
#endif /* BONSAI_PAGED_H */
