/*
 * crispybits_attention.h -- C ABI of the attention between the packed projections: causal attention over
 * packed prompts, and a paged key/value cache held in 4 bits with its append, its read and the attention
 * over it.  In libcrispybits_hip.so, with the conventions of crispybits_hip.h: device pointers, sizes and a
 * hipStream_t (as void*), asynchronous on that stream, a status code and cbk_last_error().  The reference
 * has no counterpart of these; they stand between its fused Q/K/V and its output projection.
 *
 * Types: dtype (CBK_F16 / CBK_BF16 / CBK_F32) is that of q, k, v and the outputs.  head_dim is a multiple of 8
 * up to 256.  Query head h reads kv head h / (heads / kv_heads).  Pointers to q, k, v and outputs are 16-byte
 * aligned and so is every row of a head (strides in elements, between rows at most 2^23).
 *
 * The cache.  pages is int32 [num_pages, kv_heads, cbk_kv4_page_words(head_dim, page_size)], 16-byte
 * aligned; page_size a power of two from 32 on.  Token i of sequence b lies in page
 * block_table[b, i / page_size] (int32 [num_seqs, table_width]) at slot i % page_size.  An entry outside the
 * pool (-1) is no page: a token there is not stored, reads as zeros and takes no part in attention.  A page that a
 * call writes to belongs to one sequence of it; pages read by several are fine.  A token's vector is held
 * as x = s (c - z) with 4-bit codes c, a scale s and a zero point z of its own: over lo = min(0, min x),
 * hi = max(0, max x), z = rint(-15 lo / (hi - lo)), s the float (hi - lo) / 15 (at least 2^-100) with its low four
 * mantissa bits replaced by z, c = clamp(rint(x / s) + z, 0, 15).  A vector with a value that is not finite reads
 * as NaN.
 *
 * seq_lens (int32 [num_seqs]) counts a sequence's tokens with the call's new ones.  cu_seqlens (int32
 * [num_seqs + 1], not decreasing, from 0 on) says which rows of a packed tensor are whose:
 * cu_seqlens[b] .. cu_seqlens[b + 1] - 1.  Lengths live on the device: a captured call follows them on replay.
 */
#ifndef CRISPYBITS_ATTENTION_H
#define CRISPYBITS_ATTENTION_H

#include <stdint.h>

#include "crispybits_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* int32 words of one page and kv head, or -1 for sizes that the cache does not take. */
int64_t cbk_kv4_page_words(int head_dim, int64_t page_size);

/* Stores rows of k and v [rows, kv_heads, head_dim]: row r of sequence b becomes its token
 * seq_lens[b] - (cu_seqlens[b + 1] - cu_seqlens[b]) + r - cu_seqlens[b].  cu_seqlens NULL: rows = num_seqs, row b
 * is the newest token of b.  Rows before token 0 (an idle slot: seq_lens 0) or behind the table are left out.
 * The other tokens' contents stay as they are. */
int cbk_kv4_append(int32_t* pages, int64_t num_pages, int64_t kv_heads, int head_dim, int64_t page_size,
                   const void* k, const void* v, int dtype, int64_t rows,
                   int64_t k_row, int64_t k_head, int64_t v_row, int64_t v_head,
                   const int32_t* block_table, int64_t table_width, const int32_t* seq_lens,
                   const int32_t* cu_seqlens, int64_t num_seqs, int device, void* stream);

/* The reverse: the values that the same rows are held as, into contiguous k and v [rows, kv_heads, head_dim].
 * Tokens that are not stored and rows of no sequence come back as zeros.  At most 2^28 rows, as above. */
int cbk_kv4_read(const int32_t* pages, int64_t num_pages, int64_t kv_heads, int head_dim, int64_t page_size,
                 void* k, void* v, int dtype, int64_t rows,
                 const int32_t* block_table, int64_t table_width, const int32_t* seq_lens,
                 const int32_t* cu_seqlens, int64_t num_seqs, int device, void* stream);

/* out[b, i, h] = softmax(scale q[b, i, h] . K^T) V over sequence b's tokens 0 .. seq_lens[b] - t + i, for its t
 * newest tokens: q and out contiguous [num_seqs, t, heads, head_dim].  A query that sees no token gives
 * zeros.  0 < scale <= 2^127.  partial: cbk_kv4_attention_partial_floats(...) fp32 elements (0: none needed), scratch of
 * this call alone. */
int64_t cbk_kv4_attention_partial_floats(int64_t num_seqs, int64_t t, int64_t heads, int64_t kv_heads, int head_dim,
                                         int64_t page_size, int64_t table_width);
int cbk_kv4_attention(const void* q, int dtype, int64_t num_seqs, int64_t t, int64_t heads,
                      const int32_t* pages, int64_t num_pages, int64_t kv_heads, int head_dim, int64_t page_size,
                      const int32_t* block_table, int64_t table_width, const int32_t* seq_lens, float scale,
                      float* partial, int64_t partial_floats, void* out, int device, void* stream);

/* Causal attention over packed prompts: row i of sequence b attends to rows 0 .. i of it.  q [rows, heads,
 * head_dim], k and v [rows, kv_heads, head_dim] with strides, out contiguous [rows, heads, head_dim].  max_seqlen
 * (0 < max_seqlen <= rows) bounds every sequence's length; rows of a longer one past it are not computed;
 * ceil(max_seqlen / 128) (num_seqs + 1) heads must be below 2^24.  Rows of no
 * sequence (behind the last) are set to zero when zero_tail, else left as they were.  Places that the mask
 * hides take no part whatever they hold; a visible infinity or NaN in v gives an infinity or NaN.  0 < scale <= 2^127. */
int cbk_prompt_attention(const void* q, const void* k, const void* v, int dtype, int64_t rows, int64_t heads,
                         int64_t kv_heads, int head_dim, int64_t q_row, int64_t q_head, int64_t k_row, int64_t k_head,
                         int64_t v_row, int64_t v_head, const int32_t* cu_seqlens, int64_t num_seqs,
                         int64_t max_seqlen, float scale, int zero_tail, void* out, int device, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* CRISPYBITS_ATTENTION_H */
