/* kv_cache.h -- the 4-bit KV cache and the operators on cache pages
 * (libkernels.so).
 *
 * No counterpart in the reference's C-ABI, whose cache is fp32
 * (csrc/kernels.h:25-26, src/terra/engine.t:793-856).  These stand beside the
 * bf16 pages of attn_block.h and take the same page tables, row maps, split
 * arguments, error words and status codes; head_dim is 128 and a page holds
 * 16 tokens.  Calls are stream-ordered and allocate nothing.
 *
 * 4-bit page.  A group is 32 consecutive dims of one token and KV head.  With
 * a = max |x| over the group, its scale s is a / 7.5 rounded up to four
 * significant bits (at least 2^-126) and its codes are n = rint(x / s) in
 * [-8, 7], so the value held, n * s, is within s / 2 of x and is a bf16 number.
 * A group with a NaN, an infinity or a >= 2^120 gets the scale NaN (0x7FC0) and
 * reads back as NaN.  72 bytes a token and head: 4.5 bits a value.
 *
 *   k/v cache  uint8 [pages][nkv][1152]: 1024 bytes of codes n + 8 (two a byte,
 *              the even dim in the low half), then bf16 scales [16 tokens][4]
 *   K codes    dim 32 j + 8 w + i (i < 8) of token t at byte
 *              t * 64 + w * 16 + j * 4 + i / 2
 *   V codes    dim 32 j + 4 g + i (i < 4) of token 8 a + 2 w + b at byte
 *              a * 512 + (4 g + w) * 16 + b * 8 + 2 j + i / 2
 * which is the order the decode kernel's tensor-core fragments read with
 * 16-byte loads.
 *
 * Error words (device int32, optional, set, never cleared): 1 a wait inside the
 * decode kernel gave up after two seconds and its rows are wrong, 4 a position
 * outside the page table, 5 a length that was cut, 6 a page id outside the
 * cache, 7 a sequence row outside the table, 8 no free page left.
 */
#ifndef TIME_B200_KV_CACHE_H
#define TIME_B200_KV_CACHE_H

#include <stddef.h>
#include <stdint.h>

#include "moe_layer.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Bytes of one page of the K (or V) cache: nkv * 1152. */
size_t attn_kv4_page_bytes(int nkv);

/* attn_rope_kv_write_rows into 4-bit pages: partial rotate-half RoPE (pairs
 * (i, i + rot/2), angle = float(pos) * inv_freq[i]) on the q and k heads of
 * every row, rounded to bf16; q to q_out, the rotated keys to k_out when given
 * (bf16 [B][nkv][128], what attn_prompt_packed reads), k and v quantised into
 * slot pos % 16 of page page_table[row_seq[b]][pos / 16] (row_seq null: b).
 * A token's bytes are its own, so rows may fill one page in any order; two
 * rows of a call must not name the same position of the same sequence.
 * Skipped rows and error words as in attn_rope_kv_write_rows: a skipped row's
 * outputs are left as they were.  qkv, q_out, k_out and the caches 16-byte
 * aligned. */
moe_status_t attn_kv4_rope_write_rows(const void* qkv_bf16, int B, int nq, int nkv, int head_dim, int rot,
                                      const float* inv_freq, const int32_t* positions, const int32_t* row_seq,
                                      int num_seqs, const int32_t* page_table, int max_pages, int page_size,
                                      int num_cache_pages, void* q_out_bf16, void* k_out_bf16, void* k_cache,
                                      void* v_cache, int32_t* seq_lens_out, int* error_word, cwStream_t stream);

/* Rows of the cache as the bf16 values held: k_out[b], v_out[b] (bf16
 * [B][nkv][128], either may be null) = the token at positions[b] of page-table
 * row row_seq[b].  A row outside the tables or on a page id outside the cache
 * is zeros (error words 4, 6, 7). */
moe_status_t attn_kv4_read_rows(const void* k_cache, const void* v_cache, int num_cache_pages,
                                const int32_t* positions, const int32_t* row_seq, int num_seqs,
                                const int32_t* page_table, int max_pages, int page_size, int B, int nkv, int head_dim,
                                void* k_out_bf16, void* v_out_bf16, int* error_word, cwStream_t stream);

/* Context split for attn_kv4_decode_rows that fills the GPU at this batch and
 * longest context; max_splits = ceil(max_context / split).  max_context is best
 * the longest context of the call, not what the page table has room for: the
 * split grows with it, and the grid and the workspace with max_splits. */
int attn_kv4_split_tokens(int B, int nkv, int max_context);
/* Bytes of the split-partials workspace. */
size_t attn_kv4_decode_workspace_bytes(int B, int nq, int max_splits);

/* attn_decode_paged_rows over 4-bit pages: same arguments, outputs (bf16 rows
 * and, when out_q is given, their e4m3 1x128 quantisation) and checks; NaN in a
 * bf16 row is the e4m3 NaN in out_q, whatever else the row holds.  Rows with
 * seq_lens[b] <= 0 or row_seq outside [0, num_seqs) get zeros; slots past a
 * sequence's length are not read into the result whatever they hold.
 * max_splits * split_tokens is at most 2^31 - 8193 (else MOE_ERR_UNSUPPORTED).  A
 * row's bits depend on split_tokens and on nothing else of the call.  scale is
 * finite, of any sign.  The workspace is the call's own until it has run: calls
 * that may run at the same time take one each. */
moe_status_t attn_kv4_decode_rows(const void* q_bf16, const void* k_cache, const void* v_cache, int num_cache_pages,
                                  const int32_t* page_table, int max_pages, const int32_t* row_seq, int num_seqs,
                                  const int32_t* seq_lens, int B, int nq, int nkv, int head_dim, int page_size,
                                  float scale, int split_tokens, int max_splits, void* workspace,
                                  size_t workspace_bytes, void* out_bf16, void* out_q, float* out_s, int out_ld,
                                  int* error_word, cwStream_t stream);

/* ---------------------------------------------------------------- pages
 * Operators on the pages of num_caches caches (K and V of every layer, bf16 or
 * 4-bit) of one allocation: cache c, page p at caches + c * cache_stride +
 * p * page_bytes (bytes, multiples of 16).  A sequence of len tokens owns the
 * first ceil(len / 16) entries of its page-table row; a page that no row owns
 * is free, so nothing is counted between calls and a row is freed by leaving
 * it out.  An owned entry outside [0, num_pages) is carried as -1 (error 6).
 * The workspace is the call's own until it has run, as for decode. */
size_t kv_pages_workspace_bytes(int num_pages, int num_rows);

/* New rows from old ones: table_out[i], lens_out[i] = row parents[i] of
 * table_in (-1: an empty row, length 0) with room for reserve[i] more tokens
 * (null: 0 for all).  Children share their parent's pages.  A child that will
 * append (reserve > 0) into a page in part filled keeps that page if it has
 * the most tokens in it of all rows that share it (an appending row before one
 * that is not, then the lowest row); otherwise it gets a copy.  Copies and
 * reserved pages take the free pages from the lowest id on, rows in order, a
 * row's copy before its reserved pages; free are the pages that no child owns,
 * those of parents left out among them.  Entries behind a row's pages are -1.
 * Too few free pages: the entries left over are -1 (error 8) and their copies
 * are not made.  A reservation beyond max_pages is cut (error 4), a length
 * beyond it too (error 5).  table_out and lens_out overlap no input. */
moe_status_t kv_pages_fork(void* caches, size_t cache_stride, int num_caches, int num_pages, size_t page_bytes,
                           int page_size, const int32_t* table_in, int max_pages, const int32_t* lens, int num_seqs,
                           const int32_t* parents, const int32_t* reserve, int num_out, int32_t* table_out,
                           int32_t* lens_out, void* workspace, size_t workspace_bytes, int* error_word,
                           cwStream_t stream);

/* Moves the U pages in use to ids [0, U): the used pages at or above U, in
 * order, to the free ids below U, in order; num_used (device int32) receives U
 * and pages [U, num_pages) can be given up.  table_out may be table_in. */
moe_status_t kv_pages_compact(void* caches, size_t cache_stride, int num_caches, int num_pages, size_t page_bytes,
                              int page_size, const int32_t* table_in, int max_pages, const int32_t* lens, int num_seqs,
                              int32_t* table_out, int32_t* num_used, void* workspace, size_t workspace_bytes,
                              int* error_word, cwStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* TIME_B200_KV_CACHE_H */
