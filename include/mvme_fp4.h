/*
 * mvme_fp4.h -- C ABI of the 4-bit paged KV cache and of the cache's page
 * operators, in the same shared object and under the same conventions as
 * mvme_paged.h (device pointers, int64 metadata, status codes, the caller's
 * stream, no allocation and no synchronisation).
 *
 * Packed cache.  One layer's keys (or values) are uint8
 * [num_blocks, kv_heads, record]: a record holds the block_size tokens of one
 * page and kv head, so that an attention work-group reads one contiguous run
 * per page.  In a record come
 *   block_size * head_dim / 2   code bytes, token-major; the low four bits of
 *                               a byte are the even dim,
 *   block_size * head_dim / 32  scale bytes, token-major,
 *   zeros up to a multiple of 16 bytes
 * (mvme_fp4_record_bytes).  A code is E2M1: a sign (bit 3) and one of
 * 0, 0.5, 1, 1.5, 2, 3, 4, 6.  32 consecutive dims of a token share the
 * scale 2^(byte - 127): with a the largest magnitude among them, the
 * smallest power of two in [2^-23, 2^13] with a <= 7 * scale (2^13 if none),
 * and each value is rounded to the nearest code, ties to even, at most 6.  So
 * the value whose error is largest relative to its block is off by half a
 * step of the top interval, and every value of the format is exact in fp16
 * and in bf16.  Magnitudes above 6 * 2^13 (infinities among them) become
 * 6 * 2^13; a block with a NaN has scale byte 255 and reads as NaN.
 * head_dim is a multiple of 32, at most 256 (attention: 32, 64, 96, 128, 192
 * or 256).  Caches are 16-byte aligned.
 */
#ifndef MVME_FP4_H
#define MVME_FP4_H

#include "mvme_paged.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Bytes of one record, or 0 for a block size or head dim that the format does not have. */
int64_t mvme_fp4_record_bytes(int64_t block_size, int64_t head_dim);

/*
 * Quantise and scatter through a slot mapping: for every t < tokens with
 * 0 <= slot_mapping[t] < num_blocks * block_size, token
 * slot_mapping[t] % block_size of page slot_mapping[t] / block_size takes key
 * row t and value row t ([kv_heads, head_dim] of fp16 / bf16, dense,
 * `key_token_stride` / `value_token_stride` elements apart).  Bytes of other
 * tokens stay as they are.
 */
int mvme_fp4_write_slots(void* key_cache, void* value_cache, int64_t num_blocks, int64_t block_size,
                         int64_t kv_heads, int64_t head_dim, const int64_t* slot_mapping,
                         const void* key, const void* value, int64_t tokens,
                         int64_t key_token_stride, int64_t value_token_stride, int dtype, void* stream);

/*
 * The decode step's form: row b goes to position token_offsets[b] of the
 * pages block_tables[b, :] (skipped where the position or the page does not
 * exist).
 */
int mvme_fp4_write_batch(void* key_cache, void* value_cache, int64_t num_blocks, int64_t block_size,
                         int64_t kv_heads, int64_t head_dim, const int64_t* block_tables, int64_t table_width,
                         const int64_t* token_offsets, const void* key, const void* value, int64_t batch,
                         int64_t key_token_stride, int64_t value_token_stride, int dtype, void* stream);

/*
 * Rows of the packed cache in 16 bits (exact): token slot_mapping[t] into
 * row t of key_out / value_out ([tokens, kv_heads, head_dim], dense); rows
 * whose slot does not exist are zeros.
 */
int mvme_fp4_gather_slots(void* key_out, void* value_out, const void* key_cache, const void* value_cache,
                          int64_t num_blocks, int64_t block_size, int64_t kv_heads, int64_t head_dim,
                          const int64_t* slot_mapping, int64_t tokens, int dtype, void* stream);

/* The same for positions [0, token_count) of one sequence's pages block_ids[num_ids]. */
int mvme_fp4_gather(void* key_out, void* value_out, const void* key_cache, const void* value_cache,
                    int64_t num_blocks, int64_t block_size, int64_t kv_heads, int64_t head_dim,
                    const int64_t* block_ids, int64_t num_ids, int64_t token_count, int dtype, void* stream);

/*
 * Bytes of device workspace mvme_fp4_paged_attention needs for these shapes
 * (0 when no sequence is split).  Pure host function.  partition_tokens: 0
 * selects the library's plan, > 0 partitions of that many tokens (rounded up
 * to whole rounds of 128).  At most 34 MB with the library's plan.
 */
size_t mvme_fp4_paged_attention_workspace_size(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                                               int64_t block_size, int64_t table_width, int64_t partition_tokens);

/*
 * GQA decode attention over packed pages, one query token per sequence, with
 * the arguments and the meaning of mvme_paged_attention: scale
 * 1/sqrt(head_dim), sequences of length <= 0 or beyond the table's capacity
 * produce zeros, pages out of range are skipped.  Query and output are fp16
 * or bf16 [batch, q_heads, head_dim]; scores, softmax statistics and
 * accumulators are fp32.  Probabilities are rounded to fp16 for the value
 * product, relative to a reference that keeps the largest between 2^8 and
 * 2^16: they have 11 bits from 2^-22 of the largest on and are lost below
 * 2^-33 of it.  The sum that divides is of the rounded ones.  Scores (with
 * their scale) are meant to stay below 1.1e7 in magnitude, where fp32 still
 * has their differences; rows beyond may come out as NaN.  A NaN block of a
 * key makes a head's output NaN, one of a value the 32 dims that it holds.
 */
int mvme_fp4_paged_attention(void* out, const void* query, const void* key_cache, const void* value_cache,
                             const int64_t* block_tables, const int64_t* context_lens,
                             int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                             int64_t num_blocks, int64_t block_size, int64_t table_width,
                             int64_t partition_tokens, int dtype,
                             void* workspace, size_t workspace_bytes, void* stream);

/*
 * Bytes of device workspace mvme_fp4_paged_prefill_attention needs (0 when no
 * keys are split).  Pure host function.  chunk_tokens: 0 selects the
 * library's plan, > 0 chunks of that many keys (rounded up to whole tiles of
 * 64).
 */
size_t mvme_fp4_paged_prefill_workspace_size(int64_t num_seqs, int64_t total_tokens, int64_t q_heads,
                                             int64_t kv_heads, int64_t head_dim, int64_t block_size,
                                             int64_t table_width, int64_t chunk_tokens);

/*
 * Ragged chunked prefill over packed pages, with the arguments and the
 * meaning of mvme_paged_prefill_attention: packed query row i of sequence s
 * sits at position query_starts[s] + i and attends the keys up to it.  The
 * keys of the chunk itself are read from the cache as well: they are written
 * first.  A NaN block of a key or a value makes all dims of the rows that see
 * its key NaN (decode: only the value's own 32 dims) and touches no others.
 * Scores are bounded as for decode.  Rows that no sequence owns become zeros,
 * by one work-group per kv head: leave few of them.
 */
int mvme_fp4_paged_prefill_attention(void* out, const void* q, const void* key_cache, const void* value_cache,
                                     const int64_t* cu_seqlens_q, const int64_t* query_starts,
                                     const int64_t* block_tables, const int64_t* context_lens,
                                     int64_t num_seqs, int64_t total_tokens,
                                     int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                                     int64_t num_blocks, int64_t block_size, int64_t table_width,
                                     int64_t chunk_tokens, int dtype,
                                     void* workspace, size_t workspace_bytes, void* stream);

/*
 * Copies pages in place: for every plane p < num_planes and every move
 * i < moves, page dst[i] of plane p takes the bytes of page src[i].  planes
 * is [num_planes, num_pages, page_bytes] (a plane is a layer's keys or
 * values, 16-bit or packed).  Moves with a page out of range are skipped.  A
 * page must not be the destination of two moves, nor the destination of one
 * and the source of another: the moves run at the same time.
 */
int mvme_copy_pages(void* planes, int64_t num_planes, int64_t num_pages, int64_t page_bytes,
                    const int64_t* src, const int64_t* dst, int64_t moves, void* stream);

/*
 * Compaction: mvme_copy_pages, and every entry of block_tables (`entries`
 * int64 values) that is src[i] becomes dst[i]; other entries, the padding -1
 * among them, stay.  src has to rise strictly.
 */
int mvme_compact_pages(void* planes, int64_t num_planes, int64_t num_pages, int64_t page_bytes,
                       const int64_t* src, const int64_t* dst, int64_t moves,
                       int64_t* block_tables, int64_t entries, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MVME_FP4_H */
