/*
 * mvme_long.h -- C ABI of the operators for long contexts, in the same shared
 * object and under the same conventions as mvme_paged.h (device pointers,
 * int64 metadata, status codes, the caller's stream, no allocation and no
 * synchronisation): decode attention over prefixes that sequences share,
 * attention that keeps account of the weight each cached token receives, and
 * the eviction of those that receive least.  Caches are the 16-bit ones of
 * mvme_paged.h, 16-byte aligned.
 */
#ifndef MVME_LONG_H
#define MVME_LONG_H

#include "mvme_paged.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Bytes of device workspace mvme_paged_attention_shared_prefix needs for these
 * shapes (0: none, or shapes that it refuses).  Pure host function.
 */
size_t mvme_paged_attention_shared_prefix_workspace_size(int64_t batch, int64_t q_heads, int64_t kv_heads,
                                                         int64_t head_dim, int64_t groups, int64_t block_size,
                                                         int64_t table_width, int always);

/*
 * mvme_paged_attention for a batch in which sequences share prefixes.  Group g
 * is the sequences group_offsets[g] .. group_offsets[g + 1] - 1 (offsets rise
 * from 0 or more to at most batch; sequences in no group share nothing); the
 * first prefix_lens[g] tokens of all of them are in the same pages and are read
 * once for all, through the table of the group's first sequence that has them
 * all (on pages of a multiple of 16 tokens, whole runs of 16 of them: the rest
 * is read with each sequence's own tokens).  Sequences of a group that are
 * shorter than its prefix (the empty ones of a padded batch) are attended
 * through their own tables, as are groups of one and of a prefix that is not
 * positive or passes the tables' capacity.  Offsets that fall, or leave the
 * batch, make all sequences ungrouped.  Every row's result is that of
 * mvme_paged_attention, to rounding: scale 1/sqrt(head_dim), zeros for lengths
 * <= 0 or beyond the table's capacity, pages out of range skipped.
 * Calls of few cached tokens (by the tables' capacity) are attended without
 * regard to the groups, as is every call without groups: by
 * mvme_paged_attention; always != 0 shares at any size.  Where prefixes are
 * shared scores, softmax statistics and
 * accumulators are fp32; for the value product the probabilities are rounded to
 * the inputs' type where a prefix has more than 32 query rows, and to the sum
 * of two numbers of it elsewhere.  In fp16 they are finite while scores (times
 * log2 e) are below 2^24 in magnitude, and in prefixes of more than 32 rows
 * those below 2^-33 of the largest may be zero, which makes an infinite value
 * NaN there.
 */
int mvme_paged_attention_shared_prefix(void* out, const void* query, const void* key_cache, const void* value_cache,
                                       const int64_t* block_tables, const int64_t* context_lens,
                                       const int64_t* group_offsets, const int64_t* prefix_lens,
                                       int64_t batch, int64_t groups, int64_t q_heads, int64_t kv_heads,
                                       int64_t head_dim, int64_t num_blocks, int64_t block_size, int64_t table_width,
                                       int always, int dtype, void* workspace, size_t workspace_bytes, void* stream);

/*
 * Bytes of device workspace mvme_paged_attention_weights needs for these
 * shapes: 4 per query head and token of the tables' capacity, and the pieces of
 * split sequences; 0 where sequences are taken whole, or for shapes that it
 * refuses.  Pure host function.
 */
size_t mvme_paged_attention_weights_workspace_size(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                                                   int64_t block_size, int64_t table_width);

/*
 * mvme_paged_attention, and
 *   weights[b, hk, j] += sum of the probabilities that the query heads of kv
 *                        head hk give token j,   j < context_lens[b]
 * with fp32 weights [batch, kv_heads, weight_row] (weight_row at least
 * block_size * table_width).  Entries behind the context, and of sequences
 * whose length cannot be, stay; tokens in pages out of range receive nothing.
 * The probabilities added are fp32; for the value product they are rounded to
 * the sum of two numbers of the inputs' type.
 */
int mvme_paged_attention_weights(void* out, const void* query, const void* key_cache, const void* value_cache,
                                 const int64_t* block_tables, const int64_t* context_lens, float* weights,
                                 int64_t weight_row, int64_t batch, int64_t q_heads, int64_t kv_heads,
                                 int64_t head_dim, int64_t num_blocks, int64_t block_size, int64_t table_width,
                                 int dtype, void* workspace, size_t workspace_bytes, void* stream);

/*
 * Bytes of device workspace mvme_prefill_attention_weights needs (0 for shapes
 * that it refuses, or no tokens).  Pure host function.
 */
size_t mvme_prefill_attention_weights_workspace_size(int64_t num_seqs, int64_t total_tokens, int64_t q_heads,
                                                     int64_t kv_heads, int64_t head_dim, int64_t block_size,
                                                     int64_t table_width);

/*
 * What a prompt's queries add to the weights: with the queries and metadata of
 * mvme_paged_prefill_attention (packed row i of sequence s sits at position
 * query_starts[s] + i and sees the keys up to it),
 *   weights[s, hk, j] += sum over the rows i of s and the query heads of hk of
 *                        the probability that they give token j.
 * The rows may be all of a prompt's or its last ones (then query_starts is
 * where these begin).  Keys are read from the cache; values are not needed.
 * Rows that no sequence owns, and rows that see no key, add nothing; a
 * sequence whose start or length cannot be is left out.
 */
int mvme_prefill_attention_weights(const void* q, const void* key_cache, const int64_t* cu_seqlens_q,
                                   const int64_t* query_starts, const int64_t* block_tables,
                                   const int64_t* context_lens, float* weights, int64_t weight_row, int64_t num_seqs,
                                   int64_t total_tokens, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                                   int64_t num_blocks, int64_t block_size, int64_t table_width, int dtype,
                                   void* workspace, size_t workspace_bytes, void* stream);

/*
 * Eviction.  For every layer, sequence b and kv head: of the n =
 * context_lens[b] cached tokens `keep` stay where n > keep, else all.  These
 * are the first f = min(first[b], keep) (first may be NULL: none), the last
 * r = min(recent, keep - f), and of those between the keep - f - r with the
 * largest weights: NaN above every number, -0 equal to +0, ties to the lowest
 * position.  Their key and value rows of the kv head move, in order, to the
 * positions 0 .. keep - 1 of the sequence's pages, in place; rows behind these
 * keep what they held.  kept[l, b, hk, i] is the position that row i came
 * from, -1 behind the last; new_weights its weight, 0 behind the last;
 * new_lens[b] = min(n, keep).  A sequence whose length is not positive (an
 * empty one of a padded batch) or passes the tables' capacity keeps its length
 * and nothing of it moves; nothing of it is kept, so that its new_weights are 0
 * and its kept -1: whoever needs its weights again has them in `weights`, which
 * stay as they were.  Rows from or to a page out of range are not moved.
 *   key_cache, value_cache  [layers, num_blocks, block_size, kv_heads, head_dim],
 *                           head_dim a multiple of 8 up to 1024
 *   weights, new_weights    fp32 [layers, batch, kv_heads, weight_row], not
 *                           overlapping; weight_row >= block_size * table_width
 *   kept                    [layers, batch, kv_heads, min(keep, weight_row)]
 * No page that rows move into (positions f and up) may be in two of the
 * tables, or held by anyone else.
 */
int mvme_evict_kv_cache(void* key_cache, void* value_cache, const float* weights, float* new_weights,
                        int64_t weight_row, int64_t* kept, int64_t* new_lens, const int64_t* block_tables,
                        const int64_t* context_lens, const int64_t* first, int64_t layers, int64_t batch,
                        int64_t kv_heads, int64_t head_dim, int64_t num_blocks, int64_t block_size,
                        int64_t table_width, int64_t keep, int64_t recent, int dtype, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MVME_LONG_H */
