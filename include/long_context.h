/*
 * C ABI of decode over long cached contexts that reads less than all of them
 * (part of libpaged_attention.so): attention over the blocks of a context that
 * a cheap score selects for each query, and attention of sequences that share
 * a prefix.
 *
 * Conventions are those of paged_attention.h (device pointers, strides in
 * elements with an innermost stride of 1, stream-ordered, no allocation, no
 * synchronisation, PA_* return codes; negative block-table entries read page
 * 0, entries past the pool are clamped into it, lengths are clamped to the
 * block table's span).  bf16 keys and values; K and V pools are addressed by
 * one set of page, slot and head strides.  All bf16 operands 16-byte aligned
 * with strides multiple of 8.  Cached rows below a length have to be finite;
 * rows behind it are never used.
 *
 * A block is `block` tokens, a multiple of 16 that divides the page: block j of
 * a sequence holds its tokens [j block, (j + 1) block), and lies in page
 * j block / page_size of its table.  head_dim 64, 128 or 256.
 */
#ifndef VLLM_JAX_AMD_LONG_CONTEXT_H_
#define VLLM_JAX_AMD_LONG_CONTEXT_H_

#include <stddef.h>
#include <stdint.h>

#include "paged_attention.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * bounds[page, part of the page, kv head] = [ min | max ] over the block's
 * tokens below lengths[b], per element of the key, for every block that holds
 * one of the last n_b tokens of sequence b: n_b = cu_seqlens_q[b + 1] -
 * cu_seqlens_q[b], or 1 where cu_seqlens_q is NULL; max_seqlen_q is the largest
 * n_b (it sizes the launch; longer ones take longer and are not cut).  The keys
 * are in the pool already.  Blocks whose table entry is not a page of the pool
 * are left out, and all other blocks' bounds are left as they were.  bounds:
 * [num_pages, page_size / block, num_kv_heads, 2, head_dim] with the two rows
 * of a head adjacent.
 */
int pa_block_bounds(const uint16_t* k_cache, int32_t num_pages, int32_t page_size, int64_t page_stride,
                    int64_t slot_stride, int64_t head_stride, const int32_t* block_tables, int64_t bt_stride,
                    int32_t pages_per_seq, const int32_t* lengths, const int32_t* cu_seqlens_q, int32_t batch,
                    int32_t max_seqlen_q, int32_t num_kv_heads, int32_t head_dim, int32_t block,
                    uint16_t* bounds, int64_t bounds_page_stride, int64_t bounds_block_stride,
                    int64_t bounds_head_stride, void* stream);

/*
 * scores[b, kv head, j] = scale * max over the kv head's q heads of
 * sum_d max(q_d min_d, q_d max_d), which no scaled logit of block j exceeds
 * (but for the roundings of the 32-bit sums);
 * -inf for blocks that start at or past lengths[b].  scale > 0.  q: [batch,
 * num_heads, head_dim]; scores: float32 [batch, num_kv_heads, pages_per_seq *
 * page_size / block].
 */
int pa_block_scores(const uint16_t* q, int64_t q_batch_stride, int64_t q_head_stride, const uint16_t* bounds,
                    int32_t num_pages, int32_t page_size, int64_t bounds_page_stride, int64_t bounds_block_stride,
                    int64_t bounds_head_stride, const int32_t* block_tables, int64_t bt_stride,
                    int32_t pages_per_seq, const int32_t* lengths, int32_t batch, int32_t num_heads,
                    int32_t num_kv_heads, int32_t head_dim, int32_t block, float scale, float* scores,
                    int64_t scores_batch_stride, int64_t scores_head_stride, void* stream);

/*
 * For each sequence and kv head the indices of `num_selected` of its n =
 * ceil(lengths[b] / block) blocks, ascending: the first `first`, the last
 * `recent`, and of the others those of the largest scores, equal scores by
 * the lower index, NaN below all numbers; all n, then -1, where n <=
 * num_selected.  n is clamped to the scores' width.  first + recent <=
 * num_selected.  selected: int32 [batch, num_kv_heads, num_selected].
 */
int pa_select_blocks(const float* scores, int64_t scores_batch_stride, int64_t scores_head_stride, int32_t width,
                     const int32_t* lengths, int32_t batch, int32_t num_kv_heads, int32_t block,
                     int32_t num_selected, int32_t first, int32_t recent, int32_t* selected,
                     int64_t selected_batch_stride, int64_t selected_head_stride, void* stream);

/*
 * One new token a sequence over its selected blocks: out[b, h] = softmax over
 * the tokens below lengths[b] of the blocks selected[b, kv head of h], of
 * scale * q . K (soft-capped where soft_cap > 0), times V.  Entries of
 * `selected` that are not a block of the sequence are skipped, in any place;
 * a block that stands twice counts twice.  A row without a token is zero.
 */
size_t pa_block_sparse_decode_workspace_size(int32_t batch, int32_t num_heads, int32_t num_kv_heads,
                                             int32_t head_dim, int32_t num_selected, int32_t block);
int pa_block_sparse_decode(const uint16_t* q, int64_t q_batch_stride, int64_t q_head_stride,
                           const uint16_t* k_cache, const uint16_t* v_cache, int32_t num_pages, int32_t page_size,
                           int64_t page_stride, int64_t slot_stride, int64_t head_stride,
                           const int32_t* block_tables, int64_t bt_stride, int32_t pages_per_seq,
                           const int32_t* lengths, int32_t batch, int32_t num_heads, int32_t num_kv_heads,
                           int32_t head_dim, const int32_t* selected, int64_t selected_batch_stride,
                           int64_t selected_head_stride, int32_t num_selected, int32_t block, float scale,
                           float soft_cap, uint16_t* out, int64_t out_batch_stride, int64_t out_head_stride,
                           void* workspace, size_t workspace_bytes, void* stream);

/*
 * Attention of new tokens whose sequences share prefixes in groups: group g is
 * sequences cu_groups[g] .. cu_groups[g + 1] - 1, whose first shared_lens[g]
 * tokens lie in the same pages.  Sequence b's new tokens are rows
 * cu_seqlens_q[b] .. cu_seqlens_q[b + 1] - 1 of q and out (at most
 * max_seqlen_q of them; cu_seqlens_q NULL: row b, one new token each); row i
 * of n sees the first lengths[b] - n + i + 1 of the sequence's tokens, as in
 * pa_decode and pa_prefill, and is zero if that is none.  The shared tokens are
 * read once a group, through the block table of its first sequence that has
 * tokens; shared_lens is rounded down to 64 tokens, cut to the group's shortest
 * length (sequences without tokens aside), and taken for 0 in groups of fewer than
 * two sequences.  Sequences outside all groups share nothing; cu_groups and cu_seqlens_q
 * do not fall (where they do, rows may be zero).
 * Rows outside the sequences are zeroed with zero_rest and left as they were
 * without.  head_dim 128, up to 256 q heads a kv head, any page size.  The
 * workspace (256-byte aligned) is sized with ragged = (cu_seqlens_q != NULL).
 */
size_t pa_shared_prefix_workspace_size(int32_t batch, int32_t num_groups, int32_t num_tokens, int32_t max_seqlen_q,
                                       int32_t ragged, int32_t num_heads, int32_t num_kv_heads,
                                       int32_t pages_per_seq, int32_t page_size);
int pa_shared_prefix(const uint16_t* q, int64_t q_tok_stride, int64_t q_head_stride, const uint16_t* k_cache,
                     const uint16_t* v_cache, int32_t num_pages, int32_t page_size, int64_t page_stride,
                     int64_t slot_stride, int64_t head_stride, const int32_t* block_tables, int64_t bt_stride,
                     int32_t pages_per_seq, const int32_t* lengths, const int32_t* cu_groups,
                     const int32_t* shared_lens, int32_t num_groups, const int32_t* cu_seqlens_q, int32_t batch,
                     int32_t num_tokens, int32_t max_seqlen_q, int32_t num_heads, int32_t num_kv_heads,
                     int32_t head_dim, float scale, float soft_cap, int32_t zero_rest, uint16_t* out,
                     int64_t out_tok_stride, int64_t out_head_stride, void* workspace, size_t workspace_bytes,
                     void* stream);

#ifdef __cplusplus
}
#endif

#endif /* VLLM_JAX_AMD_LONG_CONTEXT_H_ */
