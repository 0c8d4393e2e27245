/*
 * C ABI of latent attention and of the rotation beside it (part of
 * libpaged_attention.so): attention whose cache holds one latent vector and
 * one rotated key part a token in place of K and V rows per head.
 *
 *   cache row   [ c (latent_dim) | k_r (rope_dim) ], bf16
 *   K[h]      = [ W_uk[h] c | k_r ]         W_uk[h]: [nope_dim, latent_dim]
 *   V[h]      =   W_uv[h] c                 W_uv[h]: [v_dim, latent_dim]
 *   out[h]    = sum_j softmax_j(scale * q[h] . K[h]_j) V[h]_j
 *
 * Conventions are those of paged_attention.h (device pointers, strides in
 * elements with an innermost stride of 1, stream-ordered, no allocation, no
 * synchronisation, PA_* return codes).  Pools are [num_pages, page_size,
 * latent_dim + rope_dim] with caller-given page and slot strides; negative
 * block-table entries read page 0, entries past the pool are clamped into it,
 * kv lengths are clamped to the block table's span.  Cached rows below a kv
 * length have to be finite.  Supported: latent_dim 256
 * or 512, rope_dim 32 or 64, nope_dim = v_dim = 64 or 128, any page size, any
 * number of heads; all operands 16-byte aligned with strides multiple of 8.
 */
#ifndef VLLM_JAX_AMD_LATENT_ATTENTION_H_
#define VLLM_JAX_AMD_LATENT_ATTENTION_H_

#include <stddef.h>
#include <stdint.h>

#include "paged_attention.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of pa_rotary_embedding. */
#define PA_DTYPE_BF16 0
#define PA_DTYPE_FP16 1
#define PA_DTYPE_FP32 2

/*
 * Rotation of elements [start, start + rotary_dim) of every head: pair i is
 * (2i, 2i + 1) of them (interleaved) or (i, i + rotary_dim / 2), its angle
 * positions[t] * inv_freq[i] (evaluated in float64), and cos and sin are
 * multiplied by `amplitude`.  Other elements are copied.  x, out:
 * [num_tokens, num_heads, head_dim]; out may be x (same strides).  Any
 * alignment; rotary_dim even, up to 512.
 */
int pa_rotary_embedding(int32_t dtype, const void* x, int64_t x_tok_stride, int64_t x_head_stride,
                        const int32_t* positions, const double* inv_freq, float amplitude,
                        int32_t num_tokens, int32_t num_heads, int32_t head_dim, int32_t start,
                        int32_t rotary_dim, int32_t interleaved, void* out, int64_t out_tok_stride,
                        int64_t out_head_stride, void* stream);

/*
 * cache[slot[t]] = [ latent[t] * norm_weight / rms(latent[t]) | rope(k_rope[t]) ]
 * for every token whose slot lies in the pool (others are skipped), and q_out
 * = rope(q_rope) for all tokens; norm_weight NULL stores the latent rows as
 * they come, num_heads 0 leaves q out, q_out may be q_rope (same strides).  Slots
 * must be unique.
 */
int pa_latent_store(const uint16_t* latent, int64_t latent_tok_stride, const uint16_t* k_rope,
                    int64_t k_rope_tok_stride, const uint16_t* norm_weight, float eps,
                    const double* inv_freq, float amplitude, int32_t interleaved,
                    const int32_t* positions, const int32_t* slot_mapping, int32_t num_tokens,
                    int32_t latent_dim, int32_t rope_dim, const uint16_t* q_rope, int64_t q_tok_stride,
                    int64_t q_head_stride, int32_t num_heads, uint16_t* q_out, int64_t q_out_tok_stride,
                    int64_t q_out_head_stride, uint16_t* cache, int32_t num_pages, int32_t page_size,
                    int64_t page_stride, int64_t slot_stride, void* stream);

/*
 * One new token a sequence, absorbed form: q_nope [batch, num_heads, nope_dim],
 * q_rope [batch, num_heads, rope_dim] (rotated) against the first lengths[b]
 * rows of sequence b; out [batch, num_heads, v_dim].  A length of zero gives a
 * zero row.  w_kv: contiguous [num_heads, nope_dim + v_dim, latent_dim] (W_uk
 * rows, then W_uv rows of each head); w_uk_t: its W_uk transposed, contiguous
 * [num_heads, latent_dim, nope_dim].  Up to 16384 sequences.
 */
size_t pa_latent_decode_workspace_size(int32_t batch, int32_t num_heads, int32_t latent_dim,
                                       int32_t pages_per_seq, int32_t page_size);
int pa_latent_decode(const uint16_t* q_nope, int64_t qn_tok_stride, int64_t qn_head_stride,
                     const uint16_t* q_rope, int64_t qr_tok_stride, int64_t qr_head_stride,
                     const uint16_t* cache, int32_t num_pages, int32_t page_size, int64_t page_stride,
                     int64_t slot_stride, const int32_t* block_tables, int64_t bt_stride,
                     int32_t pages_per_seq, const int32_t* lengths, int32_t batch, int32_t num_heads,
                     int32_t latent_dim, int32_t rope_dim, int32_t nope_dim, int32_t v_dim,
                     const uint16_t* w_uk_t, const uint16_t* w_kv, float scale, uint16_t* out,
                     int64_t out_tok_stride, int64_t out_head_stride, void* workspace,
                     size_t workspace_bytes, void* stream);

/*
 * Ragged causal prefill: q_nope [num_tokens, num_heads, nope_dim], q_rope
 * [num_tokens, num_heads, rope_dim] (rotated); sequence b has rows
 * cu_seqlens_q[b] .. cu_seqlens_q[b + 1] (the first max_seqlen_q of them are
 * computed) over lk cached ones, itself among them, given by cu_seqlens_k or by
 * kv_lens (one of the two); row i sees the first lk - lq + i + 1.  A row that sees none is
 * zero; rows outside the sequences are zeroed with zero_rest, else left alone.
 * total_kv bounds the sum of the kv lengths (of cu_seqlens_k as it stands, or batch
 * times the block table's span) and has to hold (rows past it may be left out).
 *
 * pa_latent_prefill_route says which form a launch takes: K and V expanded for
 * a group of heads at a time, or the absorbed form of pa_latent_decode for few
 * new tokens behind long contexts and, where it needs less memory, for a total_kv
 * whose expanded rows of one head would pass 8 GiB; the workspace follows it.
 * 1 .. 65535 heads.
 */
#define PA_LATENT_EXPANDED 0
#define PA_LATENT_ABSORBED 1
int pa_latent_prefill_route(int32_t batch, int32_t num_tokens, int32_t max_seqlen_q, int32_t total_kv,
                            int32_t pages_per_seq, int32_t page_size, int32_t num_heads, int32_t latent_dim,
                            int32_t rope_dim, int32_t nope_dim);
size_t pa_latent_prefill_workspace_size(int32_t batch, int32_t num_tokens, int32_t max_seqlen_q,
                                        int32_t total_kv, int32_t pages_per_seq, int32_t page_size,
                                        int32_t num_heads, int32_t latent_dim, int32_t rope_dim,
                                        int32_t nope_dim);
int pa_latent_prefill(const uint16_t* q_nope, int64_t qn_tok_stride, int64_t qn_head_stride,
                      const uint16_t* q_rope, int64_t qr_tok_stride, int64_t qr_head_stride,
                      const uint16_t* cache, int32_t num_pages, int32_t page_size, int64_t page_stride,
                      int64_t slot_stride, const int32_t* block_tables, int64_t bt_stride,
                      int32_t pages_per_seq, const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k,
                      const int32_t* kv_lens, int32_t batch, int32_t num_tokens, int32_t max_seqlen_q,
                      int32_t total_kv, int32_t num_heads, int32_t latent_dim, int32_t rope_dim,
                      int32_t nope_dim, int32_t v_dim, const uint16_t* w_uk_t, const uint16_t* w_kv,
                      float scale, int32_t zero_rest, uint16_t* out, int64_t out_tok_stride,
                      int64_t out_head_stride, void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* VLLM_JAX_AMD_LATENT_ATTENTION_H_ */
