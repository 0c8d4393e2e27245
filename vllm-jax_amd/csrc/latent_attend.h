// Launchers of the latent-attention kernels, called by the C entries.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "latent.h"

namespace pa {

// Per-head products y[t, h, :] = W[h] x[t, h, :] (latent_product.hip): W[h] is
// [n, k] contiguous; k 64 or 128 with n a multiple of 128, or k 256 or 512 with n
// a multiple of 64.
struct HeadProduct {
  const uint16_t* x;
  int64_t x_ts, x_hs;
  const uint16_t* w;
  int64_t w_hs;
  uint16_t* y;
  int64_t y_ts, y_hs;
  int32_t tokens, heads, n, k;
  // With cu_q: tokens outside the sequences, or past max_q of theirs, get a zero
  // row (zero_rest) or are left alone.
  const int32_t* cu_q = nullptr;
  int32_t batch = 0, max_q = 0;
  bool zero_rest = false;
};
// Whether token t is one of the first max_q of a sequence of cu_q.
__device__ __forceinline__ bool token_in_sequence(const int32_t* cu_q, int batch, int max_q, int t) {
  if (batch <= 0 || t < cu_q[0] || t >= cu_q[batch]) return false;
  int lo = 0, hi = batch;  // last b with cu_q[b] <= t
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu_q[mid] <= t) lo = mid;
    else hi = mid;
  }
  return t - cu_q[lo] < max_q;
}
int head_product_launch(const char* name, const HeadProduct& p, hipStream_t s);

// Absorbed-form attention (latent_decode.hip): rows are (token, head) pairs of
// a sequence, keys the cache rows themselves, values their latent part.
struct LatentAttn {
  const uint16_t* q_lat;  // [T, H, R]
  int64_t ql_ts, ql_hs;
  const uint16_t* q_rope;  // [T, H, Dr]
  int64_t qr_ts, qr_hs;
  LatentPool pool;
  const int32_t* cu_q;    // null: token b is sequence b's only one
  const int32_t* cu_k;    // kv lengths as differences, or
  const int32_t* kv_lens;  // as they are
  int32_t batch, num_tokens, heads, max_q;
  float scale;
  uint16_t* out;  // [T, H, R]
  int64_t o_ts, o_hs;
};
// Workspace bytes of an absorbed launch; 0 with *why set: sizes out of range.
size_t latent_attn_workspace(int32_t batch, int32_t max_q, int32_t heads, int32_t latent, int64_t span,
                             const char** why);
int latent_attn_launch(const char* name, const LatentAttn& a, int latent, int rope, void* workspace, hipStream_t s);

// Expanded form (latent_expand.hip, latent_prefill.hip).  The cache rows of all
// sequences, laid end to end by cu_k, become K and V rows of `heads` heads from
// `head0` on: kv [heads][cap][nope + v], and (k_rope not null) the rotary parts
// k_rope [cap][rope].  Tokens from cap on are dropped.
//
// First row of sequence b among them.  cu_k may hold lengths past the span of a
// block-table row, which are clamped to it: rows start where the lengths before
// would end, but no later than b spans (the clamped lengths still fit between).
__device__ __forceinline__ int64_t flat_start(const int32_t* cu_k, int b, int64_t span) {
  return min((int64_t)cu_k[b] - cu_k[0], (int64_t)b * span);
}
struct LatentExpand {
  LatentPool pool;
  const int32_t* cu_k;
  int32_t batch, cap, head0, heads;
  const uint16_t* w_kv;  // [H][nope + v][latent]
  uint16_t* kv;
  uint16_t* k_rope;
};
int latent_expand_launch(const char* name, const LatentExpand& p, int latent, int rope, int nope, hipStream_t s);

// Ragged causal attention over them: row i of sequence b sees its first
// lk - lq + i + 1 keys.
struct LatentRagged {
  const uint16_t* q_nope;
  int64_t qn_ts, qn_hs;
  const uint16_t* q_rope;
  int64_t qr_ts, qr_hs;
  const uint16_t* kv;
  const uint16_t* k_rope;
  const int32_t* cu_q;
  const int32_t* cu_k;
  int32_t batch, num_tokens, max_q, cap, heads, span;  // span: of a block-table row
  float scale;
  uint16_t* out;
  int64_t o_ts, o_hs;
  // Workgroups past the items zero the rows of zero_heads heads that belong to
  // no sequence, from zero_out on (null: none).
  uint16_t* zero_out;
  int32_t zero_heads;
};
int latent_ragged_launch(const char* name, const LatentRagged& p, int nope, int rope, hipStream_t s);

}  // namespace pa
