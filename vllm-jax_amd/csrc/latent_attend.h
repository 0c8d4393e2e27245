// Launchers of the latent-attention kernels, called by the C entries.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "latent.h"

namespace pa {

// Per-head products y[t, h, :] = W[h] x[t, h, :] (latent_product.hip): W[h] is
// [n, k] with contiguous rows, k 64 .. 512 a multiple of 64, n a multiple of 32.
struct HeadProduct {
  const uint16_t* x;
  int64_t x_ts, x_hs;
  const uint16_t* w;
  int64_t w_hs;
  uint16_t* y;
  int64_t y_ts, y_hs;
  int32_t tokens, heads, n, k;
};
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

}  // namespace pa
