// Per-head products of the absorbed form: y[t, h, :] = W[h] x[t, h, :].
//
// q_lat[h] = W_uk[h]^T q_nope[h] before the attention, out[h] = W_uv[h] o_lat[h]
// behind it.  A wave computes 32 outputs for 32 or 64 tokens of one head with
// v_mfma_f32_32x32x16_bf16: A = weight rows, B = token rows, both 16 bytes a
// lane straight from memory (each weight is used once per wave, so LDS would
// only add a hop).  With few tokens the weights' read bounds it.
#include "latent_attend.h"
#include "pa_errors.h"
#include "../../include/latent_attention.h"

namespace pa {
namespace {

constexpr int kStep = 64;  // k values in flight

template <int MB>
__global__ void __launch_bounds__(256) head_product_kernel(HeadProduct p, int n_blocks, int m_blocks) {
  const int lane = threadIdx.x & 63;
  const int h2 = lane >> 5, l = lane & 31;
  const int gw = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4 + (threadIdx.x >> 6)));
  const int head = blockIdx.y;
  const int mb = gw / n_blocks, nb = gw - mb * n_blocks;
  if (mb >= m_blocks) return;
  const uint16_t* w = p.w + head * p.w_hs + (int64_t)(32 * nb + l) * p.k + 8 * h2;
  const uint16_t* x[MB];
#pragma unroll
  for (int m = 0; m < MB; ++m) {
    const int t = min((mb * MB + m) * 32 + l, p.tokens - 1);
    x[m] = p.x + t * p.x_ts + head * p.x_hs + 8 * h2;
  }
  f32x16 acc[MB] = {};
  for (int k0 = 0; k0 < p.k; k0 += kStep) {
    bf16x8 a[kStep / 16], b[MB][kStep / 16];
#pragma unroll
    for (int s = 0; s < kStep / 16; ++s) {
      a[s] = as_bf16x8(ld16(w + k0 + 16 * s));
#pragma unroll
      for (int m = 0; m < MB; ++m) b[m][s] = as_bf16x8(ld16(x[m] + k0 + 16 * s));
    }
#pragma unroll
    for (int s = 0; s < kStep / 16; ++s)
#pragma unroll
      for (int m = 0; m < MB; ++m) acc[m] = mfma32(a[s], b[m][s], acc[m]);
  }
  // lane (l, h2) holds token l, outputs 8 (i / 4) + 4 h2 + i % 4
#pragma unroll
  for (int m = 0; m < MB; ++m) {
    const int t = (mb * MB + m) * 32 + l;
    if (t >= p.tokens) continue;
    if (p.cu_q && !token_in_sequence(p.cu_q, p.batch, p.max_q, t)) {
      if (!p.zero_rest) continue;
      acc[m] = f32x16{};
    }
    uint16_t* y = p.y + t * p.y_ts + head * p.y_hs + 32 * nb + 4 * h2;
#pragma unroll
    for (int q = 0; q < 4; ++q)
      *reinterpret_cast<u32x2*>(y + 8 * q) =
          u32x2{pack_bf16x2(acc[m][4 * q], acc[m][4 * q + 1]), pack_bf16x2(acc[m][4 * q + 2], acc[m][4 * q + 3])};
  }
}

}  // namespace

int head_product_launch(const char* name, const HeadProduct& p, hipStream_t s) {
  const int n_blocks = p.n / 32;
  const bool two = p.tokens > 32;
  const int m_blocks = (p.tokens + (two ? 63 : 31)) / (two ? 64 : 32);
  const int64_t waves = (int64_t)n_blocks * m_blocks;
  const dim3 g((unsigned)((waves + 3) / 4), (unsigned)p.heads);
  if (two) head_product_kernel<2><<<g, 256, 0, s>>>(p, n_blocks, m_blocks);
  else head_product_kernel<1><<<g, 256, 0, s>>>(p, n_blocks, m_blocks);
  return launch_status(name);
}

}  // namespace pa
