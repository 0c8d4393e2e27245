// Per-head products of the absorbed form: y[t, h, :] = W[h] x[t, h, :].
//
// q_lat[h] = W_uk[h]^T q_nope[h] before the attention, out[h] = W_uv[h] o_lat[h]
// behind it.  Blocks of 32 outputs by 32 or 64 tokens of one head with
// v_mfma_f32_32x32x16_bf16: A = weight rows, B = token rows, both 16 bytes a
// lane straight from memory (each weight is used once per wave, so LDS would
// only add a hop).  With few tokens the weights' read bounds it, with many the
// latent-wide rows': 128 heads by 64 tokens, 128 to 512 and back, take 9.8 and
// 8.1 us (27 MB each, 2.8 and 3.3 TB/s), 16 heads by 256 tokens 5.8 and 6.0 us.
//
// Sums are float32.  Results are rounded to bf16 once: the next product, on the
// matrix cores, takes bf16.  Of q_lat that moves a score by 2^-8 of its size at most
// (both parts of a split q_lat would double the scores' products), of o_lat
// the result by as much as its own rounding does.
#include "latent_attend.h"
#include "pa_errors.h"
#include "../../include/latent_attention.h"

namespace pa {
namespace {

// kSplit = 1: a workgroup's four waves take 32 outputs each with the whole
// depth; kSplit = 4: they split the depth and share 64 outputs, whose sums go
// through LDS.  A wave's part, kDepth deep, is all in flight before the first
// product.  Results go out through LDS, 256 (128) contiguous bytes of a token.
template <int MB, int kDepth, int kSplit>
__global__ void __launch_bounds__(256) head_product_kernel(HeadProduct p, int n_groups) {
  constexpr int kSteps = kDepth / 16, kNb = kSplit == 1 ? 1 : 2;
  constexpr int kOuts = kSplit == 1 ? 128 : 64, kChunks = kOuts / 8;  // of the workgroup
  __shared__ f32x4 part[kSplit == 1 ? 1 : 4][kSplit == 1 ? 1 : MB][4][64];
  __shared__ u32x4 tile[32 * MB][kChunks];
  const int lane = threadIdx.x & 63;
  const int h2 = lane >> 5, l = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int head = blockIdx.y;
  const int mb = blockIdx.x / n_groups, ng = blockIdx.x - mb * n_groups;
  const int nb0 = kSplit == 1 ? 4 * ng + wave : 2 * ng;  // first 32-output block
  const int k0 = kSplit == 1 ? 0 : wave * kDepth;
  bf16x8 a[kSteps], b[MB][kSteps];
  const uint16_t* w = p.w + head * p.w_hs + (int64_t)(32 * nb0 + l) * (kDepth * kSplit) + k0 + 8 * h2;
#pragma unroll
  for (int s = 0; s < kSteps; ++s) a[s] = as_bf16x8(ld16(w + 16 * s));
#pragma unroll
  for (int m = 0; m < MB; ++m) {
    const int t = min((mb * MB + m) * 32 + l, p.tokens - 1);
    const uint16_t* x = p.x + t * p.x_ts + head * p.x_hs + k0 + 8 * h2;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) b[m][s] = as_bf16x8(ld16(x + 16 * s));
  }
  __builtin_amdgcn_sched_barrier(0);  // all of them in flight
  // outputs 8 q + 4 h2 .. + 3 of a block for token 32 m + l: half h2 of chunk 4 block + q
  auto put = [&](int m, int block, int q, const f32x4& v) __attribute__((always_inline)) {
    const int r = 32 * m + l, c = (4 * block + q) ^ (r & (kChunks - 1));
    reinterpret_cast<u32x2*>(&tile[r][c])[h2] = u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
  };
#pragma unroll
  for (int nb = 0; nb < kNb; ++nb) {
    f32x16 acc[MB] = {};
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int m = 0; m < MB; ++m) acc[m] = mfma32(a[s], b[m][s], acc[m]);
    if (nb + 1 < kNb) {
      w += (int64_t)32 * (kDepth * kSplit);
#pragma unroll
      for (int s = 0; s < kSteps; ++s) a[s] = as_bf16x8(ld16(w + 16 * s));
      __builtin_amdgcn_sched_barrier(0);
    }
    // lane (l, h2) holds token l, outputs 8 q + 4 h2 + i
    if constexpr (kSplit == 1) {
#pragma unroll
      for (int m = 0; m < MB; ++m)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          put(m, wave, q, f32x4{acc[m][4 * q], acc[m][4 * q + 1], acc[m][4 * q + 2], acc[m][4 * q + 3]});
    } else {
      if (nb > 0) __syncthreads();  // the sums of the block before are taken
#pragma unroll
      for (int m = 0; m < MB; ++m)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          part[wave][m][q][lane] = f32x4{acc[m][4 * q], acc[m][4 * q + 1], acc[m][4 * q + 2], acc[m][4 * q + 3]};
      __syncthreads();
      // wave q sums quarter q
#pragma unroll
      for (int m = 0; m < MB; ++m)
        put(m, nb, wave, (part[0][m][wave][lane] + part[1][m][wave][lane]) +
                             (part[2][m][wave][lane] + part[3][m][wave][lane]));
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 32 * MB * kChunks / 256; ++i) {
    const int e = i * 256 + threadIdx.x, r = e / kChunks, c = e & (kChunks - 1);
    const int t = mb * MB * 32 + r;
    if (t >= p.tokens) continue;
    u32x4 v = tile[r][c ^ (r & (kChunks - 1))];
    if (p.cu_q && !token_in_sequence(p.cu_q, p.batch, p.max_q, t)) {
      if (!p.zero_rest) continue;
      v = u32x4{0, 0, 0, 0};
    }
    st16(p.y + t * p.y_ts + head * p.y_hs + kOuts * ng + 8 * c, v);
  }
}

template <int kDepth, int kSplit>
void launch(const HeadProduct& p, hipStream_t s) {
  const int n_groups = p.n / (kSplit == 1 ? 128 : 64);
  // 64 tokens a wave from 33 on: 33, 64 and 256 tokens by 128 heads, both
  // products and the attention of two tiles between them: 29.1, 31.9, 81.4 us
  // against 33.8, 35.0, 90.0 with 32; 16 tokens 27.2 against 25.6
  const bool two = p.tokens > 32;
  const int m_blocks = (p.tokens + (two ? 63 : 31)) / (two ? 64 : 32);
  const dim3 g((unsigned)(n_groups * m_blocks), (unsigned)p.heads);
  if (two) head_product_kernel<2, kDepth, kSplit><<<g, 256, 0, s>>>(p, n_groups);
  else head_product_kernel<1, kDepth, kSplit><<<g, 256, 0, s>>>(p, n_groups);
}

}  // namespace

int head_product_launch(const char* name, const HeadProduct& p, hipStream_t s) {
  // (absorbing: depth 64 or 128 to a latent size; projecting: a latent size to 64 or 128)
  switch (p.k) {
    case 64: launch<64, 1>(p, s); break;
    case 128: launch<128, 1>(p, s); break;
    case 256: launch<64, 4>(p, s); break;
    case 512: launch<128, 4>(p, s); break;
    default: return fail(PA_ERR_UNSUPPORTED, "%s: depth %d", name, p.k);
  }
  return launch_status(name);
}

}  // namespace pa
