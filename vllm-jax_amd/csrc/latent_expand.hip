// Expansion of paged latent rows into K and V rows of each head, for the
// expanded form of the prefill.
//
//   kv[h][t] = [ W_uk[h] c_t | W_uv[h] c_t ],   k_rope[t] = the row's rotary part
//
// A matrix product of 256 tokens by one head's outputs per workgroup, depth R,
// v_mfma_f32_32x32x16_bf16 with A = weight rows and B = token rows.  Both come
// 64 deep at a time into a two-stage LDS ring by direct loads, the token rows
// through the block tables.
#include "latent_attend.h"
#include "lds_tiles.h"
#include "pa_errors.h"
#include "../../include/latent_attention.h"

namespace pa {
namespace {

constexpr int kXTokens = 256;
constexpr int kXThreads = 512;
constexpr int kXDepth = 64;  // elements of a k-step: rows of 128 bytes

// Cache row of flat token t (of the sequences laid end to end by cu_k).
__device__ __forceinline__ const uint16_t* flat_row(const LatentExpand& p, int t) {
  int lo = 0, hi = p.batch;  // last b with cu_k[b] - cu_k[0] <= t
  const int base = p.cu_k[0];
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.cu_k[mid] - base <= t) lo = mid;
    else hi = mid;
  }
  const int64_t span = (int64_t)p.pool.pages_per_seq * p.pool.page.d;
  const int j = (int)max((int64_t)0, min((int64_t)t - (p.cu_k[lo] - base), span - 1));
  const int pg = (int)div_by((uint32_t)j, p.pool.page);
  const int page = safe_page(p.pool.tables + lo * p.pool.bt_stride, pg, p.pool.num_pages);
  return p.pool.cache + page * p.pool.page_stride + (int64_t)(j - pg * (int)p.pool.page.d) * p.pool.slot_stride;
}

// N: outputs of a head (nope + v).
template <int N>
__global__ void __launch_bounds__(kXThreads) latent_expand_kernel(LatentExpand p, int latent, int rope) {
  constexpr int kWn = N / 64;                // waves along the outputs, 64 each
  constexpr int kWt = 8 / kWn;               // waves along the tokens
  constexpr int kTb = kXTokens / kWt / 32;   // 32-token blocks of a wave
  constexpr int kXb = kXTokens * 128, kWb = N * 128;  // bytes of a stage
  constexpr int kXDma = kXb / (1024 * 8), kWDma = kWb / (1024 * 8);
  __shared__ __attribute__((aligned(1024))) char smem[2 * (kXb + kWb)];
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void)smem;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int head = blockIdx.x % p.heads, t0 = (blockIdx.x / p.heads) * kXTokens;
  const int total = min(p.cap, p.cu_k[p.batch] - p.cu_k[0]);
  if (t0 >= total) return;

  // This wave's pieces of a stage: 1 KiB blocks of eight rows, lane l row l / 8,
  // chunk l % 8 of it (the logical one is that XOR the row's swizzle).
  const int r8 = lane >> 3, c8 = lane & 7;
  const uint16_t* xr[kXDma];
  const uint16_t* wr[kWDma];
#pragma unroll
  for (int i = 0; i < kXDma; ++i) {
    const int row = 8 * (kXDma * wave + i) + r8;
    xr[i] = flat_row(p, min(t0 + row, total - 1));
    if (p.k_rope && head == 0) {
      // the rotary parts ride along: chunks c8 .. of the same rows
      const uint16_t* src = xr[i] + latent;
      if (8 * c8 < rope && t0 + row < total) st16(p.k_rope + (int64_t)(t0 + row) * rope + 8 * c8, ld16(src + 8 * c8));
    }
    xr[i] += 8 * (c8 ^ swz128(row));
  }
#pragma unroll
  for (int i = 0; i < kWDma; ++i) {
    const int row = 8 * (kWDma * wave + i) + r8;
    wr[i] = p.w_kv + ((int64_t)(p.head0 + head) * N + row) * latent + 8 * (c8 ^ swz128(row));
  }
  auto issue = [&](int k, int st) __attribute__((always_inline)) {
    const uint32_t base = lds0 + (uint32_t)(st * (kXb + kWb));
#pragma unroll
    for (int i = 0; i < kXDma; ++i) lds_dma16(xr[i] + k, base + (uint32_t)(1024 * (kXDma * wave + i)));
#pragma unroll
    for (int i = 0; i < kWDma; ++i) lds_dma16(wr[i] + k, base + (uint32_t)(kXb + 1024 * (kWDma * wave + i)));
  };
  const int wn = wave % kWn, wt = wave / kWn;
  const int n = lane & 31, h = lane >> 5;
  f32x16 acc[2][kTb] = {};
  asm volatile("" ::: "memory");
  wait_vm<0>();  // the waits below count the direct loads alone
  issue(0, 0);
  const int steps = latent / kXDepth;
  for (int ks = 0; ks < steps; ++ks) {
    // the other stage's readers are done (barrier at the end of the last step)
    if (ks + 1 < steps) {
      issue((ks + 1) * kXDepth, (ks + 1) & 1);
      wait_vm<kXDma + kWDma>();
    } else {
      wait_vm<0>();
    }
    lds_barrier();
    const uint32_t base = lds0 + (uint32_t)((ks & 1) * (kXb + kWb));
#pragma unroll
    for (int u = 0; u < kXDepth / 16; ++u) {
      bf16x8 a[2], b[kTb];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = 64 * wn + 32 * i + n;
        a[i] = as_bf16x8(lds_ld16(base + kXb + row * 128 + 16 * ((2 * u + h) ^ swz128(row))));
      }
#pragma unroll
      for (int i = 0; i < kTb; ++i) {
        const int row = 32 * (wt * kTb + i) + n;
        b[i] = as_bf16x8(lds_ld16(base + row * 128 + 16 * ((2 * u + h) ^ swz128(row))));
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < kTb; ++j) acc[i][j] = mfma32(a[i], b[j], acc[i][j]);
    }
    wait_lgkm0();
    lds_barrier();
  }
  // lane (n, h) holds token n, outputs 8 (i / 4) + 4 h + i % 4 of its block
#pragma unroll
  for (int j = 0; j < kTb; ++j) {
    const int t = t0 + 32 * (wt * kTb + j) + n;
    if (t >= total) continue;
    uint16_t* dst = p.kv + ((int64_t)head * p.cap + t) * N + 64 * wn + 4 * h;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<u32x2*>(dst + 32 * i + 8 * q) =
            u32x2{pack_bf16x2(acc[i][j][4 * q], acc[i][j][4 * q + 1]),
                  pack_bf16x2(acc[i][j][4 * q + 2], acc[i][j][4 * q + 3])};
  }
}

}  // namespace

int latent_expand_launch(const char* name, const LatentExpand& p, int latent, int rope, int nope, hipStream_t s) {
  const int64_t blocks = ((int64_t)p.cap + kXTokens - 1) / kXTokens * p.heads;
  if (blocks > 0x7fffffff) return fail(PA_ERR_UNSUPPORTED, "%s: %lld workgroups", name, (long long)blocks);
  if (nope == 128) latent_expand_kernel<256><<<dim3((unsigned)blocks), kXThreads, 0, s>>>(p, latent, rope);
  else latent_expand_kernel<128><<<dim3((unsigned)blocks), kXThreads, 0, s>>>(p, latent, rope);
  return launch_status(name);
}

}  // namespace pa
