// Expansion of paged latent rows into K and V rows of each head, for the
// expanded form of the prefill.
//
//   kv[h][t] = [ W_uk[h] c_t | W_uv[h] c_t ],   k_rope[t] = the row's rotary part
//
// A matrix product of all tokens by all heads' outputs, depth R.  A workgroup
// keeps 256 token rows in registers, 32 a wave (R = 512: 128 of them), gathered
// once through the block tables, and streams its share of the weight rows
// through a four-stage LDS ring, 32 rows a step: v_mfma_f32_32x32x16_bf16 with A
// = weight rows (16-byte LDS reads, shared by the eight waves) and B = token
// rows.  Token rows are read once per share, weights once per 256 tokens
// (32 KiB of LDS reads per wave and step).  Results go out through a wave's own 2 KiB of LDS, 64 bytes of a
// token at a time.
//
// 24 k tokens by 64 heads (R = 512, Dn = 128): 0.49 to 0.55 ms, 750 to 840
// TFLOP/s, of the 8.5 ms that the call takes, the matrix cores busy for 56 % of
// the time at 1.75 GHz, LDS for 37 %; both operands through LDS 64 deep at a time
// took 0.85.  1 000 to 2 000 tokens by 16 heads: 18 to 22 us, most of them the
// gather's chain (sequence, page, row) and its 16-byte reads of 32 rows at a
// time.  K and V are rounded to bf16 here, as a cache of K and V rows per head
// would hold them.
#include <algorithm>

#include "latent_attend.h"
#include "lds_tiles.h"
#include "pa_errors.h"
#include "../../include/latent_attention.h"

namespace pa {
namespace {

constexpr int kXTokens = 256;
constexpr int kXThreads = 512;
constexpr int kXStages = 4;

// Cache row of flat token t (of the sequences laid end to end by cu_k).
__device__ __forceinline__ const uint16_t* flat_row(const LatentExpand& p, int t) {
  const int64_t span = (int64_t)p.pool.pages_per_seq * p.pool.page.d;
  int lo = 0, hi = p.batch;  // last b whose rows start at t or before
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (flat_start(p.cu_k, mid, span) <= t) lo = mid;
    else hi = mid;
  }
  const int j = (int)max((int64_t)0, min(t - flat_start(p.cu_k, lo, span), span - 1));
  const int pg = (int)div_by((uint32_t)j, p.pool.page);
  const int page = safe_page(p.pool.tables + lo * p.pool.bt_stride, pg, p.pool.num_pages);
  return p.pool.cache + page * p.pool.page_stride + (int64_t)(j - pg * (int)p.pool.page.d) * p.pool.slot_stride;
}

// blocks: 32-output blocks of all heads; share: those of a workgroup.
template <int R>
__global__ void __launch_bounds__(kXThreads) __attribute__((amdgpu_waves_per_eu(2, 2)))
latent_expand_kernel(LatentExpand p, int rope, int n, int blocks, int share, int tiles) {
  constexpr int kRowB = 2 * R, kStageB = 32 * kRowB, kKs = R / 16;
  constexpr int kDma = kStageB / (1024 * 8), kRowsPerDma = 1024 / kRowB;
  __shared__ __attribute__((aligned(1024))) char smem[kXStages * kStageB + 8 * 2048];
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void)smem;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // workgroups that run together work on all tokens and few weight rows
  const int part = blockIdx.x / tiles, t0 = (blockIdx.x - part * tiles) * kXTokens;
  const int64_t end = flat_start(p.cu_k, p.batch, (int64_t)p.pool.pages_per_seq * p.pool.page.d);
  const int total = (int)max((int64_t)0, min((int64_t)p.cap, end));
  if (t0 >= total) return;
  const int first = part * share, last = min(blocks, first + share);
  const int l = lane & 31, h = lane >> 5;
  const int t = t0 + 32 * wave + l;
  const bool live = t < total;

  // ---- weight rows: block b's 32 rows are contiguous; a wave loads kDma KiB
  const uint16_t* w = p.w_kv + (int64_t)p.head0 * n * R;
  uint32_t woff[kDma];
#pragma unroll
  for (int i = 0; i < kDma; ++i) {
    const int r = (kDma * wave + i) * kRowsPerDma + lane / (kRowB / 16), c = lane & (kRowB / 16 - 1);
    woff[i] = (uint32_t)(r * kRowB + 16 * (c ^ swz256(r)));
  }
  auto issue = [&](int b) __attribute__((always_inline)) {
    const char* src = (const char*)(w + (int64_t)min(b, last - 1) * 32 * R);  // past the end: the last block again
    const uint32_t st = lds0 + (uint32_t)((b - first) & (kXStages - 1)) * kStageB;
#pragma unroll
    for (int i = 0; i < kDma; ++i) lds_dma16s(woff[i], src, st + (uint32_t)(1024 * (kDma * wave + i)));
  };
  // (their latency passes under that of the gathered rows)
  issue(first);
  issue(first + 1);
  issue(first + 2);

  // ---- this wave's token rows: lane (l, h) holds chunks 2 ks + h of token l
  const uint16_t* row = flat_row(p, min(t, total - 1));
  bf16x8 x[kKs];
#pragma unroll
  for (int ks = 0; ks < kKs; ++ks) x[ks] = as_bf16x8(ld16(row + 16 * ks + 8 * h));
  if (p.k_rope && part == 0 && live) {
    for (int c = h; c < rope / 8; c += 2) st16(p.k_rope + (int64_t)t * rope + 8 * c, ld16(row + R + 8 * c));
  }

  uint32_t aoff[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) aoff[i] = lds0 + l * kRowB + 16 * ((2 * i + h) ^ swz256(l));
  const uint32_t own = lds0 + kXStages * kStageB + 2048 * wave;

#pragma unroll
  for (int ks = 0; ks < kKs; ++ks) asm volatile("" : "+v"(x[ks]));  // here, not waited for in the loop
  for (int b = first; b < last; ++b) {
    // block b has landed (loads complete in order, so at most those of the two
    // blocks behind it may be outstanding); everybody is done with block b - 1
    wait_vm<2 * kDma>();
    lds_barrier();
    issue(b + 3);
    const uint32_t st = (uint32_t)((b - first) & (kXStages - 1)) * kStageB;
    uint32_t ao[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      ao[i] = aoff[i] + st;
      asm volatile("" : "+v"(ao[i]));
    }
    constexpr int kAhead = 6;
    f32x16 acc[2] = {};
    bf16x8 a[kKs];
    auto fetch = [&](int ks) __attribute__((always_inline)) {
      a[ks] = as_bf16x8(lds_ld16(ao[ks % 8] + (ks / 8) * 256));
    };
#pragma unroll
    for (int ks = 0; ks < kAhead; ++ks) fetch(ks);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int ks = 0; ks < kKs; ++ks) {
      acc[ks & 1] = mfma32(a[ks], x[ks], acc[ks & 1]);
      if (ks + kAhead < kKs) fetch(ks + kAhead);
      __builtin_amdgcn_sched_barrier(0);
    }
    // lane (l, h) holds token l, outputs 8 q + 4 h + i: to the wave's own rows of
    // 64 bytes (16-byte chunk q of token l at q ^ (l / 4 % 4)), then out 16 bytes a lane
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const f32x16 s = acc[0] + acc[1];
      const u32x2 v = {pack_bf16x2(s[4 * q], s[4 * q + 1]), pack_bf16x2(s[4 * q + 2], s[4 * q + 3])};
      *reinterpret_cast<u32x2 __attribute__((address_space(3)))*>(
          (uintptr_t)(own + 64 * l + 16 * (q ^ (l >> 2 & 3)) + 8 * h)) = v;
    }
    wait_lgkm0();
    asm volatile("" ::: "memory");
    const int head = 32 * b / n, col = 32 * b - head * n;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = 16 * i + (lane >> 2), c = lane & 3;
      const u32x4 v = lds_ld16(own + 64 * r + 16 * (c ^ (r >> 2 & 3)));
      const int tr = t0 + 32 * wave + r;
      if (tr < total) st16(p.kv + ((int64_t)head * p.cap + tr) * n + col + 8 * c, v);
    }
  }
  wait_vm<0>();  // loads past the end are still in flight
}

}  // namespace

int latent_expand_launch(const char* name, const LatentExpand& p, int latent, int rope, int nope, hipStream_t s) {
  const int n = 2 * nope, blocks = p.heads * n / 32;
  const int64_t tiles = ((int64_t)p.cap + kXTokens - 1) / kXTokens;
  // Rounds of 256 workgroups by the time they take, in steps: each round gathers
  // token rows (about eight steps) and multiplies its share.  One round for a
  // few thousand tokens, more where one leaves CUs idle (2 044 tokens by 16 heads
  // in one round 22 us, in two 32).
  int share = blocks;
  int64_t best = INT64_MAX;
  for (int64_t rounds = 1; rounds <= 4; ++rounds) {
    const int64_t parts = std::max<int64_t>(1, std::min<int64_t>(blocks, 256 * rounds / tiles));
    const int64_t sh = (blocks + parts - 1) / parts;
    const int64_t time = (tiles * ((blocks + sh - 1) / sh) + 255) / 256 * (8 + sh);
    if (time < best) {
      best = time;
      share = (int)sh;
    }
  }
  const int64_t grid = tiles * ((blocks + share - 1) / share);
  if (grid * kXThreads > 0xffffffffll) return fail(PA_ERR_UNSUPPORTED, "%s: %lld workgroups", name, (long long)grid);
  const dim3 g((unsigned)grid), b(kXThreads);
  if (latent == 512) latent_expand_kernel<512><<<g, b, 0, s>>>(p, rope, n, blocks, share, (int)tiles);
  else latent_expand_kernel<256><<<g, b, 0, s>>>(p, rope, n, blocks, share, (int)tiles);
  return launch_status(name);
}

}  // namespace pa
