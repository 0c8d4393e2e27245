// Decode over selected blocks of a paged context for gfx950.
//
// Workgroup = (sequence, kv head, 16 of its q heads, part of the selection), four
// wavefronts.  The part's entries that are blocks of the sequence are packed
// into lanes (one entry a lane, at most 64), and its 16-token steps are dealt
// round-robin to the waves.  A wave keeps kBufs steps of K and V in flight in
// registers.  Per step, with 16 tokens t and 16 q columns q:
//
//   S^T[t][q] = K[t][:] . Q[q][:]           D / 32 x v_mfma_f32_16x16x32_bf16
//   online softmax per q column             (the reference maximum moves only
//                                           when a step exceeds it by 2^8)
//   O^T[d][q] += V^T[d][t] . P^T[t][q]      D / 16 x v_mfma_f32_16x16x16_bf16
//
// K goes through the wave's LDS into the row-per-lane layout of the first
// product; V is transposed in registers (row m of M-tile j holds
// d = (D / 16) m + j, so that a lane's load of D / 16 adjacent values feeds all
// tiles).  The waves' parts meet in LDS, the workgroups' in
// block_sparse_merge_kernel.  P is rounded to bf16 for the matrix cores; scores,
// sums and O are 32-bit.
//
// Bound by the reads of the selected rows (2 d bytes at a stride of all kv heads):
// 128 sequences by 64 blocks of 32 tokens, 32 / 8 heads of 128, 167 us, 6.4 TB/s; of
// 64 98 us, 5.5 TB/s; of 256 346 us, 6.2 TB/s (9 registers go to scratch, 13 with the
// soft cap).
// One sequence's 64 blocks, in 16 parts, take 7.4 us, a chain of loads (length,
// selection, table, K and V), and 2.2 us of merge.
#include <algorithm>

#include "../../include/long_context.h"
#include "long_context.h"

namespace pa {
namespace {

constexpr int kSparseWaves = 4;
constexpr int kSparseEntries = 64;  // of a part at most: one a lane
constexpr float kSparseSlack = 8.f;  // lazy-rescale threshold (log2 units)

typedef __attribute__((__vector_size__(4 * sizeof(__bf16)))) __bf16 bf16x4v;

struct SparseParams {
  const uint16_t* q;
  int64_t q_bs, q_hs;
  const uint16_t* k;
  const uint16_t* v;
  int32_t num_pages, page_size, block;
  int64_t page_stride, slot_stride, head_stride;
  const int32_t* block_tables;
  int64_t bt_stride;
  int32_t pages_per_seq;
  const int32_t* lengths;
  int32_t num_heads, num_kv_heads, group, hblocks;
  const int32_t* selected;
  int64_t sel_bs, sel_hs;
  int32_t num;          // entries of a selection
  int32_t per, parts;   // entries of a part, parts of a selection
  uint32_t steps_magic; // ceil(2^20 / steps of a block)
  float logit_scale;    // scale * log2 e when soft_cap is off, else scale
  float soft_cap;
  uint16_t* out;
  int64_t o_bs, o_hs;
  float* ws_o;   // [batch, num_heads, parts, D]
  float* ws_ml;  // [batch, num_heads, parts, 2] (max log2, sum)
};

template <int D>
struct SparseDims {
  static constexpr int kChunks = D / 8;       // 16-byte chunks of a row
  static constexpr int kLoads = D / 32;       // loads of a step's K (and of V, in 16 bytes) a lane
  static constexpr int kBufs = D == 256 ? 2 : (D == 128 ? 4 : 8);  // steps in flight a wave
  static constexpr int kTiles = D / 16;       // M-tiles of O^T, and values of a V row a lane
  static __device__ __forceinline__ int swz(int r) { return D == 64 ? (r >> 1) & 7 : r & 15; }
};

__device__ __forceinline__ u32x4 ld16_once(const void* p) {
  return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
}
__device__ __forceinline__ u32x2 ld8_once(const void* p) {
  return __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(p));
}
// The bf16 halves selected by `hi` of a and b, packed as (a_half, b_half).
__device__ __forceinline__ uint32_t pick_halves(uint32_t a, uint32_t b, bool hi) {
  return hi ? __builtin_amdgcn_perm(b, a, 0x07060302u) : __builtin_amdgcn_perm(b, a, 0x05040100u);
}

template <int D, bool kSoftCap>
__global__ void __launch_bounds__(64 * kSparseWaves, 2)
block_sparse_kernel(SparseParams p) {
  using A = SparseDims<D>;
  constexpr int kBufs = A::kBufs;
  __shared__ __attribute__((aligned(16))) float red_o[kSparseWaves][16][D];
  __shared__ float red_m[kSparseWaves][16], red_l[kSparseWaves][16];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int rest = blockIdx.x;
  const int vheads = p.num_kv_heads * p.hblocks;
  const int vh = rest % vheads;
  rest /= vheads;
  const int part = rest % p.parts;
  const int b = rest / p.parts;
  const int kvh = vh / p.hblocks;
  const int qc0 = 16 * (vh - kvh * p.hblocks);
  const int g_end = min(p.group, qc0 + 16);
  const int n = lane & 15;  // q column of S/O; the d chunk of V loads; the token of K reads
  const int g = lane >> 4;
  const int len = clamp_len(p.lengths, b, (int64_t)p.pages_per_seq * p.page_size);

  // the part's entries, one a lane; those that are blocks move to the front
  const int e = part * p.per + lane;
  const int n_blocks = (int)(((int64_t)len + p.block - 1) / p.block);
  const int sel = lane < p.per && e < p.num ? p.selected[b * p.sel_bs + kvh * p.sel_hs + e] : -1;
  const bool ok = sel >= 0 && sel < n_blocks;
  const uint64_t good = __ballot(ok);
  const int entries = __popcll(good);
  const int before = __popcll(good & ((1ull << lane) - 1));
  int page = 0, off = 0, rem = 0;
  if (ok) {
    const int t0 = sel * p.block;
    const int lp = t0 / p.page_size;
    page = safe_page(p.block_tables + b * p.bt_stride, lp, p.num_pages);
    off = t0 - lp * p.page_size;
    rem = min(len - t0, p.block);
  }
  const int to = 4 * (ok ? before : entries + lane - before);
  page = __builtin_amdgcn_ds_permute(to, page);
  off = __builtin_amdgcn_ds_permute(to, off);
  rem = __builtin_amdgcn_ds_permute(to, rem);

  const int per_block = p.block / 16;
  const int n_steps = entries * per_block;
  const int my_steps = n_steps > wave ? (n_steps - wave + kSparseWaves - 1) / kSparseWaves : 0;
  const int64_t head_off = (int64_t)kvh * p.head_stride;

  bf16x8 qt[A::kLoads];
  {
    const bool live = qc0 + n < g_end;
    const uint16_t* qrow = p.q + b * p.q_bs + (int64_t)(kvh * p.group + qc0 + (live ? n : 0)) * p.q_hs;
#pragma unroll
    for (int s = 0; s < A::kLoads; ++s) qt[s] = as_bf16x8(ld16(qrow + 8 * (4 * s + g)));
  }
  f32x4 acc[A::kTiles];
#pragma unroll
  for (int j = 0; j < A::kTiles; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m_run = -1e30f;  // finite, so that exp2(x - m) never sees inf - inf
  float l_run = 0.f;
  u32x4 kb[kBufs][A::kLoads];
  u32x2 vb[kBufs][4][A::kTiles / 4];  // per token 4 values (8 bytes) a piece

  // entry and 16-token part of the wave's step ks: tokens left from its first on (<= 0: none)
  auto step_at = [&](int ks, int& ent, int& sub) __attribute__((always_inline)) {
    const uint32_t i = (uint32_t)(kSparseWaves * ks + wave);
    ent = (int)((i * p.steps_magic) >> 20);
    sub = (int)i - ent * per_block;
    return ks < my_steps ? __builtin_amdgcn_readlane(rem, ent) - 16 * sub : 0;
  };
  // Loads of wave step ks; tokens past its last one are clamped onto that, and
  // a step without tokens loads q's first bytes, so that every buffer sees the
  // same number of loads issued after it.
  auto issue = [&](int j, int ks) __attribute__((always_inline)) {
    int ent, sub;
    const int left = step_at(ks, ent, sub);
    const uint16_t* kbase = p.q;
    const uint16_t* vbase = p.q;
    int64_t rs = 0;
    if (left > 0) {  // uniform
      const int64_t base = (int64_t)__builtin_amdgcn_readlane(page, ent) * p.page_stride +
                           (int64_t)(__builtin_amdgcn_readlane(off, ent) + 16 * sub) * p.slot_stride + head_off;
      kbase = p.k + base;
      vbase = p.v + base;
      rs = p.slot_stride;
    }
    const int lim = left - 1;
#pragma unroll
    for (int i = 0; i < A::kLoads; ++i) {
      const int c = 64 * i + lane;
      kb[j][i] = ld16_once(kbase + (int64_t)max(0, min(c / A::kChunks, lim)) * rs + 8 * (c % A::kChunks));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint16_t* src = vbase + (int64_t)max(0, min(4 * g + i, lim)) * rs + A::kTiles * n;
      if constexpr (D == 64) {
        vb[j][i][0] = ld8_once(src);
      } else {
#pragma unroll
        for (int w = 0; w < A::kTiles / 8; ++w) {
          const u32x4 x = ld16_once(src + 8 * w);
          vb[j][i][2 * w] = u32x2{x[0], x[1]};
          vb[j][i][2 * w + 1] = u32x2{x[2], x[3]};
        }
      }
    }
  };
  typedef u32x4 __attribute__((address_space(3))) * lds_u32x4;
  const uint32_t kst = (uint32_t)(uintptr_t)(float __attribute__((address_space(3)))*)(&red_o[wave][0][0]);
  auto consume = [&](int j, int ks) __attribute__((always_inline)) {
    int ent, sub;
    const int left = step_at(ks, ent, sub);
    if (left <= 0) return;  // uniform
    // whole rows across lanes -> row n a lane, through the wave's slice of red_o
    // (free until the combine; chunk c of row r at c ^ swz(r))
#pragma unroll
    for (int i = 0; i < A::kLoads; ++i) {
      const int c = 64 * i + lane, r = c / A::kChunks;
      *(lds_u32x4)(uintptr_t)(kst + 2 * D * r + 16 * ((c % A::kChunks) ^ A::swz(r))) = kb[j][i];
    }
    f32x4 sc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < A::kLoads; ++s) {
      const u32x4 kk = *(lds_u32x4)(uintptr_t)(kst + 2 * D * n + 16 * ((4 * s + g) ^ A::swz(n)));
      sc = mfma16(as_bf16x8(kk), qt[s], sc);
    }
    // lane holds S[q = n][token 4g + r]
    float x[4];
    float mx = -INFINITY;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float y = sc[r];
      if constexpr (kSoftCap) y = soft_cap_log2(y, soft_cap_s2(p.logit_scale, p.soft_cap), soft_cap_c(p.soft_cap));
      else y *= p.logit_scale;
      x[r] = 4 * g + r < left ? y : -INFINITY;
      mx = fmaxf(mx, x[r]);
    }
    mx = max_xor16(mx);
    mx = max_xor32(mx);
    if (__ballot(mx > m_run + kSparseSlack)) {
      const float m_new = fmaxf(m_run, mx);
      const float corr = fast_exp2(m_run - m_new);
      m_run = m_new;
      l_run *= corr;
#pragma unroll
      for (int t = 0; t < A::kTiles; ++t) acc[t] = acc[t] * corr;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      x[r] = fast_exp2(x[r] - m_run);
      l_run += x[r];
    }
    const u32x2 pw = {pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3])};
    const bf16x4v pt = __builtin_bit_cast(bf16x4v, pw);
#pragma unroll
    for (int t = 0; t < A::kTiles; ++t) {
      const int w = t >> 2, h = (t >> 1) & 1;
      const u32x2 a = {pick_halves(vb[j][0][w][h], vb[j][1][w][h], t & 1),
                       pick_halves(vb[j][2][w][h], vb[j][3][w][h], t & 1)};
      acc[t] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(bf16x4v, a), pt, acc[t], 0, 0, 0);
    }
  };
#pragma unroll
  for (int j = 0; j < kBufs; ++j) issue(j, j);
  for (int k0 = 0; k0 < my_steps; k0 += kBufs) {
#pragma unroll
    for (int j = 0; j < kBufs; ++j) {
      if (k0 + j < my_steps) consume(j, k0 + j);
      issue(j, k0 + j + kBufs);
    }
  }

  // ---- combine the waves
  l_run = sum_xor16(l_run);
  l_run = sum_xor32(l_run);
  // acc[t][r] = O^T[d = (D / 16) (4g + r) + t][q = n]
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int w = 0; w < A::kTiles / 4; ++w)
      *reinterpret_cast<f32x4*>(&red_o[wave][n][A::kTiles * (4 * g + r) + 4 * w]) =
          f32x4{acc[4 * w][r], acc[4 * w + 1][r], acc[4 * w + 2][r], acc[4 * w + 3][r]};
  if (g == 0) {
    red_m[wave][n] = m_run;
    red_l[wave][n] = l_run;
  }
  __syncthreads();
  float mm = red_m[0][n];
#pragma unroll
  for (int w = 1; w < kSparseWaves; ++w) mm = fmaxf(mm, red_m[w][n]);
  constexpr int kPerLane = D / 16;  // a lane finishes D / 16 values of column n
  const int d0 = kPerLane * (4 * wave + g);
  float o[kPerLane] = {};
  float ll = 0.f;
#pragma unroll
  for (int w = 0; w < kSparseWaves; ++w) {
    const float sw = fast_exp2(red_m[w][n] - mm);
    ll += sw * red_l[w][n];
#pragma unroll
    for (int i = 0; i < kPerLane; i += 4) {
      const f32x4 a = *reinterpret_cast<const f32x4*>(&red_o[w][n][d0 + i]);
#pragma unroll
      for (int k = 0; k < 4; ++k) o[i + k] += sw * a[k];
    }
  }
  if (qc0 + n >= g_end) return;
  const int head = kvh * p.group + qc0 + n;
  if (p.parts == 1) {
    const float inv = ll > 0.f ? 1.f / ll : 0.f;  // no token: a zero row
    uint16_t* dst = p.out + b * p.o_bs + head * p.o_hs + d0;
#pragma unroll
    for (int i = 0; i < kPerLane; i += 4)
      *reinterpret_cast<u32x2*>(dst + i) =
          u32x2{pack_bf16x2(o[i] * inv, o[i + 1] * inv), pack_bf16x2(o[i + 2] * inv, o[i + 3] * inv)};
  } else {
    const int64_t at = ((int64_t)b * p.num_heads + head) * p.parts + part;
#pragma unroll
    for (int i = 0; i < kPerLane; i += 4)
      *reinterpret_cast<f32x4*>(p.ws_o + at * D + d0 + i) = f32x4{o[i], o[i + 1], o[i + 2], o[i + 3]};
    if (wave == 0 && g == 0) {
      p.ws_ml[2 * at] = mm;
      p.ws_ml[2 * at + 1] = ll;
    }
  }
}

// One wave a (sequence, q head): out = sum_c o_c 2^(m_c - M) / sum_c l_c 2^(m_c - M)
// over the parts.
template <int D>
__global__ void __launch_bounds__(256)
block_sparse_merge_kernel(SparseParams p, int64_t rows) {
  constexpr int kPer = D / 64;
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const int64_t b = row / p.num_heads;
  const int h = (int)(row - b * p.num_heads);
  float m_run = -1e30f, lsum = 0.f, o[kPer] = {};
  // the sums follow a running max, so that no load waits for another part's
#pragma unroll 4
  for (int c = 0; c < p.parts; ++c) {
    const int64_t at = row * p.parts + c;
    const f32x2 ml = *reinterpret_cast<const f32x2*>(p.ws_ml + 2 * at);
    const float m_new = fmaxf(m_run, ml[0]);
    const float old = fast_exp2(m_run - m_new), w = fast_exp2(ml[0] - m_new);
    m_run = m_new;
    lsum = lsum * old + ml[1] * w;
#pragma unroll
    for (int i = 0; i < kPer; ++i) o[i] = o[i] * old + p.ws_o[at * D + 64 * i + lane] * w;
  }
  const float inv = lsum > 0.f ? 1.f / lsum : 0.f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const uint32_t x = pack_bf16x2(o[i] * inv, 0.f);
    p.out[b * p.o_bs + h * p.o_hs + 64 * i + lane] = (uint16_t)x;
  }
}

// Entries of a part: enough parts for two workgroups a CU, none below 128
// tokens and none above 64 entries.
int sparse_part_entries(int64_t items, int32_t num, int32_t block) {
  const int64_t want = (512 + items - 1) / std::max<int64_t>(items, 1);  // parts that fill the chip
  const int least = std::max(1, 128 / block);
  int per = (int)std::max<int64_t>((num + want - 1) / want, least);
  return std::min(std::min(per, kSparseEntries), std::max(num, 1));
}

}  // namespace
}  // namespace pa

using namespace pa;

extern "C" size_t pa_block_sparse_decode_workspace_size(int32_t batch, int32_t num_heads, int32_t num_kv_heads,
                                                        int32_t head_dim, int32_t num_selected, int32_t block) {
  if (batch <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads || num_selected <= 0 ||
      block <= 0 || !block_dim_ok(head_dim))
    return 0;
  const int64_t items = (int64_t)batch * num_kv_heads * ((num_heads / num_kv_heads + 15) / 16);
  const int per = sparse_part_entries(items, num_selected, block);
  const int64_t parts = (num_selected + per - 1) / per;
  return parts == 1 ? 0 : (size_t)batch * num_heads * parts * (head_dim + 2) * sizeof(float);
}

extern "C" int pa_block_sparse_decode(const uint16_t* q, int64_t q_batch_stride, int64_t q_head_stride,
                                      const uint16_t* k_cache, const uint16_t* v_cache, int32_t num_pages,
                                      int32_t page_size, int64_t page_stride, int64_t slot_stride,
                                      int64_t head_stride, const int32_t* block_tables, int64_t bt_stride,
                                      int32_t pages_per_seq, const int32_t* lengths, int32_t batch,
                                      int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                                      const int32_t* selected, int64_t selected_batch_stride,
                                      int64_t selected_head_stride, int32_t num_selected, int32_t block, float scale,
                                      float soft_cap, uint16_t* out, int64_t out_batch_stride,
                                      int64_t out_head_stride, void* workspace, size_t workspace_bytes,
                                      void* stream) {
  const char* name = "pa_block_sparse_decode";
  if (int rc = check_blocks(name, num_pages, page_size, block, batch, num_kv_heads, head_dim, pages_per_seq))
    return rc;
  if (num_heads <= 0 || num_heads % num_kv_heads || num_selected <= 0)
    return fail(PA_ERR_INVALID_ARGUMENT, "%s: bad sizes (num_heads=%d, num_kv_heads=%d, num_selected=%d)", name,
                num_heads, num_kv_heads, num_selected);
  if (block > 256) return fail(PA_ERR_UNSUPPORTED, "%s: block %d (256 at most)", name, block);
  if (batch == 0) return PA_OK;
  if (!q || !k_cache || !v_cache || !lengths || !selected || !out || (pages_per_seq && !block_tables))
    return fail(PA_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
  if ((((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out | (uintptr_t)workspace) & 15u) ||
      (q_batch_stride | q_head_stride | page_stride | slot_stride | head_stride | out_batch_stride |
       out_head_stride) % 8)
    return fail(PA_ERR_UNSUPPORTED, "%s: operands must be 16-byte aligned with strides multiple of 8", name);
  SparseParams p;
  p.q = q;
  p.q_bs = q_batch_stride;
  p.q_hs = q_head_stride;
  p.k = k_cache;
  p.v = v_cache;
  p.num_pages = num_pages;
  p.page_size = page_size;
  p.block = block;
  p.page_stride = page_stride;
  p.slot_stride = slot_stride;
  p.head_stride = head_stride;
  p.block_tables = block_tables;
  p.bt_stride = bt_stride;
  p.pages_per_seq = pages_per_seq;
  p.lengths = lengths;
  p.num_heads = num_heads;
  p.num_kv_heads = num_kv_heads;
  p.group = num_heads / num_kv_heads;
  p.hblocks = (p.group + 15) / 16;
  p.selected = selected;
  p.sel_bs = selected_batch_stride;
  p.sel_hs = selected_head_stride;
  p.num = num_selected;
  const int64_t items = (int64_t)batch * num_kv_heads * p.hblocks;
  p.per = sparse_part_entries(items, num_selected, block);
  p.parts = (num_selected + p.per - 1) / p.per;
  p.steps_magic = ((1u << 20) + block / 16 - 1) / (block / 16);  // exact for step numbers below 2^10
  p.logit_scale = soft_cap > 0.f ? scale : scale * kLog2e;
  p.soft_cap = soft_cap;
  p.out = out;
  p.o_bs = out_batch_stride;
  p.o_hs = out_head_stride;
  const int64_t rows = (int64_t)batch * num_heads;
  if (p.parts > 1) {
    const size_t need = (size_t)rows * p.parts * (head_dim + 2) * sizeof(float);
    if (!workspace || workspace_bytes < need)
      return fail(PA_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", name, workspace_bytes, need);
  }
  p.ws_o = (float*)workspace;
  p.ws_ml = p.ws_o + rows * p.parts * head_dim;
  const int64_t grid = items * p.parts;
  if (grid > kMaxGrid * 4 || (rows + 3) / 4 > kMaxGrid * 4)
    return fail(PA_ERR_UNSUPPORTED, "%s: %lld workgroups", name, (long long)grid);
  hipStream_t s = (hipStream_t)stream;
  auto launch = [&](auto kernel, auto merge) {
    kernel<<<dim3((unsigned)grid), dim3(64 * kSparseWaves), 0, s>>>(p);
    int rc = launch_status(name);
    if (rc || p.parts == 1) return rc;
    merge<<<dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s>>>(p, rows);
    return launch_status(name);
  };
  const bool cap = soft_cap > 0.f;
  if (head_dim == 64)
    return launch(cap ? block_sparse_kernel<64, true> : block_sparse_kernel<64, false>, block_sparse_merge_kernel<64>);
  if (head_dim == 128)
    return launch(cap ? block_sparse_kernel<128, true> : block_sparse_kernel<128, false>,
                  block_sparse_merge_kernel<128>);
  return launch(cap ? block_sparse_kernel<256, true> : block_sparse_kernel<256, false>,
                block_sparse_merge_kernel<256>);
}
