// Blocks of a long context: the bounds of their keys, the scores that bound a
// query's logits in them, and the selection by score.
#include <algorithm>

#include "../../include/long_context.h"
#include "lds_tiles.h"
#include "long_context.h"
#include "magic_div.h"

namespace pa {
namespace {

// ---------------------------------------------------------------------------
// bounds
// ---------------------------------------------------------------------------
struct BoundsParams {
  const uint16_t* k;
  int32_t num_pages, page_size, block;
  int64_t page_stride, slot_stride, head_stride;
  const int32_t* block_tables;
  int64_t bt_stride;
  int32_t pages_per_seq;
  const int32_t* lengths;
  const int32_t* cu_q;
  int32_t chunks, chunks_per_head;  // 16-byte chunks of a token's keys, of one head's
  int32_t blocks_per_seq, parts;    // workgroups a sequence: blocks, by parts of 64 chunks
  uint16_t* bounds;
  int64_t b_ps, b_bs, b_hs;
};

// Bounds of one block for 64 chunks (8 elements each) of its tokens' keys: wave
// w takes rows w, w + 4, ..., and the four meet in LDS.  Bound by the reads of
// the block's rows (whole 16-byte chunks of consecutive lanes), four (blocks of 16
// tokens) or eight of them in flight a lane.  A block is computed from all its
// rows in the pool, not from its old bounds and the new rows: a block that a page
// held before never shows through, and the order in which tokens came does not
// matter.  256 sequences' newest token, blocks of 32, 8 kv heads of 128: 4.8 us;
// 20k new tokens of 8 prompts, blocks of 16: 11.5 us, 4.3 TB/s.
template <int kRowsInFlight>
__global__ void __launch_bounds__(256)
block_bounds_kernel(BoundsParams p) {
  __shared__ u32x4 s_min[4][64], s_max[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int part = blockIdx.x % p.parts;
  const int rest = blockIdx.x / p.parts;
  const int b = rest / p.blocks_per_seq;
  const int len = clamp_len(p.lengths, b, (int64_t)p.pages_per_seq * p.page_size);
  const int n = p.cu_q ? min(p.cu_q[b + 1] - p.cu_q[b], len) : min(1, len);
  if (n <= 0) return;  // uniform over the workgroup, as all below
  const int last = (len - 1) / p.block;
  const int c = 64 * part + lane;
  const bool has = c < p.chunks;
  const int h = c / p.chunks_per_head, e = 8 * (c - h * p.chunks_per_head);
  for (int j = (len - n) / p.block + rest % p.blocks_per_seq; j <= last; j += p.blocks_per_seq) {
    const int t0 = j * p.block;
    const int32_t page = p.block_tables[(int64_t)b * p.bt_stride + t0 / p.page_size];
    if (page < 0 || page >= p.num_pages) continue;
    const int rows = min(p.block, len - t0);
    float lo[8], hi[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      lo[i] = INFINITY;
      hi[i] = -INFINITY;
    }
    if (has) {
      const uint16_t* src = p.k + (int64_t)page * p.page_stride + (int64_t)(t0 % p.page_size) * p.slot_stride +
                            (int64_t)h * p.head_stride + e;
      for (int r0 = wave; r0 < rows; r0 += 4 * kRowsInFlight) {
        u32x4 v[kRowsInFlight];
#pragma unroll
        for (int i = 0; i < kRowsInFlight; ++i)
          v[i] = ld16(src + (int64_t)min(r0 + 4 * i, rows - 1) * p.slot_stride);
#pragma unroll
        for (int i = 0; i < kRowsInFlight; ++i)
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const float a = bf16_lo(v[i][w]), z = bf16_hi(v[i][w]);
            lo[2 * w] = fminf(lo[2 * w], a);
            lo[2 * w + 1] = fminf(lo[2 * w + 1], z);
            hi[2 * w] = fmaxf(hi[2 * w], a);
            hi[2 * w + 1] = fmaxf(hi[2 * w + 1], z);
          }
      }
    }
    // (bf16 values: packing is exact)
    s_min[wave][lane] = u32x4{pack_bf16x2(lo[0], lo[1]), pack_bf16x2(lo[2], lo[3]), pack_bf16x2(lo[4], lo[5]),
                              pack_bf16x2(lo[6], lo[7])};
    s_max[wave][lane] = u32x4{pack_bf16x2(hi[0], hi[1]), pack_bf16x2(hi[2], hi[3]), pack_bf16x2(hi[4], hi[5]),
                              pack_bf16x2(hi[6], hi[7])};
    __syncthreads();
    if (wave < 2 && has) {
      u32x4 v = wave ? s_max[0][lane] : s_min[0][lane];
#pragma unroll
      for (int i = 1; i < 4; ++i) {
        const u32x4 o = wave ? s_max[i][lane] : s_min[i][lane];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float a = bf16_lo(v[w]), z = bf16_hi(v[w]), oa = bf16_lo(o[w]), oz = bf16_hi(o[w]);
          v[w] = wave ? pack_bf16x2(fmaxf(a, oa), fmaxf(z, oz)) : pack_bf16x2(fminf(a, oa), fminf(z, oz));
        }
      }
      uint16_t* dst = p.bounds + (int64_t)page * p.b_ps + (int64_t)(t0 % p.page_size / p.block) * p.b_bs +
                      (int64_t)h * p.b_hs + wave * 8 * p.chunks_per_head + e;
      st16(dst, v);
    }
    __syncthreads();  // the next block writes the rows
  }
}

// ---------------------------------------------------------------------------
// scores
// ---------------------------------------------------------------------------
struct ScoresParams {
  const uint16_t* q;
  int64_t q_bs, q_hs;
  const uint16_t* bounds;
  int32_t num_pages, page_size, block;
  int64_t b_ps, b_bs, b_hs;
  const int32_t* block_tables;
  int64_t bt_stride;
  int32_t pages_per_seq;
  const int32_t* lengths;
  int32_t batch, num_kv_heads, group;
  int32_t width, tiles;  // blocks of a table row, wave tasks over them
  MagicDiv per;          // blocks a page
  float scale;
  float* scores;
  int64_t s_bs, s_hs;
};

constexpr int kScoreBlocks = 16;  // blocks of a wave task: the rows of an MFMA

// One wave: 16 blocks of one sequence and kv head against the kv head's q heads,
// 16 at a time.  With q+ = max(q, 0) and q- = min(q, 0) the bound sum_d max(q lo,
// q hi) is q+ . hi + q- . lo: products of a 16 x 2d matrix of bounds with 2d x 16
// of q, whose products are exact and whose sums are 32-bit.  Bound by the reads of
// the bounds (4 d bytes a block and kv head), which come through LDS as whole rows
// (chunk c of row r at c ^ r, so that 16 rows' reads of one chunk land on distinct
// banks).  64 contexts of 16k to 64k tokens, blocks of 32, 8 kv heads of 128: 60
// us, 5.3 TB/s; loaded straight into the operand's layout, 64 bytes of a row at a
// time, 14 us more, and then two or four times the blocks a wave 2 and 21 more.
template <int D>
__global__ void __launch_bounds__(256)
block_scores_kernel(ScoresParams p) {
  constexpr int kS = D / 32;            // k-steps of one bound
  constexpr int kRowB = 4 * D;          // bytes of a row: min and max
  constexpr int kLoads = 16 * kRowB / 1024, kRowLanes = 64 * kLoads / 16;
  __shared__ __attribute__((aligned(1024))) char lds[4][16 * kRowB];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t task = (int64_t)blockIdx.x * 4 + wave;
  const int hkv = p.num_kv_heads;
  const int64_t bt = task / hkv;
  const int kvh = (int)(task - bt * hkv);
  const int b = (int)(bt / p.tiles);
  if (b >= p.batch) return;
  const int j0 = kScoreBlocks * (int)(bt - (int64_t)b * p.tiles);
  const int len = clamp_len(p.lengths, b, (int64_t)p.pages_per_seq * p.page_size);
  const int n_blocks = (len + p.block - 1) / p.block;
  const int n = lane & 15, g = lane >> 4;
  float* dst = p.scores + b * p.s_bs + kvh * p.s_hs;
  float best[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
  if (j0 < n_blocks) {  // uniform
    const uint32_t mine = (uint32_t)(uintptr_t)(lds_void)&lds[wave][0];
    const int j = min(j0 + n, n_blocks - 1);
    const int lp = (int)div_by((uint32_t)j, p.per);
    const int32_t page = safe_page(p.block_tables + b * p.bt_stride, lp, p.num_pages);
    const int64_t off = page * p.b_ps + (int64_t)(j - lp * (int)p.per.d) * p.b_bs + kvh * p.b_hs;
    const int lo = (int)(uint32_t)off, hi = (int)(off >> 32);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int r = (64 * i + lane) / kRowLanes, c = (64 * i + lane) % kRowLanes;
      const int64_t row = (int64_t)(uint32_t)__builtin_amdgcn_ds_bpermute(4 * r, lo) |
                          (int64_t)__builtin_amdgcn_ds_bpermute(4 * r, hi) << 32;
      lds_dma16(p.bounds + row + 8 * (c ^ r), mine + 1024 * i);
    }
    bool first = true;
    for (int c0 = 0; c0 < p.group; c0 += 16) {
      const bool live = c0 + n < p.group;
      const uint16_t* qrow = p.q + b * p.q_bs + (int64_t)(kvh * p.group + (live ? c0 + n : c0)) * p.q_hs;
      u32x4 qv[kS];
#pragma unroll
      for (int s = 0; s < kS; ++s) qv[s] = ld16(qrow + 8 * (4 * s + g));
      if (first) {
        wait_vm<0>();  // the rows have landed
        asm volatile("" ::: "memory");
        first = false;
      }
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < kS; ++s) {
        u32x4 neg, pos;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t m = ((qv[s][w] & 0x80008000u) >> 15) * 0xffffu;
          neg[w] = qv[s][w] & m;
          pos[w] = qv[s][w] & ~m;
        }
        acc = mfma16(as_bf16x8(lds_ld16(mine + kRowB * n + 16 * ((4 * s + g) ^ n))), as_bf16x8(neg), acc);
        acc = mfma16(as_bf16x8(lds_ld16(mine + kRowB * n + 16 * ((4 * (kS + s) + g) ^ n))), as_bf16x8(pos), acc);
      }
      // lane holds the bound of q head c0 + n in block j0 + 4g + i
#pragma unroll
      for (int i = 0; i < 4; ++i) best[i] = fmaxf(best[i], live ? acc[i] : -INFINITY);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) best[i] = max_row16(best[i]);
  }
  const int i = n & 3, at = j0 + 4 * g + i;
  const float x = i == 0 ? best[0] : (i == 1 ? best[1] : (i == 2 ? best[2] : best[3]));
  if (n < 4 && at < p.width) dst[at] = at < n_blocks ? x * p.scale : -INFINITY;
}

// ---------------------------------------------------------------------------
// selection
// ---------------------------------------------------------------------------
struct SelectParams {
  const float* scores;
  int64_t s_bs, s_hs;
  int32_t width;
  const int32_t* lengths;
  int32_t num_kv_heads, block, num, first, recent;
  int32_t* selected;
  int64_t o_bs, o_hs;
};

// A float's bits as an unsigned key of the same order; -0 as 0, NaN below all.
__device__ __forceinline__ uint32_t score_key(uint32_t u) {
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0;
  if (u == 0x80000000u) u = 0;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// One workgroup a (sequence, kv head): the k-th largest key, bit by bit (one
// wave) or by histograms of its digits, then the blocks in order.  A thread keeps
// its keys in registers (kPer of them; 0: reads them again), key j of thread t
// being candidate j * threads + t, so that counts are ballots and their sums
// scalar.  Bound by its chain of steps: 250 candidates 4.2 us, of which 3.5 are the
// launch and the loads; 512 workgroups of up to 4096 10 us, bit by bit 17.8.  One wave
// and bits up to 1024 candidates, against four and histograms, calls in a graph: 32
// workgroups of 260 10.2 and 8.3 us, of 1000 10.7 and 8.3; 512 of 260 10.3 and 9.2, of
// 1000 11.7 and 10.2: the bits cost up to a quarter of the call at every size measured.
template <int kWavesN, int kPer>
__global__ void __launch_bounds__(64 * kWavesN)
select_blocks_kernel(SelectParams p) {
  constexpr int kThreadsN = 64 * kWavesN;
  constexpr int kDigits = 2048;
  __shared__ int s_hist[kWavesN > 1 ? kDigits : 1], s_count[kWavesN], s_found[3];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int b = blockIdx.x / p.num_kv_heads, kvh = blockIdx.x - b * p.num_kv_heads;
  const int len = max(0, p.lengths[b]);
  const int n = min((int)(((int64_t)len + p.block - 1) / p.block), p.width);
  int32_t* out = p.selected + b * p.o_bs + kvh * p.o_hs;
  if (n <= p.num) {  // uniform over the workgroup
    for (int i = tid; i < p.num; i += kThreadsN) out[i] = i < n ? i : -1;
    return;
  }
  const int k = p.num - p.first - p.recent;          // to choose
  const int m = n - p.first - p.recent;              // among m > k
  for (int i = tid; i < p.first; i += kThreadsN) out[i] = i;
  for (int i = tid; i < p.recent; i += kThreadsN) out[p.num - p.recent + i] = n - p.recent + i;
  if (k == 0) return;
  const uint32_t* src = reinterpret_cast<const uint32_t*>(p.scores + b * p.s_bs + kvh * p.s_hs) + p.first;
  uint32_t keys[kPer ? kPer : 1];
  if constexpr (kPer > 0) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int i = j * kThreadsN + tid;
      keys[j] = i < m ? src[i] : 0;
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) keys[j] = j * kThreadsN + tid < m ? score_key(keys[j]) : 0;
  }
  // whether candidate round * threads + tid is one, and its key
  auto key_of = [&](int j, uint32_t& key) __attribute__((always_inline)) {
    const int i = j * kThreadsN + tid;
    if constexpr (kPer > 0) key = keys[j];
    else key = i < m ? score_key(src[i]) : 0;
    return i < m;
  };
  const int used = (m + kThreadsN - 1) / kThreadsN;  // rounds that hold candidates
  // t: the k-th largest key, or a lower one that no key lies between
  uint32_t t = 0;
  if constexpr (kWavesN == 1) {
    // bit by bit, the largest t with at least k keys >= t (t > 0: places past m hold 0)
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t cand = t | 1u << bit;
      int count = 0;
#pragma unroll
      for (int j = 0; j < kPer; ++j) count += __popcll(__ballot(keys[j] >= cand));
      if (count >= k) t = cand;
      if (count == k) break;  // uniform
    }
  } else {
    // by digits of 11, 11 and 10 bits: a histogram of the keys with the digits
    // found so far, and the digit in which the r-th largest of them lies
    constexpr int kMine = kDigits / kThreadsN;  // bins of a thread, from the top down
    int r = k;
    int shift = 21;
    for (int pass = 0; pass < 3; ++pass) {
      const uint32_t known = pass == 0 ? 0 : ~0u << (pass == 1 ? 21 : 10);  // bits of t found
      for (int i = tid; i < kDigits; i += kThreadsN) s_hist[i] = 0;
      __syncthreads();
      if constexpr (kPer > 0) {
#pragma unroll
        for (int j = 0; j < kPer; ++j)
          if (j * kThreadsN + tid < m && (keys[j] & known) == t) atomicAdd(&s_hist[keys[j] >> shift & (kDigits - 1)], 1);
      } else {
        for (int j = 0; j < used; ++j) {
          uint32_t key;
          if (key_of(j, key) && (key & known) == t) atomicAdd(&s_hist[key >> shift & (kDigits - 1)], 1);
        }
      }
      __syncthreads();
      const int top = kDigits - 1 - kMine * tid;
      int have[kMine], total = 0;
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        have[i] = s_hist[top - i];
        total += have[i];
      }
      int upto = (int)wave_scan((uint32_t)total);
      if (lane == 63) s_count[wave] = upto;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kWavesN; ++w) upto += w < wave ? s_count[w] : 0;
      int above = upto - total;  // keys in higher bins
      if (above < r && upto >= r) {  // one thread
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
          if (above < r && above + have[i] >= r) {
            s_found[0] = top - i;
            s_found[1] = above;
            s_found[2] = have[i];
          }
          above += have[i];
        }
      }
      __syncthreads();
      // (the last pass has 10 bits: its digit's top bit is known, and kept out of t)
      t |= ((uint32_t)s_found[0] << shift) & ~known;
      r -= s_found[1];
      if (s_found[2] == r) break;  // all keys of the bin: uniform
      shift = pass == 0 ? 10 : 0;
    }
  }
  // all keys above t, and of those equal to it the first ones: their places are
  // sums over the (round, wave) pairs before
  constexpr int kPairs = kPer ? kPer * kWavesN : kWavesN;  // pairs of a scan (kPer 0: of one round)
  static_assert(kPairs <= 64 * 4, "at most four pairs a lane");
  constexpr int kEach = (kPairs + 63) / 64;
  __shared__ uint32_t s_pair[kPairs];  // above t in the low half, equal in the high half (of 64 at most)
  int gt_base = 0, eq_base = 0;        // (kPer 0) above t and equal to it before this round
  uint32_t before_gt[kEach], before_eq[kEach];
  int all_gt = 0;
  auto scan_pairs = [&]() __attribute__((always_inline)) {
    int gt_run = 0, eq_run = 0;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const uint32_t v = 64 * e + lane < kPairs ? s_pair[64 * e + lane] : 0;
      const uint32_t gt = wave_scan(v & 0xffffu), eq = wave_scan(v >> 16);
      before_gt[e] = gt_run + gt - (v & 0xffffu);
      before_eq[e] = eq_run + eq - (v >> 16);
      gt_run += __builtin_amdgcn_readlane((int)gt, 63);
      eq_run += __builtin_amdgcn_readlane((int)eq, 63);
    }
    all_gt = gt_run;
    return eq_run;
  };
  auto write = [&](int pair, int j, uint64_t gt, uint64_t eq, int ties) __attribute__((always_inline)) {
    int gt_at = gt_base, eq_at = eq_base;
#pragma unroll
    for (int e = 0; e < kEach; ++e)
      if (pair >> 6 == e) {  // uniform
        gt_at += __builtin_amdgcn_readlane((int)before_gt[e], pair & 63);
        eq_at += __builtin_amdgcn_readlane((int)before_eq[e], pair & 63);
      }
    const uint64_t below = (1ull << lane) - 1;
    gt_at += __popcll(gt & below);
    eq_at += __popcll(eq & below);
    if ((gt >> lane & 1) || ((eq >> lane & 1) && eq_at < ties))
      out[p.first + gt_at + min(eq_at, ties)] = p.first + j * kThreadsN + tid;
  };
  if constexpr (kPer > 0) {
    uint64_t gt[kPer], eq[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const bool is = j * kThreadsN + tid < m;
      gt[j] = __ballot(is && keys[j] > t);
      eq[j] = __ballot(is && keys[j] == t);
      if (lane == 0) s_pair[j * kWavesN + wave] = (uint32_t)__popcll(gt[j]) | (uint32_t)__popcll(eq[j]) << 16;
    }
    __syncthreads();
    scan_pairs();
    const int ties = k - all_gt;
#pragma unroll
    for (int j = 0; j < kPer; ++j) write(j * kWavesN + wave, j, gt[j], eq[j], ties);
  } else {
    uint32_t above = 0;
    for (int j = 0; j < used; ++j) {
      uint32_t key;
      const bool is = key_of(j, key);
      above += (uint32_t)__popcll(__ballot(is && key > t));
    }
    if (lane == 0) s_count[wave] = (int)above;
    __syncthreads();
    int ties = k;
#pragma unroll
    for (int w = 0; w < kWavesN; ++w) ties -= s_count[w];
    for (int j = 0; j < used; ++j) {
      uint32_t key;
      const bool is = key_of(j, key);
      const uint64_t gt = __ballot(is && key > t), eq = __ballot(is && key == t);
      __syncthreads();  // the last round's counts have been read
      if (lane == 0) s_pair[wave] = (uint32_t)__popcll(gt) | (uint32_t)__popcll(eq) << 16;
      __syncthreads();
      const int eqs = scan_pairs();
      write(wave, j, gt, eq, ties);
      gt_base += all_gt;
      eq_base += eqs;
    }
  }
}

template <int kWavesN, int kPer>
int select_launch(const char* name, const SelectParams& prm, int64_t items, hipStream_t s) {
  SelectParams p = prm;
  // whole sequences at a time
  const int64_t seqs = std::max<int64_t>(1, kMaxGrid / p.num_kv_heads);
  for (int64_t b0 = 0; b0 * p.num_kv_heads < items; b0 += seqs) {
    const int64_t n = std::min(items - b0 * p.num_kv_heads, seqs * p.num_kv_heads);
    select_blocks_kernel<kWavesN, kPer><<<dim3((unsigned)n), dim3(64 * kWavesN), 0, s>>>(p);
    if (int rc = launch_status(name)) return rc;
    p.scores += seqs * p.s_bs;
    p.lengths += seqs;
    p.selected += seqs * p.o_bs;
  }
  return PA_OK;
}

}  // namespace
}  // namespace pa

using namespace pa;

extern "C" int pa_block_bounds(const uint16_t* k_cache, int32_t num_pages, int32_t page_size, int64_t page_stride,
                               int64_t slot_stride, int64_t head_stride, const int32_t* block_tables,
                               int64_t bt_stride, int32_t pages_per_seq, const int32_t* lengths,
                               const int32_t* cu_seqlens_q, int32_t batch, int32_t max_seqlen_q,
                               int32_t num_kv_heads, int32_t head_dim, int32_t block, uint16_t* bounds,
                               int64_t bounds_page_stride, int64_t bounds_block_stride, int64_t bounds_head_stride,
                               void* stream) {
  const char* name = "pa_block_bounds";
  if (int rc = check_blocks(name, num_pages, page_size, block, batch, num_kv_heads, head_dim, pages_per_seq))
    return rc;
  if (max_seqlen_q < 0) return fail(PA_ERR_INVALID_ARGUMENT, "%s: max_seqlen_q %d", name, max_seqlen_q);
  if (num_kv_heads > (1 << 16)) return fail(PA_ERR_UNSUPPORTED, "%s: %d kv heads", name, num_kv_heads);
  if (batch == 0 || pages_per_seq == 0) return PA_OK;
  if (!k_cache || !block_tables || !lengths || !bounds)
    return fail(PA_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
  if ((((uintptr_t)k_cache | (uintptr_t)bounds) & 15u) ||
      (page_stride | slot_stride | head_stride | bounds_page_stride | bounds_block_stride | bounds_head_stride) % 8)
    return fail(PA_ERR_UNSUPPORTED, "%s: operands must be 16-byte aligned with strides multiple of 8", name);
  BoundsParams p;
  p.k = k_cache;
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
  p.cu_q = cu_seqlens_q;
  p.chunks_per_head = head_dim / 8;
  p.chunks = num_kv_heads * p.chunks_per_head;
  p.parts = (p.chunks + 63) / 64;
  const int64_t span = (int64_t)pages_per_seq * page_size;
  const int64_t most = cu_seqlens_q ? std::min<int64_t>(std::max(max_seqlen_q, 1), span) : 1;
  // blocks that so many tokens touch; a workgroup takes several where one
  // launch could not hold them all
  const int64_t touched = std::min<int64_t>((most + block - 2) / block + 1, (span + block - 1) / block);
  p.blocks_per_seq = (int32_t)std::max<int64_t>(1, std::min<int64_t>(touched, kMaxGrid / p.parts));
  p.bounds = bounds;
  p.b_ps = bounds_page_stride;
  p.b_bs = bounds_block_stride;
  p.b_hs = bounds_head_stride;
  auto kernel = block == 16 ? block_bounds_kernel<4> : block_bounds_kernel<8>;
  const int64_t per = (int64_t)p.parts * p.blocks_per_seq;
  const int64_t seqs = std::max<int64_t>(1, kMaxGrid / per);
  for (int64_t b0 = 0; b0 < batch; b0 += seqs) {
    kernel<<<dim3((unsigned)(std::min<int64_t>(batch - b0, seqs) * per)), dim3(256), 0, (hipStream_t)stream>>>(p);
    if (int rc = launch_status(name)) return rc;
    p.block_tables += seqs * bt_stride;
    p.lengths += seqs;
    if (p.cu_q) p.cu_q += seqs;
  }
  return PA_OK;
}

extern "C" int pa_block_scores(const uint16_t* q, int64_t q_batch_stride, int64_t q_head_stride,
                               const uint16_t* bounds, int32_t num_pages, int32_t page_size,
                               int64_t bounds_page_stride, int64_t bounds_block_stride, int64_t bounds_head_stride,
                               const int32_t* block_tables, int64_t bt_stride, int32_t pages_per_seq,
                               const int32_t* lengths, int32_t batch, int32_t num_heads, int32_t num_kv_heads,
                               int32_t head_dim, int32_t block, float scale, float* scores,
                               int64_t scores_batch_stride, int64_t scores_head_stride, void* stream) {
  const char* name = "pa_block_scores";
  if (int rc = check_blocks(name, num_pages, page_size, block, batch, num_kv_heads, head_dim, pages_per_seq))
    return rc;
  if (num_heads <= 0 || num_heads % num_kv_heads)
    return fail(PA_ERR_INVALID_ARGUMENT, "%s: %d heads of %d kv heads", name, num_heads, num_kv_heads);
  if (!(scale > 0.f)) return fail(PA_ERR_INVALID_ARGUMENT, "%s: scale %g must be positive", name, (double)scale);
  if (batch == 0 || pages_per_seq == 0) return PA_OK;
  if (!q || !bounds || !block_tables || !lengths || !scores)
    return fail(PA_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
  if ((((uintptr_t)q | (uintptr_t)bounds) & 15u) ||
      (q_batch_stride | q_head_stride | bounds_page_stride | bounds_block_stride | bounds_head_stride) % 8)
    return fail(PA_ERR_UNSUPPORTED, "%s: operands must be 16-byte aligned with strides multiple of 8", name);
  ScoresParams p;
  p.q = q;
  p.q_bs = q_batch_stride;
  p.q_hs = q_head_stride;
  p.bounds = bounds;
  p.num_pages = num_pages;
  p.page_size = page_size;
  p.block = block;
  p.b_ps = bounds_page_stride;
  p.b_bs = bounds_block_stride;
  p.b_hs = bounds_head_stride;
  p.block_tables = block_tables;
  p.bt_stride = bt_stride;
  p.pages_per_seq = pages_per_seq;
  p.lengths = lengths;
  p.num_kv_heads = num_kv_heads;
  p.group = num_heads / num_kv_heads;
  p.per = magic_div((uint32_t)(page_size / block));
  p.width = (int32_t)((int64_t)pages_per_seq * (page_size / block));
  p.tiles = (p.width + kScoreBlocks - 1) / kScoreBlocks;
  p.scale = scale;
  p.scores = scores;
  p.s_bs = scores_batch_stride;
  p.s_hs = scores_head_stride;
  const int64_t per_seq = (int64_t)p.tiles * num_kv_heads;
  if (per_seq > 4 * kMaxGrid) return fail(PA_ERR_UNSUPPORTED, "%s: %d blocks by %d kv heads", name, p.width, num_kv_heads);
  const int64_t seqs = std::max<int64_t>(1, 4 * kMaxGrid / per_seq);
  auto kernel = head_dim == 64 ? block_scores_kernel<64>
                               : (head_dim == 128 ? block_scores_kernel<128> : block_scores_kernel<256>);
  for (int64_t b0 = 0; b0 < batch; b0 += seqs) {
    p.batch = (int32_t)std::min<int64_t>(batch - b0, seqs);
    kernel<<<dim3((unsigned)((p.batch * per_seq + 3) / 4)), dim3(256), 0, (hipStream_t)stream>>>(p);
    if (int rc = launch_status(name)) return rc;
    p.q += seqs * p.q_bs;
    p.block_tables += seqs * bt_stride;
    p.lengths += seqs;
    p.scores += seqs * p.s_bs;
  }
  return PA_OK;
}

extern "C" int pa_select_blocks(const float* scores, int64_t scores_batch_stride, int64_t scores_head_stride,
                                int32_t width, const int32_t* lengths, int32_t batch, int32_t num_kv_heads,
                                int32_t block, int32_t num_selected, int32_t first, int32_t recent,
                                int32_t* selected, int64_t selected_batch_stride, int64_t selected_head_stride,
                                void* stream) {
  const char* name = "pa_select_blocks";
  if (batch < 0 || num_kv_heads <= 0 || width < 0 || block <= 0 || num_selected <= 0 || first < 0 || recent < 0)
    return fail(PA_ERR_INVALID_ARGUMENT, "%s: bad sizes (batch=%d, num_kv_heads=%d, width=%d, block=%d, "
                "num_selected=%d, first=%d, recent=%d)", name, batch, num_kv_heads, width, block, num_selected, first,
                recent);
  if ((int64_t)first + recent > num_selected)
    return fail(PA_ERR_INVALID_ARGUMENT, "%s: first %d and recent %d blocks do not fit num_selected %d", name, first,
                recent, num_selected);
  if (num_kv_heads > (1 << 16)) return fail(PA_ERR_UNSUPPORTED, "%s: %d kv heads", name, num_kv_heads);
  if (batch == 0) return PA_OK;
  if ((width && !scores) || !lengths || !selected) return fail(PA_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
  SelectParams p;
  p.scores = scores;
  p.s_bs = scores_batch_stride;
  p.s_hs = scores_head_stride;
  p.width = width;
  p.lengths = lengths;
  p.num_kv_heads = num_kv_heads;
  p.block = block;
  p.num = num_selected;
  p.first = first;
  p.recent = recent;
  p.selected = selected;
  p.o_bs = selected_batch_stride;
  p.o_hs = selected_head_stride;
  const int64_t items = (int64_t)batch * num_kv_heads;
  const int64_t most = (int64_t)width - first - recent;  // candidates
  hipStream_t s = (hipStream_t)stream;
  if (most <= 64 * 4) return select_launch<1, 4>(name, p, items, s);
  if (most <= 64 * 16) return select_launch<1, 16>(name, p, items, s);
  if (most <= 256 * 16) return select_launch<4, 16>(name, p, items, s);
  if (most <= 1024 * 16) return select_launch<16, 16>(name, p, items, s);
  return select_launch<16, 0>(name, p, items, s);
}
