// Absorbed-form latent attention for gfx950: every cache row is key and value
// of all heads at once.
//
//   s[n, j] = q_lat[n] . c_j + q_rope[n] . k_j,   o[n] = sum_j softmax_j(scale s) c_j
//
// for the rows n = (token, head) of a sequence.  Workgroup = kRows rows of one
// sequence and a range of 32-token kv tiles; a tile (latent rows, then rotary
// rows) sits in one stage of a four-stage LDS ring filled by direct loads
// through the block table and serves both products.
//
// Eight waves in two roles, one of each on every SIMD:
//   waves 0-3 (scores):  S^T[16 tokens][32 rows] per tile, v_mfma_f32_16x16x32
//       with Q in registers (R = 512: 144), the running maximum and sum, P to LDS
//   waves 4-7 (values):  O^T[R / 4][all rows] in registers, v_mfma_f32_32x32x16
//       with V^T by transposing LDS reads and P^T from LDS
// so that one wave's exponentials run under the other's matrix instructions:
// the values' wave reads tile t - 1's operands while the scores' wave multiplies
// tile t, and multiplies while that takes its exponentials, with one barrier a
// tile.  Both issue loads, two tiles ahead.
//
// Work is cut on the device: the kv tiles of all (sequence, row tile) units,
// laid end to end (a unit's start counted as some more of them), are dealt to the
// workgroups in equal contiguous shares; a workgroup that gets the whole of a unit
// writes its rows, one that gets a part leaves O (float32), maximum and sum to
// latent_merge_kernel.
//
// P is rounded to bf16 for the matrix cores, once: its reference is a whole number
// of log2 units, so that bringing P or O from one to another multiplies by a power
// of two.  It may lag behind the row's maximum (by 2^8 from tile to tile, 2^64
// inside one), which costs range and no bits.  Scores, maxima, sums, O and the parts are float32; the joined rows are
// rounded to bf16 once.
//
// Few heads are bound by the cache's reads: 256 sequences of 512-8 192 tokens by
// 16 heads (1.28 GB) 220 us, 5.8 TB/s, of a call of 246.  At 64 rows nothing is
// full: 64 sequences by 128 heads 108 us, 740 TFLOP/s, of a call of 139, at 1.1 us
// a tile; over next turns of eight conversations (350 us) the counters have the
// matrix cores busy for 41 % of the time, LDS for 34 % (a third of that bank
// conflicts) and a wave waiting for 32 % of its own, most likely in the chain
// through the one barrier a tile: the scores' products, their exponentials, the
// values' products.  15 us of the 108 are around the loop, much of it the parts'
// 50 MB.  One sequence of 32 k tokens by 64 heads: 21 us, and 5 us joining 128
// parts.
#include <algorithm>
#include <cmath>

#include "latent_attend.h"
#include "lds_tiles.h"
#include "pa_errors.h"
#include "../../include/latent_attention.h"

namespace pa {
namespace {

constexpr int kWgs = 256;      // one per CU
constexpr int kTile = 32;      // kv tokens per tile
constexpr int kLStages = 4;
constexpr int kLThreads = 512;
constexpr int kMaxBatch = 16384;  // their prefix sums fit the ring
constexpr float kSlack = 8.f;  // log2 units a tile's reference may lag behind the maximum of those before it
constexpr float kJump = 64.f;  // and a half tile's behind its own
constexpr int kLead = 7;
constexpr int kDirect = 6, kDirectMany = 16;  // tiles of a sequence up to which it is not cut
constexpr float kNoMax = -1e30f;

// Tiles that a workgroup takes at least of `total`: more workgroups each do
// less and leave more to join.  64 heads, one sequence of 32, 64, 128, 256, 512,
// 1 024 tiles, whole calls: 23.4, 24.2, 26.4, 29.8, 34.4, 36.4 us with 2, 25.0,
// 25.5, 26.6, 28.3, 31.0, 36.3 with 4, 28.7, 29.9, 30.0, 30.7, 32.0, 34.9 with 8.
__host__ __device__ inline int min_share(int64_t total) { return total <= 64 ? 2 : total <= 384 ? 4 : 8; }

struct AttnParams {
  LatentAttn a;
  MagicDiv heads;
  float scale_log2;
  int32_t wgs;
  int32_t lead;     // of a unit, in the cut: tiles that its start is counted as
  bool pages8;      // eight aligned rows lie in one page, within 32-bit byte offsets
  // What latent_merge_kernel has to join, [4] each: sequence, row tile, parts (0: nothing), first
  // workgroup; one entry a unit where there are no more units than workgroups
  // (row_tiles > 0: those of a sequence), else one a workgroup.
  int32_t* joins;
  int32_t row_tiles;
  int32_t unit_tiles;  // not 0: a workgroup a unit, this many row tiles a sequence, no cut and nothing to join
  float* parts;     // [2 wgs][rows * R]
  float* stats;     // [2 wgs][rows][2]
};

template <int R, int DR, int ROWS>
struct Dims {
  static constexpr int kRowB = 2 * R;               // bytes of a latent row
  static constexpr int kRopeB = 2 * DR;
  static constexpr int kLatB = kTile * kRowB;
  static constexpr int kStageB = kLatB + kTile * kRopeB;
  static constexpr int kRing = kLStages * kStageB;
  // Of even and odd tiles: P [ROWS][32] bf16, for each half tile and row its
  // maximum and the reference of its P, and for each row the reference that the
  // value waves ask for.  Sums [2][ROWS] at the end.
  static constexpr int kPB = ROWS * 64, kRefB = 2 * ROWS * 4;
  static constexpr int kPOff = kRing;
  static constexpr int kMaxOff = kPOff + 2 * kPB;
  static constexpr int kRefOff = kMaxOff + 2 * kRefB;
  static constexpr int kAskOff = kRefOff + 2 * kRefB;
  static constexpr int kSumOff = kAskOff + kRefB;
  static constexpr int kLds = kSumOff + 2 * ROWS * 4;
  static constexpr int kKs = R / 32, kRs = DR / 32;   // 32-deep k-steps of the scores
  static constexpr int kNr = ROWS / 32;               // 16-row blocks of a score wave
  static constexpr int kDt = R / 128;                 // 32-row blocks of O^T of a value wave
  static constexpr int kRb = ROWS / 32;               // its 32-row blocks of rows
  static constexpr int kRowsPerDma = 1024 / kRowB;
  static constexpr int kLatDma = 8 / kRowsPerDma;     // a value wave loads eight rows of a tile
  // loads of a tile: a value wave's, a score wave's (the rotary parts among them)
  static constexpr int kVDma = kLatDma / 2, kSDma = kLatDma + 1 - kVDma;
  static_assert(ROWS * (kRowB + kRopeB) <= 2 * kStageB, "Q in two stages");
  static_assert(kLds <= 160 * 1024 && kRing >= 4 * kMaxBatch + 64, "LDS");
};

template <int DR>
__device__ __forceinline__ int rope_swz(int r) {
  return DR == 64 ? swz128(r) : swz64(r);
}

// The same value, as one that the compiler makes anew here: what hangs on it is
// not carried in registers from outside the loops (the roles' 250 are full).
__device__ __forceinline__ int fresh(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// A wave-uniform pointer, in scalar registers.
__device__ __forceinline__ const uint16_t* uniform_ptr(const uint16_t* p) {
  const uint64_t x = (uint64_t)(uintptr_t)p;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)x);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(x >> 32));
  return (const uint16_t*)(uintptr_t)((uint64_t)hi << 32 | lo);
}

// An address as the base of reads with constant offsets.
__device__ __forceinline__ uint32_t fresh_addr(uint32_t x) {
  asm volatile("" : "+v"(x));
  return x;
}

// Direct loads of kCount of a tile's pieces from piece kFirst on, into the ring:
// the pieces of waves w and w + 4 are the eight rows 8 w .. 8 w + 7, 1 KiB of
// latent rows each and the rotary parts last.  prepare() finds a tile's rows,
// load(i) issues a piece, so that they can be spread through other work (the CU
// takes one in 20 to 30 cycles).  Where pages hold eight aligned rows and all of
// them are there, a piece is one scalar base (made for 64 tiles at a time, one
// a lane) and a lane offset kept in a register; other tiles are looked up row
// by row (load_rows).
//
// kOnce (32 rows: one row tile a sequence, every cached row read by one
// workgroup): loads that do not stay in the caches, 239 us against 258 for 256
// sequences by 16 heads; at 64 rows they cost 152 against 139 (64 sequences by
// 128 heads, two row tiles) and 37.2 against 34.9 (one of 32 k tokens, 64 heads).
template <typename D, int R, int DR, int kFirst, int kCount, bool kOnce>
struct TileLoader {
  static constexpr int kC = D::kRopeB / 16;  // chunks of a rotary row
  const LatentPool& pool;
  const int32_t* bt;
  uint32_t lds0;
  int w, lane, t0, lk;
  bool pages8;
  uint32_t voff[kCount];
  const uint16_t* base;
  uint32_t stage, base_lo, base_hi;
  int bases_at, first_row;  // bases_at: tile of lane 0
  bool rows8;

  __device__ __forceinline__ TileLoader(const LatentPool& pool_, const int32_t* bt_, uint32_t lds0_, int w_, int lane_,
                                        int t0_, int lk_, bool pages8_)
      : pool(pool_), bt(bt_), lds0(lds0_), w(w_), lane(lane_), t0(t0_), lk(lk_), pages8(pages8_) {
    base = nullptr;
    stage = base_lo = base_hi = 0;
    bases_at = t0 - 64;
    first_row = 0;
    rows8 = false;
    const uint32_t sb = 2u * (uint32_t)pool.slot_stride;
#pragma unroll
    for (int k = 0; k < kCount; ++k) {
      const int i = kFirst + k;
      if (i < D::kLatDma) {
        const int r = i * D::kRowsPerDma + (D::kRowsPerDma == 1 ? 0 : lane >> 5);
        voff[k] = (uint32_t)r * sb + 16 * ((lane & (D::kRowB / 16 - 1)) ^ swz256(8 * w + r));
      } else {
        const int rr = lane / kC;
        voff[k] = (uint32_t)rr * sb + 2 * R + 16 * ((lane & (kC - 1)) ^ rope_swz<DR>(8 * w + rr));
      }
    }
  }
  __device__ __forceinline__ uint32_t piece(int i) const {
    return stage + (i < D::kLatDma ? (uint32_t)(8 * w * D::kRowB + 1024 * i)
                                   : (uint32_t)(D::kLatB + 8 * w * D::kRopeB));
  }
  __device__ __forceinline__ void prepare(int t) {
    stage = lds0 + (uint32_t)((t - t0) & (kLStages - 1)) * D::kStageB;
    first_row = t * kTile + 8 * w;
    rows8 = pages8 && first_row + 8 <= lk;
    if (t - bases_at >= 64) {
      bases_at = t;
      const int j = min(first_row + kTile * lane, (lk - 1) & ~7);
      const int pg = (int)div_by((uint32_t)j, pool.page);
      const int page = safe_page(bt, pg, pool.num_pages);
      const uint64_t at = (uint64_t)(uintptr_t)(pool.cache + page * pool.page_stride +
                                                (int64_t)(j - pg * (int)pool.page.d) * pool.slot_stride);
      base_lo = (uint32_t)at;
      base_hi = (uint32_t)(at >> 32);
      asm volatile("" : "+v"(base_lo), "+v"(base_hi));
    }
    const uint32_t lo = __builtin_amdgcn_readlane(base_lo, t - bases_at);
    const uint32_t hi = __builtin_amdgcn_readlane(base_hi, t - bases_at);
    base = (const uint16_t*)(uintptr_t)((uint64_t)hi << 32 | lo);
  }
  // Piece k of this wave's (rows8).
  __device__ __forceinline__ void load(int k) {
    if (kFirst + k < D::kLatDma || 8 * kC == 64 || fresh(lane) < 8 * kC) {
      if constexpr (kOnce) lds_dma16v_once(voff[k], uniform_ptr(base), piece(kFirst + k));
      else lds_dma16v(voff[k], uniform_ptr(base), piece(kFirst + k));
    }
  }
  __device__ __forceinline__ void load_rows() {
    const int ln = fresh(lane), rr = ln / kC;
    const uint16_t* rows[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int j = min(first_row + i, lk - 1);  // rows past the end repeat the last
      const int pg = (int)div_by((uint32_t)j, pool.page);
      const int page = safe_page_scalar(bt, pg, pool.num_pages);
      rows[i] = pool.cache + page * pool.page_stride + (int64_t)(j - pg * (int)pool.page.d) * pool.slot_stride;
    }
#pragma unroll
    for (int k = 0; k < kCount; ++k) {
      const int i = kFirst + k;
      if (i < D::kLatDma) {
        if constexpr (D::kRowsPerDma == 1) {
          lds_dma16(rows[i & 7] + 8 * (ln ^ swz256(8 * w + i)), piece(i));
        } else {
          const uint16_t* own = ln >> 5 ? rows[(2 * i + 1) & 7] : rows[(2 * i) & 7];
          lds_dma16(own + 8 * ((ln & 31) ^ swz256(8 * w + 2 * i + (ln >> 5))), piece(i));
        }
      } else {
        const uint16_t* mine = rows[0];
#pragma unroll
        for (int r = 1; r < 8; ++r) mine = rr == r ? rows[r] : mine;
        if (ln < 8 * kC) lds_dma16(mine + R + 8 * ((ln & (kC - 1)) ^ rope_swz<DR>(8 * w + rr)), piece(i));
      }
    }
  }
  // All of tile t's pieces at once.
  __device__ __forceinline__ void issue(int t) {
    prepare(t);
    if (rows8) {
#pragma unroll
      for (int k = 0; k < kCount; ++k) load(k);
    } else {
      load_rows();
    }
  }
};

// Waits until all tiles but the newest one issued have landed (`open`: there is
// a newer one), for a wave with kCount loads a tile.
template <int kCount>
__device__ __forceinline__ void landed(bool open) {
  if (open) wait_vm<kCount>();
  else wait_vm<0>();
}

struct Seq {
  int q0, lq, lk, nt, nrt;
  int first;  // token i sees first + i + 1 rows
};

__device__ __forceinline__ Seq seq_of(const AttnParams& p, int b, int rows) {
  Seq s;
  s.q0 = b;
  s.lq = 1;
  int lq_all = 1;
  if (p.a.cu_q) {
    s.q0 = p.a.cu_q[b];
    lq_all = p.a.cu_q[b + 1] - s.q0;
    s.lq = min(lq_all, p.a.max_q);
    if (s.q0 < 0 || s.q0 >= p.a.num_tokens) s.lq = 0;
    s.lq = max(0, min(s.lq, p.a.num_tokens - s.q0));
  }
  s.lk = latent_kv_len(p.a.pool, p.a.kv_lens ? p.a.kv_lens[b] : p.a.cu_k[b + 1] - p.a.cu_k[b]);
  s.first = s.lk - lq_all;
  s.nt = (s.lk + kTile - 1) / kTile;
  s.nrt = (s.lq * p.a.heads + rows - 1) / rows;
  return s;
}

// Inclusive sum over the workgroup's threads (blockDim.x == kLThreads) below
// and at this one; tmp: kLThreads / 64 ints.
__device__ __forceinline__ int block_scan(int v, int* tmp, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int incl = (int)wave_scan((uint32_t)v);
  __syncthreads();
  if (lane == 63) tmp[wave] = incl;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kLThreads / 64; ++w) {
    const int x = tmp[w];
    before += w < wave ? x : 0;
    total += x;
  }
  return incl + before;
}

// Zero rows for row tile rt of a sequence without any cached token.
template <int R, int ROWS>
__device__ __forceinline__ void zero_unit(const AttnParams& p, const Seq& sq, int rt, int wave, int waves, int lane) {
  const int rows = min((rt + 1) * ROWS, sq.lq * p.a.heads);
  for (int i = rt * ROWS + wave; i < rows; i += waves) {
    const int tok = (int)div_by((uint32_t)i, p.heads), hd = i - tok * p.a.heads;
    uint16_t* o = p.a.out + (int64_t)(sq.q0 + tok) * p.a.o_ts + hd * p.a.o_hs;
    if (8 * lane < R) st16(o + 8 * lane, u32x4{0, 0, 0, 0});
  }
}

template <int R, int DR, int ROWS>
__global__ void __launch_bounds__(kLThreads) __attribute__((amdgpu_waves_per_eu(2, 2)))
latent_attn_kernel(AttnParams p) {
  using D = Dims<R, DR, ROWS>;
  __shared__ __attribute__((aligned(1024))) char smem[D::kLds];
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void)smem;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const LatentPool& pool = p.a.pool;

  // ---- this workgroup's share of the tiles.  Workgroups are dealt round-robin
  // to the 8 XCDs: neighbours in the tile order go to one XCD, so that the row
  // tiles of a sequence share its L2.
  int g = blockIdx.x;
  if (p.wgs % 8 == 0) g = (g & 7) * (p.wgs >> 3) + (g >> 3);
  int4* joins = reinterpret_cast<int4*>(p.joins);
  int4 join = make_int4(0, 0, 0, g);
  int at, end, b, seq_at, share = 1;
  if (p.unit_tiles > 0) {
    b = g / p.unit_tiles;
    const int rt = g - b * p.unit_tiles;
    const Seq sq = seq_of(p, b, ROWS);
    if (rt >= sq.nrt) return;
    if (sq.nt == 0) {
      zero_unit<R, ROWS>(p, sq, rt, tid >> 6, kLThreads / 64, lane);
      return;
    }
    seq_at = 0;
    at = rt * sq.nt;  // (the lead is zero here)
    end = at + sq.nt;
  } else {
    int* pref = reinterpret_cast<int*>(smem);
    int* tmp = pref + kMaxBatch;
    int total = 0;
    for (int c = 0; c < p.a.batch; c += kLThreads) {
      const int b = c + tid;
      int v = 0;
      if (b < p.a.batch) {
        const Seq s = seq_of(p, b, ROWS);
        v = s.nt > 0 ? (s.nt + p.lead) * s.nrt : 0;
      }
      int sum;
      const int incl = block_scan(v, tmp, sum);
      if (b < p.a.batch) pref[b] = total + incl - v;
      total += sum;
    }
    __syncthreads();
    share = max(min_share(total), (total + p.wgs - 1) / p.wgs);
    int64_t at64 = (int64_t)g * share;
    if (at64 >= total) {  // uniform
      if (tid == 0 && p.row_tiles == 0) joins[g] = join;
      return;
    }
    at = (int)at64;
    end = (int)min((int64_t)total, at64 + share);
    {
      int lo = 0, hi = p.a.batch;  // last b with pref[b] <= at (sequences without tiles lie before it)
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (pref[mid] <= at) lo = mid;
        else hi = mid;
      }
      b = __builtin_amdgcn_readfirstlane(lo);
    }
    seq_at = __builtin_amdgcn_readfirstlane(pref[b]);
    at = __builtin_amdgcn_readfirstlane(at);
    __syncthreads();  // the ring is free from here on
  }

  while (at < end) {
    const Seq sq = seq_of(p, b, ROWS);
    const int unit = sq.nt + p.lead, seq_span = sq.nt > 0 ? unit * sq.nrt : 0;
    if (at >= seq_at + seq_span) {
      seq_at += seq_span;
      ++b;
      continue;
    }
    const int rt = __builtin_amdgcn_readfirstlane((at - seq_at) / unit);
    const int off = at - seq_at - rt * unit, take = min(unit - off, end - at);
    const int t0 = max(0, off - p.lead), t1 = off + take - p.lead;
    at += take;
    if (t1 <= t0) continue;  // the share ends before the unit's first tile
    // a unit that starts here and goes on: its parts are this one and those of
    // the workgroups behind
    if (t0 == 0 && p.unit_tiles == 0) {
      if (t1 < sq.nt) join = make_int4(b, rt, 1 + (sq.nt - t1 + share - 1) / share, g);
      if (tid == 0 && p.row_tiles > 0) joins[b * p.row_tiles + rt] = join;
    }
    const int n_rows = min(ROWS, sq.lq * p.a.heads - rt * ROWS);
    const int lk = sq.lk;

    const int32_t* bt = pool.tables + (int64_t)b * pool.bt_stride;

    // ---- Q's rows, whole lines at a time, into the last two stages (rows past the
    // end repeat the last): those of a wave are an eighth
    {
      constexpr int kMine = ROWS / 8;
      const int ln = fresh(lane);
      const uint32_t qa = lds0 + 2 * D::kStageB;
      auto row_of = [&](int r, int& tok, int& hd) __attribute__((always_inline)) {
        const int row = rt * ROWS + min(r, n_rows - 1);
        tok = (int)div_by((uint32_t)row, p.heads);
        hd = row - tok * p.a.heads;
      };
#pragma unroll
      for (int i = 0; i < kMine / D::kRowsPerDma; ++i) {
        const int r = kMine * wave + i * D::kRowsPerDma + (D::kRowsPerDma == 1 ? 0 : ln >> 5);
        int tok, hd;
        row_of(r, tok, hd);
        lds_dma16(p.a.q_lat + (int64_t)(sq.q0 + tok) * p.a.ql_ts + hd * p.a.ql_hs +
                      8 * ((ln & (D::kRowB / 16 - 1)) ^ swz256(r)),
                  qa + (uint32_t)(kMine * wave * D::kRowB + 1024 * i));
      }
      constexpr int kC = D::kRopeB / 16;
      if (ln < kMine * kC) {
        const int r = kMine * wave + ln / kC;
        int tok, hd;
        row_of(r, tok, hd);
        lds_dma16(p.a.q_rope + (int64_t)(sq.q0 + tok) * p.a.qr_ts + hd * p.a.qr_hs +
                      8 * ((ln & (kC - 1)) ^ rope_swz<DR>(r)),
                  qa + (uint32_t)(ROWS * D::kRowB + kMine * wave * D::kRopeB));
      }
    }

    if (wave < 4) {
      // ================= scores
      const int tb = wave & 1, rw = (wave >> 1) * 16 * D::kNr;
      const int ln = fresh(lane), l16 = ln & 15, qd = ln >> 4;
      TileLoader<D, R, DR, D::kVDma, D::kSDma, ROWS == 32> loader(pool, bt, lds0, wave, ln, t0, lk, p.pages8);
#pragma unroll 1
      for (int t = t0; t < min(t0 + 2, t1); ++t) loader.issue(t);
      bf16x8 q[D::kNr][D::kKs + D::kRs];
      int lim[D::kNr];  // tokens a row sees
#pragma unroll
      for (int r = 0; r < D::kNr; ++r) {
        const int row = rt * ROWS + min(rw + 16 * r + l16, n_rows - 1);
        lim[r] = min(lk, max(0, sq.first + (int)div_by((uint32_t)row, p.heads) + 1));
      }
      // first tile a row of this tile does not see in full
      const int tok_first = (int)div_by((uint32_t)(rt * ROWS), p.heads);
      const int free_tiles = max(0, min(lk, sq.first + tok_first + 1)) / kTile;
      // The reference of a half tile's P: the one the value waves ask for (the
      // maximum two tiles ago, where that passes O's reference by the slack) or
      // this wave's own last one; a half tile whose maximum passes that by kJump
      // takes its maximum, rounded up.  The value waves bring the halves together.
      float own_ref[D::kNr], l_sum[D::kNr];
#pragma unroll
      for (int r = 0; r < D::kNr; ++r) {
        own_ref[r] = kNoMax;
        l_sum[r] = 0.f;
      }
      // reads of K: row 16 tb + l16, chunk 4 ks + qd
      const int krow = 16 * tb + l16;
      uint32_t koff[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) koff[i] = lds0 + krow * D::kRowB + 16 * ((4 * i + qd) ^ swz256(krow));
      uint32_t roff[D::kRs];
#pragma unroll
      for (int i = 0; i < D::kRs; ++i)
        roff[i] = lds0 + D::kLatB + krow * D::kRopeB + 16 * ((4 * i + qd) ^ rope_swz<DR>(krow));
      wait_vm<0>();
      lds_barrier();  // Q and the first two tiles are there
#pragma unroll
      for (int r = 0; r < D::kNr; ++r) {
        const int row = rw + 16 * r + l16;
        const uint32_t qa = lds0 + 2 * D::kStageB;
#pragma unroll
        for (int ks = 0; ks < D::kKs; ++ks)
          q[r][ks] = as_bf16x8(lds_ld16(qa + row * D::kRowB + 16 * ((4 * ks + qd) ^ swz256(row))));
#pragma unroll
        for (int ks = 0; ks < D::kRs; ++ks)
          q[r][D::kKs + ks] = as_bf16x8(
              lds_ld16(qa + ROWS * D::kRowB + row * D::kRopeB + 16 * ((4 * ks + qd) ^ rope_swz<DR>(row))));
      }
      wait_lgkm0();
      lds_barrier();  // the stages that held Q are free
      for (int t = t0; t < t1; ++t) {
        const uint32_t st = (uint32_t)((t - t0) & (kLStages - 1)) * D::kStageB;
        float ask[D::kNr];  // (first two tiles: not written yet)
        {
          const float* asks = reinterpret_cast<const float*>(smem + D::kAskOff + ((t - 1) & 1) * (ROWS * 4));
#pragma unroll
          for (int r = 0; r < D::kNr; ++r) ask[r] = asks[rw + 16 * r + l16];
        }
        f32x4 s[D::kNr];
        float mx[D::kNr];
#pragma unroll
        for (int r = 0; r < D::kNr; ++r) s[r] = f32x4{0.f, 0.f, 0.f, 0.f};
        uint32_t ka[4], ra[D::kRs];
#pragma unroll
        for (int i = 0; i < 4; ++i) ka[i] = fresh_addr(koff[i] + st);
#pragma unroll
        for (int i = 0; i < D::kRs; ++i) ra[i] = fresh_addr(roff[i] + st);
        // tile t + 2's loads (into the stage of tile t - 2) go between the products
        const bool more = t + 2 < t1;
        bool spread = false;
        if (more) {
          loader.prepare(t + 2);
          spread = loader.rows8;
          if (!spread) loader.load_rows();
        }
        // every read is issued kAhead k-steps before the products it feeds
        constexpr int kAll = D::kKs + D::kRs, kAhead = 6, kEach = kAll / D::kSDma;
        bf16x8 a[kAll];
        auto read_k = [&](int ks) __attribute__((always_inline)) {
          a[ks] = as_bf16x8(ks < D::kKs ? lds_ld16(ka[ks & 3] + (ks >> 2) * 256)
                                        : lds_ld16(ra[(ks - D::kKs) % D::kRs]));
        };
#pragma unroll
        for (int ks = 0; ks < kAhead; ++ks) read_k(ks);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int ks = 0; ks < kAll; ++ks) {
#pragma unroll
          for (int r = 0; r < D::kNr; ++r)
            s[r] = mfma16(a[ks], q[r][ks], s[r]);
          if (ks + kAhead < kAll) read_k(ks + kAhead);
          __builtin_amdgcn_sched_barrier(0);
          if (ks % kEach == kEach - 1 && ks / kEach < D::kSDma) {
            if (spread) loader.load(ks / kEach);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
        const int j0 = t * kTile + 16 * tb + 4 * qd;
        if (t >= free_tiles) {
#pragma unroll
          for (int r = 0; r < D::kNr; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[r][i] = j0 + i < lim[r] ? s[r][i] : -INFINITY;
        }
#pragma unroll
        for (int r = 0; r < D::kNr; ++r)
          mx[r] = __builtin_fmaxf(__builtin_fmaxf(s[r][0], s[r][1]), __builtin_fmaxf(s[r][2], s[r][3]));
#pragma unroll
        for (int r = 0; r < D::kNr; ++r) mx[r] = max_xor16(mx[r]);
#pragma unroll
        for (int r = 0; r < D::kNr; ++r) mx[r] = max_xor32(mx[r]);
        float corr[D::kNr];
#pragma unroll
        for (int r = 0; r < D::kNr; ++r) {
          mx[r] *= p.scale_log2;  // positive
          const float base = t > t0 + 1 ? __builtin_fmaxf(own_ref[r], ask[r]) : own_ref[r];
          const float ref = mx[r] > base + kJump ? __builtin_ceilf(mx[r]) : base;
          corr[r] = fast_exp2(own_ref[r] - ref);
          own_ref[r] = ref;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int r = 0; r < D::kNr; ++r) s[r][i] = fast_exp2(__builtin_fmaf(s[r][i], p.scale_log2, -own_ref[r]));
#pragma unroll
        for (int r = 0; r < D::kNr; ++r) {
          // tokens 16 tb + 4 qd .. + 3 of the row: chunk 2 tb + (qd & 1), half
          // qd >> 1 of it, the order in which the transposing reads take V
          const int row = rw + 16 * r + l16;
          const int c = (2 * tb + (qd & 1)) ^ ((row >> 2) & 3);
          *reinterpret_cast<u32x2*>(smem + D::kPOff + (t & 1) * D::kPB + row * 64 + 16 * c + 8 * (qd >> 1)) =
              u32x2{pack_bf16x2(s[r][0], s[r][1]), pack_bf16x2(s[r][2], s[r][3])};
        }
        // lanes 16 r + l16 write row block r
        if (qd < D::kNr) {
          const int at = (t & 1) * D::kRefB + (tb * ROWS + rw + ln) * 4;
          *reinterpret_cast<float*>(smem + D::kMaxOff + at) = qd == 0 ? mx[0] : mx[D::kNr - 1];
          *reinterpret_cast<float*>(smem + D::kRefOff + at) = qd == 0 ? own_ref[0] : own_ref[D::kNr - 1];
        }
#pragma unroll
        for (int r = 0; r < D::kNr; ++r) l_sum[r] = l_sum[r] * corr[r] + ((s[r][0] + s[r][1]) + (s[r][2] + s[r][3]));
        landed<D::kSDma>(more);
        wait_lgkm0();
        lds_barrier();
      }
      lds_barrier();  // the value waves' last step
      // ---- row sums, relative to the last tile's references
      float* sums = reinterpret_cast<float*>(smem + D::kSumOff);
#pragma unroll
      for (int r = 0; r < D::kNr; ++r) {
        const float l = sum_xor32(sum_xor16(l_sum[r]));
        const int row = rw + 16 * r + l16;
        if (qd == 0) sums[tb * ROWS + row] = l;
      }
      wait_lgkm0();
      lds_barrier();
    } else {
      // ================= values
      const int pw = wave - 4;
      const int lv = fresh(lane), n = lv & 31, h = lv >> 5;
      TileLoader<D, R, DR, 0, D::kVDma, ROWS == 32> loader(pool, bt, lds0, pw, lv, t0, lk, p.pages8);
      f32x16 acc[D::kDt][D::kRb] = {};
      // transposing reads of V^T: lane 16 gamma + s reads row 4 h + s / 4 (+ 8)
      // of a 16-token step, columns 32 dt + 16 (gamma % 2) + 4 (s % 4)
      const int ts = lv & 15, gamma = lv >> 4;
      const int tr = 4 * h + (ts >> 2);
      uint32_t voff0[D::kDt], voff1[D::kDt];
#pragma unroll
      for (int dt = 0; dt < D::kDt; ++dt) {
        const int c = 4 * (pw * D::kDt + dt) + 2 * (gamma & 1) + ((ts & 3) >> 1);
        voff0[dt] = lds0 + tr * D::kRowB + 16 * (c ^ swz256(tr)) + 8 * (ts & 1);
        voff1[dt] = lds0 + (tr + 8) * D::kRowB + 16 * (c ^ swz256(tr + 8)) + 8 * (ts & 1);
      }
      uint32_t poff[D::kRb][2];
#pragma unroll
      for (int rb = 0; rb < D::kRb; ++rb)
#pragma unroll
        for (int u = 0; u < 2; ++u)
          poff[rb][u] = lds0 + D::kPOff + (32 * rb + n) * 64 + 16 * ((2 * u + h) ^ ((n >> 2) & 3));
      float m_ref[D::kRb];  // reference of O
#pragma unroll
      for (int rb = 0; rb < D::kRb; ++rb) m_ref[rb] = kNoMax;
      bf16x8 pt[D::kRb][2];
      bf16x8 v0[D::kDt], v1[D::kDt];  // V^T of the first and second 16 tokens of a tile
      auto read_v = [&](bf16x8(&v)[D::kDt], int u, int t) __attribute__((always_inline)) {
        const uint32_t st = (uint32_t)((t - t0) & (kLStages - 1)) * D::kStageB;
#pragma unroll
        for (int dt = 0; dt < D::kDt; ++dt) {
          const u32x2 lo = lds_tr8(fresh_addr(voff0[dt] + st) + 16 * u * D::kRowB);
          const u32x2 hi = lds_tr8(fresh_addr(voff1[dt] + st) + 16 * u * D::kRowB);
          v[dt] = as_bf16x8(u32x4{lo[0], lo[1], hi[0], hi[1]});
        }
      };
      // The products of 16 tokens; between(i) runs behind the i-th.
      auto product = [&](const bf16x8(&v)[D::kDt], int u, auto&& between) __attribute__((always_inline)) {
#pragma unroll
        for (int dt = 0; dt < D::kDt; ++dt)
#pragma unroll
          for (int rb = 0; rb < D::kRb; ++rb) {
            acc[dt][rb] = mfma32(v[dt], pt[rb][u], acc[dt][rb]);
            between(dt * D::kRb + rb);
          }
      };
#pragma unroll 1
      for (int t = t0; t < t0 + 3; ++t) {
        if (t == t0 + 2) {
          wait_vm<0>();
          lds_barrier();  // Q and the first two tiles are there
          lds_barrier();  // Q is in the score waves' registers
        }
        if (t < t1) loader.issue(t);
      }
      landed<D::kVDma>(t0 + 2 < t1);
      lds_barrier();  // the score waves' first step is done
      bool spread = false;  // the next tile's loads go between the products
      auto plan = [&](int t) __attribute__((always_inline)) {
        if (t < t1) loader.prepare(t);
        spread = t < t1 && loader.rows8;
      };
      // Step t: tile t - 1's operands while the score waves multiply tile t, then its
      // products while they take the exponentials, with tile t + 2's loads (into the
      // stage of tile t - 2) between them.
      for (int t = t0 + 1; t <= t1; ++t) {
        constexpr int kProducts = 2 * D::kDt * D::kRb;
        const uint32_t odd = (uint32_t)((t - 1) & 1);
        const float* refs = reinterpret_cast<const float*>(smem + D::kRefOff + odd * D::kRefB);
        const float* maxes = reinterpret_cast<const float*>(smem + D::kMaxOff + odd * D::kRefB);
        float a0[D::kRb], a1[D::kRb], m0[D::kRb], m1[D::kRb];
#pragma unroll
        for (int rb = 0; rb < D::kRb; ++rb) {
          a0[rb] = refs[32 * rb + n];
          a1[rb] = refs[ROWS + 32 * rb + n];
          m0[rb] = maxes[32 * rb + n];
          m1[rb] = maxes[ROWS + 32 * rb + n];
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int rb = 0; rb < D::kRb; ++rb) pt[rb][u] = as_bf16x8(lds_ld16(poff[rb][u] + odd * D::kPB));
        read_v(v0, 0, t - 1);
        read_v(v1, 1, t - 1);
        __builtin_amdgcn_sched_barrier(0);
        plan(t + 2);
        if (t + 2 < t1 && !spread) loader.load_rows();
        // O's reference is the largest of those of its parts: where a half tile's
        // is another (seldom), O or that half's P is brought to it.
        // (two branches: with one the compiler keeps two copies of O)
        bool moved = false, differ = false;
#pragma unroll
        for (int rb = 0; rb < D::kRb; ++rb) moved |= __builtin_fmaxf(a0[rb], a1[rb]) > m_ref[rb];
        if (__builtin_amdgcn_ballot_w64(moved) != 0) {
#pragma unroll
          for (int rb = 0; rb < D::kRb; ++rb) {
            const float m_new = __builtin_fmaxf(m_ref[rb], __builtin_fmaxf(a0[rb], a1[rb]));
            const float up = fast_exp2(m_ref[rb] - m_new);
            m_ref[rb] = m_new;
#pragma unroll
            for (int dt = 0; dt < D::kDt; ++dt) acc[dt][rb] = acc[dt][rb] * up;
          }
        }
#pragma unroll
        for (int rb = 0; rb < D::kRb; ++rb) differ |= (a0[rb] != m_ref[rb]) | (a1[rb] != m_ref[rb]);
        if (__builtin_amdgcn_ballot_w64(differ) != 0) {
#pragma unroll
          for (int rb = 0; rb < D::kRb; ++rb)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              // a power of two: bf16 values times it are exact
              const float f = __builtin_amdgcn_ldexpf(1.f, (int)fmaxf((u ? a1[rb] : a0[rb]) - m_ref[rb], -256.f));
              u32x4 w = as_u32x4(pt[rb][u]);
#pragma unroll
              for (int e = 0; e < 4; ++e) w[e] = pack_bf16x2(bf16_lo(w[e]) * f, bf16_hi(w[e]) * f);
              pt[rb][u] = as_bf16x8(w);
            }
        }
        auto loads = [&](int i) __attribute__((always_inline)) {
          __builtin_amdgcn_sched_barrier(0);
          if (spread) {
#pragma unroll
            for (int k = i * D::kVDma / kProducts; k < (i + 1) * D::kVDma / kProducts; ++k) loader.load(k);
          }
          __builtin_amdgcn_sched_barrier(0);
        };
        product(v0, 0, loads);
        product(v1, 1, [&](int i) __attribute__((always_inline)) { loads(kProducts / 2 + i); });
        if (pw == 0) {
#pragma unroll
          for (int rb = 0; rb < D::kRb; ++rb) {
            const float mx = __builtin_fmaxf(m0[rb], m1[rb]);
            *reinterpret_cast<float*>(smem + D::kAskOff + (t & 1) * (ROWS * 4) + (32 * rb + n) * 4) =
                mx > m_ref[rb] + kSlack ? __builtin_ceilf(mx) : m_ref[rb];
          }
        }
        landed<D::kVDma>(t + 2 < t1);
        wait_lgkm0();
        lds_barrier();
      }
      lds_barrier();  // sums are there
      const int le = fresh(lane), ne = le & 31, he = le >> 5;
      // a row's sum: those of its half tiles, brought to O's reference
      const float* sums = reinterpret_cast<const float*>(smem + D::kSumOff);
      const float* refs = reinterpret_cast<const float*>(smem + D::kRefOff + ((t1 - 1) & 1) * D::kRefB);
      auto row_sum = [&](int r, float m) __attribute__((always_inline)) {
        return sums[r] * fast_exp2(refs[r] - m) + sums[ROWS + r] * fast_exp2(refs[ROWS + r] - m);
      };
      if (t0 == 0 && t1 == sq.nt) {
#pragma unroll
        for (int rb = 0; rb < D::kRb; ++rb) {
          const int r = 32 * rb + ne;
          const float l = row_sum(r, m_ref[rb]);
          const float inv = l > 0.f ? 1.f / l : 0.f;
          if (r < n_rows) {
            const int row = rt * ROWS + r;
            const int tok = (int)div_by((uint32_t)row, p.heads), hd = row - tok * p.a.heads;
            uint16_t* o = p.a.out + (int64_t)(sq.q0 + tok) * p.a.o_ts + hd * p.a.o_hs + pw * (R / 4) + 4 * he;
#pragma unroll
            for (int dt = 0; dt < D::kDt; ++dt)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const f32x16& v = acc[dt][rb];
                *reinterpret_cast<u32x2*>(o + 32 * dt + 8 * i) =
                    u32x2{pack_bf16x2(v[4 * i] * inv, v[4 * i + 1] * inv),
                          pack_bf16x2(v[4 * i + 2] * inv, v[4 * i + 3] * inv)};
              }
          }
        }
      } else {
        const int slot = 2 * g + (t0 == 0 ? 1 : 0);
        float* dst = p.parts + (int64_t)slot * (ROWS * R) + 4 * le;
#pragma unroll
        for (int dt = 0; dt < D::kDt; ++dt)
#pragma unroll
          for (int rb = 0; rb < D::kRb; ++rb)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const f32x16& v = acc[dt][rb];
              *reinterpret_cast<f32x4*>(dst + 256 * (((pw * D::kDt + dt) * D::kRb + rb) * 4 + i)) =
                  f32x4{v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]};
            }
        if (pw == 0 && he == 0) {
#pragma unroll
          for (int rb = 0; rb < D::kRb; ++rb)
            *reinterpret_cast<f32x2*>(p.stats + ((int64_t)slot * ROWS + 32 * rb + ne) * 2) =
                f32x2{m_ref[rb], row_sum(32 * rb + ne, m_ref[rb])};
        }
      }
    }
    __syncthreads();  // LDS is free for the next segment
  }
  if (tid == 0 && p.row_tiles == 0 && p.unit_tiles == 0) joins[g] = join;
}

// Joins the parts of every (sequence, row tile) that more than one workgroup
// worked on: o = sum_p w_p o_p / sum_p w_p l_p, w_p = 2^(m_p - max m), and gives
// sequences without any cached token zero rows.  A part's O lies as the
// accumulators held it, 256 floats a slice (column block, row block, quarter).
// Few parts: each wave joins slices of its own.  Many: the waves of a workgroup
// share a slice's parts and add up through LDS.
constexpr int kJoinWaves = 8, kJoinFly = 4;  // parts in flight a wave

struct Joined {
  float m, l;
  f32x4 acc;
};

template <int R, int ROWS>
__device__ __forceinline__ Joined join_parts(const AttnParams& p, int g, int parts, int first, int step, int sl, int r,
                                             int lane) {
  Joined j = {kNoMax, 0.f, {0.f, 0.f, 0.f, 0.f}};
  for (int i0 = first; i0 < parts; i0 += step * kJoinFly) {
    f32x2 ml[kJoinFly];
    f32x4 v[kJoinFly];
#pragma unroll
    for (int k = 0; k < kJoinFly; ++k) {
      const int i = min(i0 + step * k, parts - 1);  // past the last: that one again, without weight
      const int64_t slot = 2 * (g + i) + (i == 0 ? 1 : 0);
      ml[k] = *reinterpret_cast<const f32x2*>(p.stats + (slot * ROWS + r) * 2);
      v[k] = *reinterpret_cast<const f32x4*>(p.parts + slot * (ROWS * R) + 256 * sl + 4 * lane);
    }
    float m_new = j.m;
#pragma unroll
    for (int k = 0; k < kJoinFly; ++k) m_new = __builtin_fmaxf(m_new, ml[k][0]);
    const float ca = fast_exp2(j.m - m_new);
    j.acc = j.acc * ca;
    j.l *= ca;
#pragma unroll
    for (int k = 0; k < kJoinFly; ++k) {
      // (a part whose rows saw nothing has l = 0 and O = 0)
      const float c = i0 + step * k < parts ? fast_exp2(ml[k][0] - m_new) : 0.f;
      j.acc = j.acc + v[k] * c;
      j.l += ml[k][1] * c;
    }
    j.m = m_new;
  }
  return j;
}

template <int R, int ROWS>
__global__ void __launch_bounds__(64 * kJoinWaves) latent_merge_kernel(AttnParams p) {
  constexpr int kRb = ROWS / 32, kSlices = ROWS * R / 256;
  __shared__ f32x4 s_acc[kJoinWaves][64];
  __shared__ f32x2 s_ml[kJoinWaves][32];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 31, h = lane >> 5;
  const int4 join = reinterpret_cast<const int4*>(p.joins)[blockIdx.x];
  for (int b = blockIdx.x * gridDim.y + blockIdx.y; b < p.a.batch; b += gridDim.x * gridDim.y) {
    const Seq sq = seq_of(p, b, ROWS);
    if (sq.nt > 0) continue;
    for (int rt = 0; rt < sq.nrt; ++rt) zero_unit<R, ROWS>(p, sq, rt, wave, kJoinWaves, lane);
  }
  // Where the entries are the units', one is written by the workgroup that starts
  // its unit: there is none for a unit without tiles or without rows.
  int b = join.x, rt = join.y;
  if (p.row_tiles > 0) {
    b = blockIdx.x / p.row_tiles;
    rt = blockIdx.x - b * p.row_tiles;
  }
  if (p.row_tiles == 0 && join.z == 0) return;
  const Seq sq = seq_of(p, b, ROWS);
  if (sq.nt == 0 || rt >= sq.nrt || join.z == 0) return;
  const int parts = join.z, g = join.w;
  const int n_rows = min(ROWS, sq.lq * p.a.heads - rt * ROWS);
  auto store = [&](int sl, int r, const f32x4& o, float l) __attribute__((always_inline)) {
    if (r >= n_rows) return;
    const float inv = l > 0.f ? 1.f / l : 0.f;
    const int row = rt * ROWS + r;
    const int tok = (int)div_by((uint32_t)row, p.heads), hd = row - tok * p.a.heads;
    const int d = 32 * (sl / (4 * kRb)) + 8 * (sl & 3) + 4 * h;
    *reinterpret_cast<u32x2*>(p.a.out + (int64_t)(sq.q0 + tok) * p.a.o_ts + hd * p.a.o_hs + d) =
        u32x2{pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv)};
  };
  if (parts <= 2 * kJoinFly) {
    for (int sl = blockIdx.y * kJoinWaves + wave; sl < kSlices; sl += gridDim.y * kJoinWaves) {
      const int r = 32 * ((sl >> 2) % kRb) + n;
      const Joined j = join_parts<R, ROWS>(p, g, parts, 0, 1, sl, r, lane);
      store(sl, r, j.acc, j.l);
    }
    return;
  }
  for (int sl = blockIdx.y; sl < kSlices; sl += gridDim.y) {
    const int r = 32 * ((sl >> 2) % kRb) + n;
    const Joined j = join_parts<R, ROWS>(p, g, parts, wave, kJoinWaves, sl, r, lane);
    s_acc[wave][lane] = j.acc;
    if (h == 0) s_ml[wave][n] = f32x2{j.m, j.l};
    __syncthreads();
    if (wave == 0) {
      float mm = kNoMax;
#pragma unroll
      for (int w = 0; w < kJoinWaves; ++w) mm = __builtin_fmaxf(mm, s_ml[w][n][0]);
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
      float l = 0.f;
#pragma unroll
      for (int w = 0; w < kJoinWaves; ++w) {
        const float c = fast_exp2(s_ml[w][n][0] - mm);
        o = o + s_acc[w][lane] * c;
        l += s_ml[w][n][1] * c;
      }
      store(sl, r, o, l);
    }
    __syncthreads();
  }
}

// Rows of a workgroup: 64, or 32 where a sequence has no more (4 096 tokens each,
// 256 sequences by 16 heads: 203 us against 234 with 64 rows, 64 by 32 heads 78
// against 91).
int rows_of(int max_q, int heads) { return (int64_t)max_q * heads <= 32 ? 32 : 64; }

// Workgroups of a cut launch of at most `most_tiles`: as many as min_share
// leaves work for, whatever there is.
int wgs_of(int64_t most_tiles) {
  int64_t n = 1;
  for (const int64_t t : {std::min<int64_t>(most_tiles, 64), std::min<int64_t>(most_tiles, 384), most_tiles})
    n = std::max<int64_t>(n, (t + min_share(t) - 1) / min_share(t));
  return (int)std::min<int64_t>(n, kWgs);
}

size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

}  // namespace

size_t latent_attn_workspace(int32_t batch, int32_t max_q, int32_t heads, int32_t latent, int64_t span,
                             const char** why) {
  const int rows = rows_of(max_q, heads);
  const int64_t row_tiles = ((int64_t)max_q * heads + rows - 1) / rows;
  const int64_t tiles = (span + kTile - 1) / kTile + kLead;
  *why = nullptr;
  if (batch > kMaxBatch) *why = "more than 16384 sequences";
  else if (span > 0x7fffffff - 65 * kTile ||  // a loader makes row numbers up to 64 tiles ahead
           (int64_t)max_q * heads > 0x7fffffff - 64 ||
           tiles > (0x7fffffff - kWgs) / std::max<int64_t>(1, row_tiles * batch))
    *why = "more than 2^31 tiles of work";
  if (*why) return 0;
  const int wgs = wgs_of(row_tiles * batch * (tiles - kLead));
  return align256((size_t)16 * wgs) + align256((size_t)2 * wgs * rows * 8) + (size_t)2 * wgs * rows * latent * 4;
}

template <int R, int DR, int ROWS>
static int attn_launch(const char* name, AttnParams p, int64_t units, void* workspace, hipStream_t s) {
  char* ws = (char*)workspace;
  p.joins = (int32_t*)ws;
  ws += align256((size_t)16 * p.wgs);
  p.stats = (float*)ws;
  ws += align256((size_t)2 * p.wgs * ROWS * 8);
  p.parts = (float*)ws;
  latent_attn_kernel<R, DR, ROWS><<<dim3((unsigned)p.wgs), dim3(kLThreads), 0, s>>>(p);
  if (int rc = launch_status(name)) return rc;
  if (p.unit_tiles > 0) return PA_OK;
  // a slice a wave, or a slice a workgroup for few joins (of many parts)
  const int64_t joins = p.row_tiles > 0 ? units : p.wgs;
  constexpr int kSlices = ROWS * R / 256;
  const unsigned ny = (unsigned)std::max<int64_t>(16, std::min<int64_t>(kSlices, 1024 / joins));
  latent_merge_kernel<R, ROWS><<<dim3((unsigned)joins, ny), dim3(64 * kJoinWaves), 0, s>>>(p);
  return launch_status(name);
}

int latent_attn_launch(const char* name, const LatentAttn& a, int latent, int rope, void* workspace, hipStream_t s) {
  AttnParams p;
  p.a = a;
  p.heads = magic_div((uint32_t)a.heads);
  p.scale_log2 = a.scale * kLog2e;
  // eight rows' byte offsets from the first fit 32 bits
  p.pages8 = a.pool.page.d % 8 == 0 && a.pool.slot_stride >= 0 && a.pool.slot_stride < (1 << 27);
  const int rows = rows_of(a.max_q, a.heads);
  const int64_t row_tiles = ((int64_t)a.max_q * a.heads + rows - 1) / rows;
  const int64_t span = (int64_t)a.pool.pages_per_seq * a.pool.page.d;
  const int64_t units = row_tiles * a.batch;
  p.wgs = wgs_of(units * ((span + kTile - 1) / kTile));
  p.row_tiles = units <= p.wgs ? (int)row_tiles : 0;
  // Short block tables take a workgroup a unit, without the cut's scan and the
  // merge's launch.  16 heads, whole calls: 4 sequences of 4 tiles 18.9 us against
  // 20.1, of 8 tiles 22.5 against 20.5 cut; 64 sequences of 8 tiles 26.6 against
  // 30.6, of 16 tiles 33.1 against 35.7, of 24 tiles 39.6 against 37.9.
  const int64_t tiles = (span + kTile - 1) / kTile;
  // (a grid has fewer than 2^32 threads along x)
  p.unit_tiles = tiles <= (units < 64 ? kDirect : kDirectMany) && units * kLThreads <= 0xffffffffll ? (int)row_tiles : 0;
  if (p.unit_tiles > 0) p.wgs = (int)units;
  // The start and end of a unit (Q, the first tiles, O) take about as long as
  // kLead tiles; counted as such, a workgroup that gets several short pieces
  // gets fewer tiles: 64 sequences of 512-8 192 tokens by 128 heads 157.7 us with
  // 0, 143.8, 138.7, 138.0 with 4, 7, 10; by 32 heads 89.2, 84.8, 78.6, 78.2; 256
  // by 16 heads 247.0, 240.3, 239.5, 242.7.  Where a workgroup has few tiles anyway
  // they are dealt as they are.
  p.lead = p.unit_tiles == 0 && units * tiles >= 16 * kWgs ? kLead : 0;
  p.joins = nullptr;
  p.parts = p.stats = nullptr;
#define PA_LATENT_CASE(R, DR)                                                 \
  if (latent == R && rope == DR)                                              \
    return rows == 32 ? attn_launch<R, DR, 32>(name, p, units, workspace, s)  \
                      : attn_launch<R, DR, 64>(name, p, units, workspace, s);
  PA_LATENT_CASE(512, 64)
  PA_LATENT_CASE(512, 32)
  PA_LATENT_CASE(256, 64)
  PA_LATENT_CASE(256, 32)
#undef PA_LATENT_CASE
  return fail(PA_ERR_UNSUPPORTED, "%s: latent_dim %d with rope_dim %d", name, latent, rope);
}

}  // namespace pa

using namespace pa;

static int latent_decode_need(const char* name, int32_t batch, int32_t num_heads, int32_t latent_dim,
                              int32_t pages_per_seq, int32_t page_size, size_t& q_bytes, size_t& need) {
  const char* why;
  const size_t attn = latent_attn_workspace(batch, 1, num_heads, latent_dim, (int64_t)pages_per_seq * page_size, &why);
  if (why) return fail(PA_ERR_UNSUPPORTED, "%s: %s", name, why);
  q_bytes = ((size_t)batch * num_heads * latent_dim * 2 + 255) & ~(size_t)255;
  need = 2 * q_bytes + attn;  // absorbed q, latent outputs, the attention's own
  return PA_OK;
}

extern "C" size_t pa_latent_decode_workspace_size(int32_t batch, int32_t num_heads, int32_t latent_dim,
                                                  int32_t pages_per_seq, int32_t page_size) {
  if (batch <= 0 || num_heads <= 0 || latent_dim <= 0 || pages_per_seq < 0 || page_size <= 0) return 0;
  size_t q, need;
  return latent_decode_need("pa_latent_decode_workspace_size", batch, num_heads, latent_dim, pages_per_seq, page_size,
                            q, need) == PA_OK
             ? need
             : 0;
}

extern "C" int pa_latent_decode(const uint16_t* q_nope, int64_t qn_tok_stride, int64_t qn_head_stride,
                                const uint16_t* q_rope, int64_t qr_tok_stride, int64_t qr_head_stride,
                                const uint16_t* cache, int32_t num_pages, int32_t page_size, int64_t page_stride,
                                int64_t slot_stride, const int32_t* block_tables, int64_t bt_stride,
                                int32_t pages_per_seq, const int32_t* lengths, int32_t batch, int32_t num_heads,
                                int32_t latent_dim, int32_t rope_dim, int32_t nope_dim, int32_t v_dim,
                                const uint16_t* w_uk_t, const uint16_t* w_kv, float scale, uint16_t* out,
                                int64_t out_tok_stride, int64_t out_head_stride, void* workspace,
                                size_t workspace_bytes, void* stream) {
  const char* name = "pa_latent_decode";
  if (batch < 0 || num_heads <= 0 || num_pages <= 0 || page_size <= 0 || pages_per_seq < 0)
    return fail(PA_ERR_INVALID_ARGUMENT, "%s: bad sizes (batch=%d, num_heads=%d, num_pages=%d, page_size=%d, "
                "pages_per_seq=%d)", name, batch, num_heads, num_pages, page_size, pages_per_seq);
  if (!latent_dims_ok(latent_dim, rope_dim) || !latent_head_ok(nope_dim, v_dim))
    return fail(PA_ERR_UNSUPPORTED, "%s: latent_dim %d, rope_dim %d, nope_dim %d, v_dim %d not supported", name,
                latent_dim, rope_dim, nope_dim, v_dim);
  if (num_heads > 65535) return fail(PA_ERR_UNSUPPORTED, "%s: %d heads", name, num_heads);
  if (!(scale > 0.f) || !(scale < INFINITY)) return fail(PA_ERR_INVALID_ARGUMENT, "%s: scale must be positive", name);
  if (batch == 0) return PA_OK;
  if (!q_nope || !q_rope || !cache || !lengths || !w_uk_t || !w_kv || !out || (pages_per_seq && !block_tables))
    return fail(PA_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
  const uintptr_t align = (uintptr_t)q_nope | (uintptr_t)q_rope | (uintptr_t)cache | (uintptr_t)w_uk_t |
                          (uintptr_t)w_kv | (uintptr_t)out | (uintptr_t)workspace;
  if ((align & 15u) || (qn_tok_stride | qn_head_stride | qr_tok_stride | qr_head_stride | page_stride | slot_stride |
                        out_tok_stride | out_head_stride) % 8)
    return fail(PA_ERR_UNSUPPORTED, "%s: operands must be 16-byte aligned with strides multiple of 8", name);
  size_t q_bytes, need;
  if (int rc = latent_decode_need(name, batch, num_heads, latent_dim, pages_per_seq, page_size, q_bytes, need))
    return rc;
  if (!workspace || workspace_bytes < need)
    return fail(PA_ERR_WORKSPACE, "%s: workspace of %zu bytes given, %zu needed", name, workspace_bytes, need);
  hipStream_t s = (hipStream_t)stream;
  uint16_t* q_lat = (uint16_t*)workspace;
  uint16_t* o_lat = (uint16_t*)((char*)workspace + q_bytes);
  HeadProduct hp;
  hp.x = q_nope;
  hp.x_ts = qn_tok_stride;
  hp.x_hs = qn_head_stride;
  hp.w = w_uk_t;
  hp.w_hs = (int64_t)latent_dim * nope_dim;
  hp.y = q_lat;
  hp.y_ts = (int64_t)num_heads * latent_dim;
  hp.y_hs = latent_dim;
  hp.tokens = batch;
  hp.heads = num_heads;
  hp.n = latent_dim;
  hp.k = nope_dim;
  if (int rc = head_product_launch(name, hp, s)) return rc;
  LatentAttn a;
  a.q_lat = q_lat;
  a.ql_ts = (int64_t)num_heads * latent_dim;
  a.ql_hs = latent_dim;
  a.q_rope = q_rope;
  a.qr_ts = qr_tok_stride;
  a.qr_hs = qr_head_stride;
  a.pool = LatentPool{cache, num_pages, magic_div((uint32_t)page_size), page_stride, slot_stride,
                      block_tables, bt_stride, pages_per_seq};
  a.cu_q = nullptr;
  a.cu_k = nullptr;
  a.kv_lens = lengths;
  a.batch = batch;
  a.num_tokens = batch;
  a.heads = num_heads;
  a.max_q = 1;
  a.scale = scale;
  a.out = o_lat;
  a.o_ts = (int64_t)num_heads * latent_dim;
  a.o_hs = latent_dim;
  if (int rc = latent_attn_launch(name, a, latent_dim, rope_dim, (char*)workspace + 2 * q_bytes, s)) return rc;
  hp.x = o_lat;
  hp.x_ts = (int64_t)num_heads * latent_dim;
  hp.x_hs = latent_dim;
  hp.w = w_kv + (int64_t)nope_dim * latent_dim;
  hp.w_hs = (int64_t)(nope_dim + v_dim) * latent_dim;
  hp.y = out;
  hp.y_ts = out_tok_stride;
  hp.y_hs = out_head_stride;
  hp.n = v_dim;
  hp.k = latent_dim;
  return head_product_launch(name, hp, s);
}
