// Attention of sequences that share a prefix, for gfx950.
//
// Sequences stand in groups; the first tokens of a group's sequences lie in the
// same pages.  Decode row by row reads such a prefix once a sequence; here all
// rows of a group, (token, q head of the kv head) pairs, go over it together as
// the rows of one matrix product, and each sequence's own tokens behind it are
// attended to as ever.  The two meet by the log-sum-exp rule
//
//   out = (o_p 2^(m_p - M) + o_s 2^(m_s - M)) / (l_p 2^(m_p - M) + l_s 2^(m_s - M)).
//
// Launches:
//   shared_plan_kernel    reads the lengths, cuts prefixes and own parts for the
//                         chip and writes the lists of work
//   shared_part_kernel    parts of prefixes (128 rows against 32-token tiles,
//                         shared_tile.h), then of the sequences' own tokens: where
//                         each has one new token by decode_run, else by row tiles
//   shared_tile_kernel    both by prefill_run's loop (256 rows against 64-token
//                         tiles), where sequences have many new tokens
//   shared_merge_kernel   adds the parts up
//
// 128 sequences of 64 to 1024 own tokens behind 8192 shared ones, 32 / 8 heads: plan
// 6.8 us, parts 64 (behind the prefix alone 42, the own tokens alone 50), merge 6.0;
// the plain decode takes 560 for the same step.
#include <algorithm>
#include <type_traits>

#include "../../include/long_context.h"
#include "decode_impl.h"
#include "long_context.h"
#include "prefill_impl.h"
#include "shared_tile.h"

namespace pa {
namespace {

constexpr int kShPlanThreads = 1024;
constexpr int kShPlanMax = 2048;     // sequences (and groups) that the plan keeps in LDS
constexpr int kShTileSlots = 256;    // workgroups resident at once: of shared_tile_kernel (one a CU)
constexpr int kShPartSlots = 512;    // ... of shared_part_kernel (two a CU)
constexpr int kShMinTiles = 8;       // shortest part of a row tile, in 64-token tiles
constexpr int kShMinChunk = 512;     // shortest part of a sequence's own tokens, in tokens
constexpr int64_t kShMergeFew = 128; // (32 rows, kv head) pairs up to which the merge takes four teams
constexpr int kShBins = 256;         // classes of chunks by length, of 16 tokens
// Time of a 64-token step of a row tile and of a chunk in shared_part_kernel
constexpr int kShTileCost = 3, kShChunkCost = 4;

// One part of a (row range, row tile) pair; every kv head has it.
struct alignas(16) ShTile {
  int32_t table, tile, q0, tokens;  // block-table row, row tile, first token, tokens
  int32_t lk, lo, hi, unit;         // kv length, 64-token tiles [lo, hi), first unit of kv head 0
  int32_t step, pad[3];             // units a kv head
};
// One part of a sequence's own tokens.
struct alignas(16) ShChunk {
  int32_t b, t0, t1, slot;  // slot: part number, bit 31: the whole row
};
// Where the rows of a sequence find their parts.
struct alignas(16) ShSeq {
  int32_t p_unit, p_parts, p_step, p_q0;  // prefix: first unit, parts, units a kv head, first token of the group
  int32_t s_unit, s_parts, s_step, s_q0;  // own part likewise (chunks: first slot; s_step: no parts to add up)
};
constexpr int kShHeader = 64;  // ints: number of tile parts, of chunks

struct SharedParams {
  PrefillParams pre;
  DecodeParams dec;
  const int32_t* cu_q;  // null: one new token a sequence
  const int32_t* lengths;
  const int32_t* cu_groups;
  const int32_t* shared_lens;
  int32_t batch, groups, num_tokens, num_kv_heads, group, span, max_seqlen_q;
  int32_t light;        // row tiles of 128 rows (shared_part_kernel), else of tile_tokens tokens in 256 rows
  int32_t tile_tokens;
  int32_t chunk_cap, zero_rest;
  int32_t cap_tiles, cap_chunks, cap_units;  // what the workspace holds
  int32_t* header;
  int32_t* group_shared;  // [groups] and [batch], where the plan's LDS does not hold them
  ShSeq* seqs;
  ShTile* tiles;
  ShChunk* chunks;
  int32_t* positions;  // [num_tokens] kv index of each token (with cu_q)
  int32_t* owner;      // [num_tokens] its sequence, or -1 (with cu_q)
};

// Sequence b: first token, new tokens that are computed, tokens in all.
__device__ __forceinline__ int3 sh_sequence(const SharedParams& p, int b) {
  const int len = clamp_len(p.lengths, b, p.span);
  if (!p.cu_q) return make_int3(b, len > 0 ? 1 : 0, len);
  const int q0 = p.cu_q[b];
  int n = p.cu_q[b + 1] - q0;
  n = q0 < 0 || q0 >= p.num_tokens ? 0 : min(min(n, p.max_seqlen_q), p.num_tokens - q0);
  return make_int3(q0, max(n, 0), len);
}

__host__ __device__ __forceinline__ int sh_ceil(int a, int b) { return (a + b - 1) / b; }
// Row tiles of `tokens` tokens in a row, and the units (32 rows) of each.
__device__ __forceinline__ int sh_row_tiles(const SharedParams& p, int tokens) {
  return p.light ? sh_ceil(tokens * p.group, kLtRows) : sh_ceil(tokens, p.tile_tokens);
}
__device__ __forceinline__ int sh_units(const SharedParams& p, int tokens, int n) {
  const int most = p.light ? kLtWaves : kWaves;
  return n > 1 ? most : min(most, sh_ceil(tokens * p.group, 32));
}
// 64-token tiles [0, n) that the part k of `parts` ends before.
__device__ __forceinline__ int sh_cut(int n, int k, int parts) { return (int)((double)n * k / parts); }

// Sums and exclusive sums over the workgroup of three numbers a thread.
struct Sh3 {
  int a, b, c;
};
__device__ __forceinline__ Sh3 sh_scan(const Sh3& v, Sh3* s_wave, Sh3& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const Sh3 u = {(int)wave_scan((uint32_t)v.a), (int)wave_scan((uint32_t)v.b), (int)wave_scan((uint32_t)v.c)};
  __syncthreads();  // the last scan's sums have been read
  if (lane == 63) s_wave[wave] = u;
  __syncthreads();
  Sh3 before = {0, 0, 0};
  total = {0, 0, 0};
  for (int i = 0; i < waves; ++i) {
    const Sh3 w = s_wave[i];
    if (i < wave) before = {before.a + w.a, before.b + w.b, before.c + w.c};
    total = {total.a + w.a, total.b + w.b, total.c + w.c};
  }
  return {before.a + u.a - v.a, before.b + u.b - v.b, before.c + u.c - v.c};
}

// Sum and minimum over the wave's lanes (DPP, as wave_scan); every lane gets it.
template <int kCtrl, int kRowMask>
__device__ __forceinline__ float add_dpp(float x) {
  return x + __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), kCtrl, kRowMask, 0xF,
                                                                   false));
}
__device__ __forceinline__ float wave_sum(float x) {
  x = add_dpp<0x111, 0xF>(x);
  x = add_dpp<0x112, 0xF>(x);
  x = add_dpp<0x114, 0xF>(x);
  x = add_dpp<0x118, 0xF>(x);
  x = add_dpp<0x142, 0xA>(x);
  x = add_dpp<0x143, 0xC>(x);
  return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(x), 63));
}
template <int kCtrl, int kRowMask>
__device__ __forceinline__ int min_dpp(int x) {
  return min(x, __builtin_amdgcn_update_dpp(INT_MAX, x, kCtrl, kRowMask, 0xF, false));
}
__device__ __forceinline__ int wave_min(int x) {
  x = min_dpp<0x111, 0xF>(x);
  x = min_dpp<0x112, 0xF>(x);
  x = min_dpp<0x114, 0xF>(x);
  x = min_dpp<0x118, 0xF>(x);
  x = min_dpp<0x142, 0xA>(x);
  x = min_dpp<0x143, 0xC>(x);
  return __builtin_amdgcn_readlane(x, 63);
}

// Workgroup 0 plans; the others (with cu_q) map tokens to sequences and kv
// positions, a token a thread.  kLds: sequences and groups fit the plan's LDS,
// and are read from memory once.
template <bool kLds>
__global__ void __launch_bounds__(kShPlanThreads)
shared_plan_kernel(SharedParams p) {
  const int tid = threadIdx.x, threads = blockDim.x;
  if (blockIdx.x > 0) {
    const int t = (blockIdx.x - 1) * threads + tid;
    if (t >= p.num_tokens) return;
    int lo = 0, hi = p.batch;  // last b with cu_q[b] <= t
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (p.cu_q[mid] <= t) lo = mid;
      else hi = mid;
    }
    const int3 s = sh_sequence(p, lo);
    const int i = t - s.x;
    const bool in = i >= 0 && i < s.y;
    // new token i of n stands at kv index len - n + i, n counted uncut
    p.owner[t] = in ? lo : -1;
    p.positions[t] = in ? s.z - (p.cu_q[lo + 1] - s.x) + i : -1;
    return;
  }
  constexpr int kMax = kLds ? kShPlanMax : 1;
  __shared__ int32_t s_len[kMax], s_q0[kMax], s_n[kMax];     // sequences
  __shared__ int16_t s_of[kMax];                             // their group, or -1
  __shared__ int32_t s_cu[kMax + 1], s_want[kMax];           // groups: cu_groups, then shared tokens
  __shared__ int32_t s_table[kMax], s_gunit[kMax];           // first sequence with tokens, first unit
  __shared__ int32_t s_bins[kShBins];
  __shared__ Sh3 s_wave[kShPlanThreads / 64];
  __shared__ float s_total[3][kShPlanThreads / 64];
  const int lane = tid & 63, wave = tid >> 6, waves = threads >> 6;
  const int hkv = p.num_kv_heads;
  for (int i = tid; i < kShBins; i += threads) s_bins[i] = 0;
  if constexpr (kLds) {
    for (int b = tid; b < p.batch; b += threads) {
      const int3 s = sh_sequence(p, b);
      s_q0[b] = s.x;
      s_n[b] = s.y;
      s_len[b] = s.z;
      s_of[b] = -1;
    }
    for (int g = tid; g <= p.groups; g += threads) s_cu[g] = p.cu_groups[g];
    for (int g = tid; g < p.groups; g += threads) s_want[g] = p.shared_lens[g];
  }
  auto seq = [&](int b) { return kLds ? make_int3(s_q0[b], s_n[b], s_len[b]) : sh_sequence(p, b); };
  auto cu_group = [&](int g) { return kLds ? s_cu[g] : p.cu_groups[g]; };
  auto shared_of = [&](int g) { return kLds ? s_want[g] : p.group_shared[g]; };
  // first token and tokens of a group
  auto group_rows = [&](int g) {
    const int g0 = max(0, cu_group(g)), g1 = min(p.batch, cu_group(g + 1));
    return p.cu_q ? make_int2(p.cu_q[g0], p.cu_q[g1] - p.cu_q[g0]) : make_int2(g0, g1 - g0);
  };
  __syncthreads();
  // ---- groups, a wave each: the shared tokens (whole 64-token tiles, no further
  // than the shortest sequence)
  for (int g = wave; g < p.groups; g += waves) {
    const int g0 = max(0, cu_group(g)), g1 = min(p.batch, cu_group(g + 1));
    int active = 0, least = INT_MAX, first = INT_MAX;  // active, first: uniform
    for (int b0 = g0; b0 < g1; b0 += 64) {
      const int b = b0 + lane;
      int3 s = make_int3(0, 0, 0);
      if (b < g1) {
        s = seq(b);
        if constexpr (kLds) s_of[b] = (int16_t)g;
      }
      const bool has = s.y > 0 && s.z > 0;
      const uint64_t who = __ballot(has);
      if (who && !active) first = b0 + __ffsll((unsigned long long)who) - 1;
      active += __popcll(who);
      if (has) least = min(least, s.z);
    }
    least = wave_min(least);
    if (lane == 0) {
      int shared = 0;
      if (active > 1) {
        const int2 r = group_rows(g);
        if (r.x >= 0 && r.y > 0 && r.y <= p.num_tokens - r.x)
          shared = max(0, min(kLds ? s_want[g] : p.shared_lens[g], least)) & ~(kTileN - 1);
      }
      if constexpr (kLds) {
        s_want[g] = shared;
        s_table[g] = first;
      } else {
        p.group_shared[g] = shared;
        p.group_shared[p.groups + g] = first;
      }
    }
  }
  __syncthreads();
  auto group_of = [&](int b) {
    if constexpr (kLds) return (int)s_of[b];
    int lo = 0, hi = p.groups;  // last g with cu_groups[g] <= b
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (p.cu_groups[mid] <= b) lo = mid;
      else hi = mid;
    }
    return p.groups > 0 && p.cu_groups[lo] <= b && b < p.cu_groups[lo + 1] ? lo : -1;
  };
  auto group_tiles = [&](int g) { return shared_of(g) ? sh_row_tiles(p, group_rows(g).y) : 0; };
  // 64-token tiles of row tile i of n of sequence s behind `shared` tokens
  auto own_tiles = [&](int b, const int3& s, int shared, int i) {
    const int end = p.light ? sh_ceil((i + 1) * kLtRows, p.group) : (i + 1) * p.tile_tokens;  // tokens up to it
    const int hi = min(s.z, s.z - (p.cu_q[b + 1] - p.cu_q[b]) + min(end, s.y));
    return hi <= shared ? 0 : sh_ceil(hi, kTileN) - shared / kTileN;
  };
  // ---- work in all: 64-token tiles of row tiles, row tiles, tokens of chunks
  float tiles = 0.f, pairs = 0.f, own = 0.f;
  for (int g = tid; g < p.groups; g += threads) {
    const int n = group_tiles(g);
    pairs += (float)n;
    tiles += (float)n * (float)(shared_of(g) / kTileN);
  }
  for (int b = tid; b < p.batch; b += threads) {
    const int3 s = seq(b);
    const int g = group_of(b);
    const int shared = g >= 0 ? shared_of(g) : 0;
    if (!p.cu_q) {
      own += (float)max(0, s.z - shared);
    } else if (s.y > 0) {
      const int n = sh_row_tiles(p, s.y);
      pairs += (float)n;
      tiles += (float)n * (float)own_tiles(b, s, shared, n - 1);  // (its row tiles are cut alike)
    }
  }
  tiles = wave_sum(tiles);
  pairs = wave_sum(pairs);
  own = wave_sum(own);
  if (lane == 0) {
    s_total[0][wave] = tiles;
    s_total[1][wave] = pairs;
    s_total[2][wave] = own;
  }
  __syncthreads();
  tiles = pairs = own = 0.f;
  for (int i = 0; i < waves; ++i) {
    tiles += s_total[0][i];
    pairs += s_total[1][i];
    own += s_total[2][i];
  }
  // lists that do not fit (cu_groups or cu_q that fall) are not run: every row is
  // zero.  More row tiles than any that do not fall have are known here already, and
  // below that number the sums of the lists stay far from 2^31.
  auto run_nothing = [&]() {
    if (tid == 0) p.header[0] = p.header[1] = 0;
    for (int b = tid; b < p.batch; b += threads) p.seqs[b] = ShSeq{0, 0, 0, 0, 0, 0, 0, 0};
  };
  if (pairs > (float)p.cap_tiles * 1.001f) {  // uniform
    run_nothing();
    return;
  }
  // (the sums' roundings, below 2^-15 of them, must not make the shares short)
  const float all_tiles = tiles * (float)hkv * 1.0001f, all_pairs = pairs * (float)hkv * 1.0001f;
  const float all_own = own * (float)(hkv * p.dec.hblocks) * 1.0001f;
  // Parts of at most `most` tiles and `chunk` tokens.  Every row tile rounds up,
  // so where there are few of them, and nothing else, an even share of the
  // slots that they leave over makes one round; else a share of all.
  const float slots = (float)(p.light ? kShPartSlots : kShTileSlots);
  float share;
  if (all_own == 0.f && 2.f * all_pairs <= slots) share = all_tiles / (slots - all_pairs);
  else share = (all_tiles * kShTileCost + all_own / kTileN * kShChunkCost) / (slots * kShTileCost);
  const int most = max(kShMinTiles, (int)fminf(share, 1e9f) + 1);
  const int chunk = min(p.chunk_cap, max(kShMinChunk, ((int)fminf(all_own / slots, 1e9f) + 16) & ~15));
  // ---- the lists
  Sh3 base = {0, 0, 0}, sum;  // tile parts, units (of one kv head) and chunks before this round
  for (int g0 = 0; g0 < p.groups; g0 += threads) {
    const int g = g0 + tid;
    int n = 0, parts = 0, step = 0;
    if (g < p.groups) {
      n = group_tiles(g);
      parts = n ? sh_ceil(shared_of(g) / kTileN, most) : 0;
      step = n ? sh_units(p, group_rows(g).y, n) : 0;
    }
    const Sh3 at = sh_scan({n * parts, n * parts * step, 0}, s_wave, sum);
    // a wave writes the entries of each of its groups
    uint64_t todo = __ballot(n > 0);
    while (todo) {
      const int l = __ffsll((unsigned long long)todo) - 1;
      todo &= todo - 1;
      const int gg = __shfl(g, l), nn = __shfl(n, l), pp = __shfl(parts, l), st = __shfl(step, l);
      const int first = base.a + __shfl(at.a, l), unit = base.b + __shfl(at.b, l);
      const int shared = shared_of(gg), kv = shared / kTileN;
      const int table = kLds ? s_table[gg] : p.group_shared[p.groups + gg];
      const int2 r = group_rows(gg);
      for (int i = lane; i < nn * pp && first + i < p.cap_tiles; i += 64) {
        // the parts of one range of tokens stand together: its row tiles share them
        const int k = i / nn, t = i - k * nn;
        p.tiles[first + i] = ShTile{table, t, r.x, r.y, shared, sh_cut(kv, k, pp), sh_cut(kv, k + 1, pp),
                                    (unit + (t * pp + k) * st) * hkv, st, {0, 0, 0}};
      }
      if (lane == l) {
        if constexpr (kLds) s_gunit[gg] = unit * hkv;
        else p.group_shared[2 * p.groups + gg] = unit * hkv;
      }
    }
    base = {base.a + sum.a, base.b + sum.b, 0};
  }
  __syncthreads();
  for (int b0 = 0; b0 < p.batch; b0 += threads) {
    const int b = b0 + tid;
    int3 s = make_int3(0, 0, 0);
    ShSeq q = {0, 0, 0, 0, 0, 0, 0, 0};
    int shared = 0;
    if (b < p.batch) {
      s = seq(b);
      const int g = s.y > 0 ? group_of(b) : -1;
      const int n = g >= 0 ? group_tiles(g) : 0;
      const int2 r = n ? group_rows(g) : make_int2(0, 0);
      if (n && (s.x < r.x || s.x + s.y > r.x + r.y)) {
        s.y = s.z = 0;  // (cu_q falls) rows that the group's tiles do not have: zeros
      } else if (n) {
        shared = shared_of(g);
        q.p_unit = kLds ? s_gunit[g] : p.group_shared[2 * p.groups + g];
        q.p_parts = sh_ceil(shared / kTileN, most);
        q.p_step = sh_units(p, r.y, n);
        q.p_q0 = r.x;
      }
    }
    if (!p.cu_q) {
      const int tokens = max(0, s.z - shared);
      const int parts = sh_ceil(tokens, chunk), size = parts ? (sh_ceil(tokens, parts) + 15) & ~15 : 0;
      const Sh3 at = sh_scan({0, 0, parts}, s_wave, sum);
      const int first = base.c + at.c;
      q.s_unit = first;
      q.s_parts = parts;
      const bool whole = parts == 1 && q.p_parts == 0;
      q.s_step = whole;
      // the longest first, by the tokens of a sequence's parts
      const int bin = kShBins - 1 - min(size / 16, kShBins - 1);
      if (parts) atomicAdd(&s_bins[bin], parts);
      __syncthreads();
      if (wave == 0) {  // ranks before each bin
        int run = base.c;
        for (int i = 0; i < kShBins; i += 64) {
          const int have = s_bins[i + lane], upto = (int)wave_scan((uint32_t)have);
          s_bins[i + lane] = run + upto - have;
          run += __builtin_amdgcn_readlane(upto, 63);
        }
      }
      __syncthreads();
      const int rank = parts ? atomicAdd(&s_bins[bin], parts) : 0;
      for (int k = 0; k < parts && rank + k < p.cap_chunks; ++k)
        p.chunks[rank + k] = ShChunk{b, shared + k * size, min(shared + (k + 1) * size, s.z),
                                     (int)((uint32_t)(first + k) | (whole ? 0x80000000u : 0u))};
      __syncthreads();
      for (int i = tid; i < kShBins; i += threads) s_bins[i] = 0;
      __syncthreads();
    } else {
      const int n = s.y > 0 ? sh_row_tiles(p, s.y) : 0;
      const int parts = n ? sh_ceil(own_tiles(b, s, shared, n - 1), most) : 0;
      const int step = n ? sh_units(p, s.y, n) : 0;
      const Sh3 at = sh_scan({n * parts, n * parts * step, 0}, s_wave, sum);
      const int first = base.a + at.a, unit = base.b + at.b;
      q.s_unit = unit * hkv;
      q.s_parts = parts;
      q.s_step = step;
      q.s_q0 = s.x;
      const int lo = shared / kTileN;
      for (int i = 0; i < n * parts && first + i < p.cap_tiles; ++i) {
        const int k = i / n, t = i - k * n;
        const int kv = own_tiles(b, s, shared, t);
        p.tiles[first + i] = ShTile{b, t, s.x, s.y, s.z, lo + sh_cut(kv, k, parts), lo + sh_cut(kv, k + 1, parts),
                                    (unit + (t * parts + k) * step) * hkv, step, {0, 0, 0}};
      }
    }
    if (b < p.batch) p.seqs[b] = q;
    base = {base.a + sum.a, base.b + sum.b, base.c + sum.c};
  }
  const bool fits = base.a <= p.cap_tiles && base.c <= p.cap_chunks && (long long)base.b * hkv <= p.cap_units;
  if (fits) {
    if (tid == 0) {
      p.header[0] = base.a;
      p.header[1] = base.c;
    }
  } else {
    __syncthreads();  // the entries of all sequences have been written
    run_nothing();
  }
}

// Parts of 256-row tiles: workgroup = (part, kv head).  64 questions of 20 to 100
// tokens about 32 768 shared ones, 32 / 8 heads: 1.1 PFLOP/s; with q rounded once
// more, scale included, as the plain prefill has it, 6 % less time and an error of
// 0.29 % of the output's norm in place of 0.23 %.
template <bool kSoftCap, int kPaging>
__global__ void __launch_bounds__(kThreads, 1)
shared_tile_kernel(SharedParams p) {
  const int hkv = p.num_kv_heads;
  const int rank = blockIdx.x / hkv, kvh = blockIdx.x - rank * hkv;
  const __attribute__((address_space(4))) int32_t* hd = (const __attribute__((address_space(4))) int32_t*)p.header;
  const __attribute__((address_space(4))) int32_t* e =
      (const __attribute__((address_space(4))) int32_t*)(p.tiles + rank);
  if (rank >= hd[0]) return;  // uniform over the workgroup; the list has room for every rank of the grid
  PrefillWork w;
  w.b = e[0];
  w.qt = e[1];
  w.q0 = e[2];
  w.lq_rows = e[3];
  w.lk = e[4];
  w.kvh = kvh;
  w.kv_pos_off = p.cu_q ? 0 : 1;  // positions: kv indices, or (one token each) the lengths
  PrefillPart part;
  part.lo = e[5];
  part.hi = e[6];
  part.slot = e[7] + kvh * e[8];
  prefill_run<kSoftCap, kPaging, kPHeadDim, true, true>(p.pre, w, part);
}

// The chunk of a rank, for the kv head and block of 16 q heads vh.
template <bool kAligned, bool kSoftCap, bool kShared>
__device__ __forceinline__ void shared_chunk(const SharedParams& p, int rank, int vh, DecodeLds& red) {
  const ShChunk c = p.chunks[rank];
  DecodeWork w;
  w.b = __builtin_amdgcn_readfirstlane(c.b);
  w.vh = vh;
  w.t_begin = __builtin_amdgcn_readfirstlane(c.t0);
  w.t_end = __builtin_amdgcn_readfirstlane(c.t1);
  w.len = w.t_end;
  const int slot = __builtin_amdgcn_readfirstlane(c.slot);
  w.single = slot < 0;
  w.part = (int64_t)(slot & 0x7fffffff) * p.num_kv_heads + vh / p.dec.hblocks;
  decode_run<kDecodeWaves, kAligned, kSoftCap, false, kShared>(p.dec, w, &red.o[0][0][0], &red.m[0][0], &red.l[0][0]);
}

// Parts of 128-row tiles (the first tile_ranks ranks of all kv heads), then
// chunks of sequences' own tokens, one new token a sequence.  The tiles are bound
// by the matrix cores and the chunks by their reads, and a CU has one of each.
template <bool kSoftCap, bool kShared>
__global__ void __launch_bounds__(64 * kDecodeWaves, 2)
shared_part_kernel(SharedParams p, int tile_blocks) {
  __shared__ __attribute__((aligned(1024))) char lds[kLtLdsB];
  static_assert(sizeof(DecodeLds) <= kLtLdsB, "a chunk's combine fits the ring");
  const __attribute__((address_space(4))) int32_t* hd = (const __attribute__((address_space(4))) int32_t*)p.header;
  const int hkv = p.num_kv_heads;
  if ((int)blockIdx.x < tile_blocks) {
    const int rank = blockIdx.x / hkv, kvh = blockIdx.x - rank * hkv;
    if (rank >= hd[0]) return;  // uniform over the workgroup, as below
    const __attribute__((address_space(4))) int32_t* e =
        (const __attribute__((address_space(4))) int32_t*)(p.tiles + rank);
    LtParams a;
    a.q = p.pre.q;
    a.q_ts = p.pre.q_ts;
    a.q_hs = p.pre.q_hs;
    a.k = p.pre.k_cache;
    a.v = p.pre.v_cache;
    a.num_pages = p.pre.num_pages;
    a.page_size = p.pre.page_size;
    a.page_stride = p.pre.page_stride;
    a.slot_stride = p.pre.slot_stride;
    a.head_stride = p.pre.head_stride;
    a.pages_per_seq = p.pre.pages_per_seq;
    a.group = p.group;
    a.logit_scale = p.pre.logit_scale;
    a.soft_cap = p.pre.soft_cap;
    a.parts = p.pre.parts;
    const int row0 = e[1] * kLtRows, q0 = e[2], rows = e[3] * p.group;
    const int t0 = e[5] * kTileN, t1 = min(e[6] * kTileN, e[4]);
    const int r = min(row0 + (int)(threadIdx.x >> 6) * 32 + (int)(threadIdx.x & 31), rows - 1);
    const int token = q0 + r / p.group;
    const int limit = p.cu_q ? p.positions[token] + 1 : clamp_len(p.lengths, token, p.span);
    lt_run<kSoftCap>(a, p.pre.block_tables + (int64_t)e[0] * p.pre.bt_stride, kvh, q0, rows, row0, t0, t1, limit,
                     e[7] + kvh * e[8], (uint32_t)(uintptr_t)(lds_void)&lds[0]);
    return;
  }
  const int vheads = hkv * p.dec.hblocks;
  const int bid = blockIdx.x - tile_blocks, step = (gridDim.x - tile_blocks) / vheads;
  const int first = bid / vheads, vh = bid - first * vheads;
  for (int rank = first; rank < hd[1]; rank += step) {
    if (rank != first) __syncthreads();  // the last chunk's combine has been read
    shared_chunk<true, kSoftCap, kShared>(p, rank, vh, *reinterpret_cast<DecodeLds*>(&lds[0]));
  }
}

// The chunks alone, over pages that are not of whole 16-token steps.
template <bool kSoftCap, bool kShared>
__global__ void __launch_bounds__(64 * kDecodeWaves, 2)
shared_chunk_kernel(SharedParams p) {
  __shared__ DecodeLds red;
  const int vheads = p.num_kv_heads * p.dec.hblocks;
  const int first = blockIdx.x / vheads;
  for (int rank = first; rank < p.header[1]; rank += gridDim.x / vheads) {
    if (rank != first) __syncthreads();
    shared_chunk<false, kSoftCap, kShared>(p, rank, blockIdx.x - first * vheads, red);
  }
}

// One workgroup a (32 rows, kv head), 4 kTeams waves: a wave has 32 d (a lane row n,
// d = 32 dt + 8 q4 + 4 h .. + 4, as the tiles' accumulators) of every kTeams'th
// part; the teams meet in LDS.  Launches of few rows have many parts a row and
// take four teams (57 parts of two sequences' 32k shared tokens: 74 -> 49 us the call).
template <int kTeams>
__global__ void __launch_bounds__(256 * kTeams)
shared_merge_kernel(SharedParams p) {
  const int hkv = p.num_kv_heads;
  const int block = blockIdx.x / hkv, kvh = blockIdx.x - block * hkv;
  const int lane = threadIdx.x & 63, dt = threadIdx.x >> 6 & 3;
  const int team = kTeams == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
  const int n = lane & 31, h = lane >> 5;
  const int64_t row = (int64_t)32 * block + n;
  const int token = (int)min(row / p.group, (int64_t)p.num_tokens - 1), head = (int)(row - row / p.group * p.group);
  const bool is = row < (int64_t)p.num_tokens * p.group;
  const int b = p.cu_q ? p.owner[token] : token;
  f32x4 o[4] = {};
  float m_run = -INFINITY, lsum = 0.f;
  auto add = [&](const float* po, int stride, float m, float l) __attribute__((always_inline)) {
    const float m_new = fmaxf(m_run, m);
    const float ms = m_new == -INFINITY ? 0.f : m_new;
    const float old = fast_exp2(m_run - ms), wgt = fast_exp2(m - ms);
    m_run = m_new;
    lsum = lsum * old + l * wgt;
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4)
      o[q4] = o[q4] * old + *reinterpret_cast<const f32x4*>(po + stride * q4) * wgt;
  };
  auto add_tiles = [&](int unit, int parts, int step, int q0) __attribute__((always_inline)) {
    const int at = token - q0;
    int t, r;  // row tile, row of it
    if (p.light) {
      r = at * p.group + head;
      t = r / kLtRows;
      r -= t * kLtRows;
    } else {
      t = at / p.tile_tokens;
      r = (at - t * p.tile_tokens) * p.group + head;
    }
    const float* src = p.pre.parts + ((int64_t)unit + ((int64_t)t * parts * hkv + kvh) * step + (r >> 5)) * kLtUnit;
    const float* po = src + 4 * (dt * 4 * 64 + 32 * h + (r & 31));
    const float* ml = src + 32 * kHeadDim + 2 * (r & 31);
    const int64_t next = (int64_t)hkv * step * kLtUnit;
#pragma unroll 4
    for (int k = team; k < parts; k += kTeams) {
      const f32x2 v = *reinterpret_cast<const f32x2*>(ml + k * next);
      add(po + k * next, 256, v[0], v[1]);
    }
  };
  bool done = !is || (b < 0 && !p.zero_rest);
  if (!done && b >= 0) {
    const ShSeq s = p.seqs[b];
    done = !p.cu_q && s.s_step;  // its one part wrote the row
    if (!done) {
      if (s.p_parts) add_tiles(s.p_unit, s.p_parts, s.p_step, s.p_q0);
      if (p.cu_q) {
        if (s.s_parts) add_tiles(s.s_unit, s.s_parts, s.s_step, s.s_q0);
      } else {
#pragma unroll 2
        for (int k = team; k < s.s_parts; k += kTeams) {
          const int64_t at = ((int64_t)(s.s_unit + k) * hkv + kvh) * p.group + head;
          const f32x2 v = *reinterpret_cast<const f32x2*>(p.dec.ws_ml + 2 * at);
          add(p.dec.ws_o + at * kHeadDim + 32 * dt + 4 * h, 8, v[0], v[1]);
        }
      }
    }
  }
  if constexpr (kTeams > 1) {
    __shared__ __attribute__((aligned(16))) float s_o[kTeams - 1][4][4][64][4];
    __shared__ float s_ml[kTeams - 1][4][64][2];
    if (team) {
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) *reinterpret_cast<f32x4*>(s_o[team - 1][dt][q4][lane]) = o[q4];
      s_ml[team - 1][dt][lane][0] = m_run;
      s_ml[team - 1][dt][lane][1] = lsum;
    }
    __syncthreads();
    if (team) return;
#pragma unroll
    for (int k = 0; k + 1 < kTeams; ++k) add(s_o[k][dt][0][lane], 256, s_ml[k][dt][lane][0], s_ml[k][dt][lane][1]);
  }
  if (done) return;
  const float inv = lsum > 0.f ? 1.f / lsum : 0.f;  // rows that see no key are zeros
  uint16_t* dst = p.pre.out + (int64_t)token * p.pre.o_ts + (int64_t)(kvh * p.group + head) * p.pre.o_hs + 32 * dt +
                  4 * h;
#pragma unroll
  for (int q4 = 0; q4 < 4; ++q4)
    *reinterpret_cast<u32x2*>(dst + 8 * q4) =
        u32x2{pack_bf16x2(o[q4][0] * inv, o[q4][1] * inv), pack_bf16x2(o[q4][2] * inv, o[q4][3] * inv)};
}
static_assert(kPartFloats<kPHeadDim> == kLtUnit, "both kinds of tiles leave partials of one layout");

// Whether a launch takes 128-row tiles that share a CU: pages of whole 16-token steps,
// and one new token a sequence or fewer than 256 rows of one.  Calls in a graph, 128-row
// tiles then 256-row tiles, 32 / 8 heads, pages of 64.  One new token: 128 sequences of
// 64 to 1024 own tokens behind 8192 shared ones 87 and 129 us (the chunks have a launch
// of their own beside 256-row tiles), 256 behind 32768 255 and 320; with hardly any own
// tokens the tiles alone count: 128 behind 2048 36 and 42, behind 32768 110 and 98.
// Several: 32 sequences by 2 behind 8192 38 and 41, by 5 55 and 54, by 20 145 and 113,
// by 60 329 and 283, by 64 (256 rows) 334 and 283, by 200 1085 and 927; 64 by 5 behind
// 32768 288 and 192.  So below 256 rows of a sequence the rule gives up to a third away
// where the groups are large.
bool shared_light(bool ragged, int64_t max_q, int64_t group, int64_t page) {
  if (page % 16) return false;
  return !ragged || max_q * group < kRows;
}

// What a launch of a shape needs: entries of the lists and bytes of the workspace.
struct ShSizes {
  bool light;
  int64_t tiles, units, chunks;
  int32_t chunk_cap;
  size_t header, groups, seqs, list, chunk_list, positions, owner, parts, dec_o, dec_ml, bytes;
};
size_t sh_up(size_t x) { return (x + 255) & ~(size_t)255; }

ShSizes shared_sizes(int64_t batch, int64_t groups, int64_t tokens, int64_t max_q, bool ragged, int64_t heads,
                     int64_t hkv, int64_t pages, int64_t page) {
  ShSizes z = {};
  const int64_t group = heads / hkv;
  z.light = shared_light(ragged, max_q, group, page);
  const int64_t most = z.light ? kLtWaves : kWaves;  // units of a row tile
  const int64_t slots = z.light ? kShPartSlots : kShTileSlots;
  const int64_t span = pages * page;
  // row tiles of groups, and of sequences: a range of n tokens rounds up once
  auto row_tiles = [&](int64_t ranges) {
    const int64_t whole = z.light ? tokens * group / kLtRows : tokens / (kRows / group);
    return std::min(ranges, tokens) + whole;
  };
  const int64_t prefix = groups ? row_tiles(groups) : 0, mine = ragged ? row_tiles(batch) : 0;
  // units of a sequence's row tile: of those of one tile what its rows take
  const int64_t rows = std::min(max_q, tokens) * group;
  const int64_t step = std::min(most, (rows + 31) / 32);
  // parts of a share of the slots: one a row tile and `extra` more
  const int64_t extra = slots / hkv + 1;
  z.tiles = prefix + mine ? prefix + mine + extra : 0;
  z.units = hkv * (most * (prefix + extra) + step * mine);
  z.chunk_cap = (int32_t)std::max<int64_t>(16, std::min<int64_t>(2048, 62 * page) & ~(int64_t)15);
  if (!ragged) {
    const int64_t least = std::min<int64_t>(kShMinChunk, z.chunk_cap);
    const int64_t per = (span + z.chunk_cap - 1) / z.chunk_cap;  // of the longest sequence at the longest chunk
    z.chunks = std::min(batch * ((span + least - 1) / least),
                        batch + std::max(kShPartSlots / hkv + 1, batch * per));
  }
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t r = at;
    at += sh_up(bytes);
    return r;
  };
  z.header = take(kShHeader * sizeof(int32_t));
  z.groups = take(3 * groups * sizeof(int32_t));
  z.seqs = take(batch * sizeof(ShSeq));
  z.list = take(z.tiles * sizeof(ShTile));
  z.chunk_list = take((z.chunks + 8) * sizeof(ShChunk));
  z.positions = take(ragged ? tokens * sizeof(int32_t) : 0);
  z.owner = take(ragged ? tokens * sizeof(int32_t) : 0);
  z.parts = take(z.tiles ? (size_t)z.units * kLtUnit * sizeof(float) : 0);
  z.dec_o = take((size_t)z.chunks * heads * kHeadDim * sizeof(float));
  z.dec_ml = take((size_t)z.chunks * heads * 2 * sizeof(float));
  z.bytes = at;
  return z;
}

}  // namespace
}  // namespace pa

using namespace pa;

extern "C" size_t pa_shared_prefix_workspace_size(int32_t batch, int32_t num_groups, int32_t num_tokens,
                                                  int32_t max_seqlen_q, int32_t ragged, int32_t num_heads,
                                                  int32_t num_kv_heads, int32_t pages_per_seq, int32_t page_size) {
  if (batch <= 0 || num_groups < 0 || num_tokens <= 0 || max_seqlen_q <= 0 || num_heads <= 0 || num_kv_heads <= 0 ||
      num_heads % num_kv_heads || num_heads / num_kv_heads > kRows || pages_per_seq < 0 || page_size <= 0)
    return 0;
  return shared_sizes(batch, num_groups, num_tokens, max_seqlen_q, ragged != 0, num_heads, num_kv_heads,
                      pages_per_seq, page_size).bytes;
}

extern "C" int pa_shared_prefix(const uint16_t* q, int64_t q_tok_stride, int64_t q_head_stride,
                                const uint16_t* k_cache, const uint16_t* v_cache, int32_t num_pages,
                                int32_t page_size, int64_t page_stride, int64_t slot_stride, int64_t head_stride,
                                const int32_t* block_tables, int64_t bt_stride, int32_t pages_per_seq,
                                const int32_t* lengths, const int32_t* cu_groups, const int32_t* shared_lens,
                                int32_t num_groups, const int32_t* cu_seqlens_q, int32_t batch, int32_t num_tokens,
                                int32_t max_seqlen_q, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                                float scale, float soft_cap, int32_t zero_rest, uint16_t* out,
                                int64_t out_tok_stride, int64_t out_head_stride, void* workspace,
                                size_t workspace_bytes, void* stream) {
  const char* name = "pa_shared_prefix";
  if (num_pages <= 0 || page_size <= 0 || batch < 0 || num_groups < 0 || num_tokens < 0 || max_seqlen_q < 0 ||
      num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads || pages_per_seq < 0)
    return fail(PA_ERR_INVALID_ARGUMENT, "%s: bad sizes (num_pages=%d, page_size=%d, batch=%d, num_groups=%d, "
                "num_tokens=%d, max_seqlen_q=%d, num_heads=%d, num_kv_heads=%d, pages_per_seq=%d)", name, num_pages,
                page_size, batch, num_groups, num_tokens, max_seqlen_q, num_heads, num_kv_heads, pages_per_seq);
  if (!cu_seqlens_q && num_tokens != batch)
    return fail(PA_ERR_INVALID_ARGUMENT, "%s: %d tokens of %d sequences without cu_seqlens_q", name, num_tokens,
                batch);
  if (head_dim != kPHeadDim) return fail(PA_ERR_UNSUPPORTED, "%s: head_dim %d not supported (128)", name, head_dim);
  const int group = num_heads / num_kv_heads;
  if (group > kRows) return fail(PA_ERR_UNSUPPORTED, "%s: %d q heads a kv head (%d at most)", name, group, kRows);
  if (num_kv_heads > (1 << 16)) return fail(PA_ERR_UNSUPPORTED, "%s: %d kv heads", name, num_kv_heads);
  if ((int64_t)pages_per_seq * page_size > 0x7fffffff - 4096)
    return fail(PA_ERR_UNSUPPORTED, "%s: block tables of %d pages span 2^31 tokens or more", name, pages_per_seq);
  if (!prefill_offsets_fit(slot_stride))
    return fail(PA_ERR_UNSUPPORTED, "%s: slot stride %lld", name, (long long)slot_stride);
  if (num_tokens == 0) return PA_OK;
  if (batch == 0 || pages_per_seq == 0 || max_seqlen_q == 0)
    return fail(PA_ERR_INVALID_ARGUMENT, "%s: %d tokens of %d sequences (%d pages, %d new tokens at most)", name,
                num_tokens, batch, pages_per_seq, max_seqlen_q);
  if (!q || !k_cache || !v_cache || !out || !lengths || !block_tables ||
      (num_groups && (!cu_groups || !shared_lens)))
    return fail(PA_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
  if ((((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out) & 15u) ||
      ((uintptr_t)workspace & 255u) ||
      (q_tok_stride | q_head_stride | page_stride | slot_stride | head_stride | out_tok_stride | out_head_stride) % 8)
    return fail(PA_ERR_UNSUPPORTED, "%s: operands must be 16-byte aligned with strides multiple of 8, the workspace "
                "256-byte aligned", name);
  const bool ragged = cu_seqlens_q != nullptr;
  const ShSizes z = shared_sizes(batch, num_groups, num_tokens, max_seqlen_q, ragged, num_heads, num_kv_heads,
                                 pages_per_seq, page_size);
  if (z.units > 0x7fffffff || z.chunks * num_heads > 0x7fffffff)
    return fail(PA_ERR_UNSUPPORTED, "%s: %d tokens of %d sequences need %zu bytes of partials", name, num_tokens, batch,
                z.bytes);
  if (!workspace || workspace_bytes < z.bytes)
    return fail(PA_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", name, workspace_bytes, z.bytes);
  char* ws = (char*)workspace;
  SharedParams p = {};
  p.cu_q = cu_seqlens_q;
  p.lengths = lengths;
  p.cu_groups = cu_groups;
  p.shared_lens = shared_lens;
  p.batch = batch;
  p.groups = num_groups;
  p.num_tokens = num_tokens;
  p.num_kv_heads = num_kv_heads;
  p.group = group;
  p.light = z.light;
  p.tile_tokens = kRows / group;
  p.span = pages_per_seq * page_size;
  p.max_seqlen_q = max_seqlen_q;
  p.chunk_cap = z.chunk_cap;
  p.zero_rest = zero_rest;
  p.cap_tiles = (int32_t)z.tiles;
  p.cap_chunks = (int32_t)z.chunks;
  p.cap_units = (int32_t)z.units;
  p.header = (int32_t*)(ws + z.header);
  p.group_shared = (int32_t*)(ws + z.groups);
  p.seqs = (ShSeq*)(ws + z.seqs);
  p.tiles = (ShTile*)(ws + z.list);
  p.chunks = (ShChunk*)(ws + z.chunk_list);
  p.positions = (int32_t*)(ws + z.positions);
  p.owner = (int32_t*)(ws + z.owner);
  PrefillParams& a = p.pre;
  a.q = q;
  a.q_ts = q_tok_stride;
  a.q_hs = q_head_stride;
  a.k_cache = k_cache;
  a.v_cache = v_cache;
  a.num_pages = num_pages;
  a.page_size = page_size;
  a.page_stride = page_stride;
  a.slot_stride = slot_stride;
  a.head_stride = head_stride;
  a.block_tables = block_tables;
  a.bt_stride = bt_stride;
  a.pages_per_seq = pages_per_seq;
  a.positions = ragged ? p.positions : lengths;
  a.num_tokens = num_tokens;
  a.num_heads = num_heads;
  a.num_kv_heads = num_kv_heads;
  a.group = group;
  a.tile_tokens = p.tile_tokens;
  a.logit_scale = soft_cap > 0.f ? scale : scale * kLog2e;
  a.soft_cap = soft_cap;
  a.out = out;
  a.o_ts = out_tok_stride;
  a.o_hs = out_head_stride;
  a.parts = (float*)(ws + z.parts);
  DecodeParams& d = p.dec;
  d.q = q;
  d.q_bs = q_tok_stride;
  d.q_hs = q_head_stride;
  d.k_cache = k_cache;
  d.v_cache = v_cache;
  d.num_pages = num_pages;
  d.page_size = page_size;
  d.page_stride = page_stride;
  d.slot_stride = slot_stride;
  d.head_stride = head_stride;
  d.block_tables = block_tables;
  d.bt_stride = bt_stride;
  d.pages_per_seq = pages_per_seq;
  d.lengths = lengths;
  d.batch = batch;
  d.num_heads = num_heads;
  d.num_kv_heads = num_kv_heads;
  d.group = group;
  d.hblocks = (group + 15) / 16;
  d.logit_scale = a.logit_scale;
  d.soft_cap = soft_cap;
  d.ws_o = (float*)(ws + z.dec_o);
  d.ws_ml = (float*)(ws + z.dec_ml);
  d.out = out;
  d.out_bs = out_tok_stride;
  d.out_hs = out_head_stride;
  hipStream_t s = (hipStream_t)stream;
  const bool cap = soft_cap > 0.f;
  const int64_t merges = ((int64_t)num_tokens * group + 31) / 32 * num_kv_heads;
  if (z.tiles * num_kv_heads > kMaxGrid || z.chunks * num_kv_heads * d.hblocks > 2 * kMaxGrid || merges > 4 * kMaxGrid)
    return fail(PA_ERR_UNSUPPORTED, "%s: %lld parts of %lld rows", name, (long long)(z.tiles + z.chunks),
                (long long)merges * 32);
  const bool small = batch <= 256 && num_groups <= 256;  // (short barriers where few threads do)
  const int threads = small ? 256 : kShPlanThreads;
  const int64_t maps = ragged ? (num_tokens + threads - 1) / threads : 0;
  const bool fits = batch <= kShPlanMax && num_groups <= kShPlanMax;
  auto plan = fits ? shared_plan_kernel<true> : shared_plan_kernel<false>;
  plan<<<dim3((unsigned)(1 + maps)), dim3(threads), 0, s>>>(p);
  if (int rc = launch_status(name)) return rc;
  const int64_t tile_blocks = z.tiles * num_kv_heads;
  // ranks that have a workgroup (further ones come behind in their loops): where
  // the chunk is a share of the slots there are no more
  const int64_t ranks = std::min<int64_t>(z.chunks, ((batch + kShPartSlots / (num_kv_heads * d.hblocks) + 1) + 7) / 8 * 8);
  auto by_flags = [&](auto launch) {
    if (cap && d.hblocks > 1) launch(std::true_type{}, std::true_type{});
    else if (cap) launch(std::true_type{}, std::false_type{});
    else if (d.hblocks > 1) launch(std::false_type{}, std::true_type{});
    else launch(std::false_type{}, std::false_type{});
    return launch_status(name);
  };
  const dim3 small_blk(64 * kDecodeWaves);
  if (z.light) {
    const int64_t chunk_blocks = ranks * num_kv_heads * d.hblocks;
    const int rc = by_flags([&](auto c, auto sh) {
      shared_part_kernel<decltype(c)::value, decltype(sh)::value>
          <<<dim3((unsigned)(tile_blocks + chunk_blocks)), small_blk, 0, s>>>(p, (int)tile_blocks);
    });
    if (rc) return rc;
  } else {
    if (tile_blocks) {
      const dim3 grid((unsigned)tile_blocks), blk(kThreads);
      auto launch = [&](auto c) {
        constexpr bool kCap = decltype(c)::value;
        const int paging = prefill_paging(page_size, slot_stride);
        if (paging == kPageTile) shared_tile_kernel<kCap, kPageTile><<<grid, blk, 0, s>>>(p);
        else if (paging == kPageWave) shared_tile_kernel<kCap, kPageWave><<<grid, blk, 0, s>>>(p);
        else shared_tile_kernel<kCap, kPageLane><<<grid, blk, 0, s>>>(p);
      };
      if (cap) launch(std::true_type{});
      else launch(std::false_type{});
      if (int rc = launch_status(name)) return rc;
    }
    if (!ragged) {
      const int rc = by_flags([&](auto c, auto sh) {
        shared_chunk_kernel<decltype(c)::value, decltype(sh)::value>
            <<<dim3((unsigned)(ranks * num_kv_heads * d.hblocks)), small_blk, 0, s>>>(p);
      });
      if (rc) return rc;
    }
  }
  if (merges <= kShMergeFew) shared_merge_kernel<4><<<dim3((unsigned)merges), dim3(1024), 0, s>>>(p);
  else shared_merge_kernel<1><<<dim3((unsigned)merges), dim3(256), 0, s>>>(p);
  return launch_status(name);
}
