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
//   shared_tile_kernel    prefill_run's loop over one part of a prefix (256 rows
//                         against 64-token tiles), and, where sequences have
//                         several new tokens, over their own part too
//   shared_decode_kernel  decode_run over a sequence's own part, where each has
//                         one new token
//   shared_merge_kernel   adds the parts up
#include <algorithm>
#include <type_traits>

#include "../../include/long_context.h"
#include "decode_impl.h"
#include "long_context.h"
#include "prefill_impl.h"

namespace pa {
namespace {

constexpr int kShPlanThreads = 1024;
constexpr int kShPlanWaves = kShPlanThreads / 64;
constexpr int kShTileSlots = 256;    // tile workgroups resident at once (one a CU)
constexpr int kShDecodeSlots = 512;  // decode workgroups resident at once (two a CU)
constexpr int kShMinTiles = 8;       // shortest part of a tile item
constexpr int kShMinChunk = 512;     // shortest part of a decode item, tokens

// One part of a (row range, q tile) pair; every kv head has it.
struct alignas(16) ShTile {
  int32_t table, qt, q0, rows;    // block-table row, q tile, first token, tokens
  int32_t lk, lo, hi, unit;       // kv length, kv tiles [lo, hi), first unit of kv head 0
  int32_t step, pad[3];           // units a kv head
};
// One part of a sequence's own tokens.
struct alignas(16) ShChunk {
  int32_t b, t0, t1, slot;  // slot: part number, bit 31: the whole row
};
// Where the rows of a sequence find their parts.
struct alignas(16) ShSeq {
  int32_t p_unit, p_parts, p_step, p_q0;  // prefix: first unit, parts, units a kv head, first token of the group
  int32_t s_unit, s_parts, s_step, s_q0;  // own part likewise (decode: first slot)
};
struct alignas(16) ShGroup {
  int32_t shared, table, q0, tokens;  // shared tokens (whole tiles), table row, first token, tokens
};
constexpr int kShHeader = 64;  // ints: number of tile parts, of chunks

struct SharedParams {
  PrefillParams pre;
  DecodeParams dec;
  const int32_t* cu_q;  // null: one new token a sequence
  const int32_t* lengths;
  const int32_t* cu_groups;
  const int32_t* shared_lens;
  int32_t batch, groups, num_tokens, num_kv_heads, group, tile_tokens, span, max_seqlen_q;
  int32_t chunk_cap, zero_rest;
  int32_t cap_tiles, cap_chunks, cap_units;  // what the workspace holds
  int32_t* header;
  ShGroup* group_info;
  ShSeq* seqs;
  ShTile* tiles;
  ShChunk* chunks;
  int32_t* positions;  // [num_tokens] kv index of each token (with cu_q)
  int32_t* owner;      // [num_tokens] its sequence, or -1 (with cu_q)
};

// Sequence b: first token, new tokens, tokens in all.
__device__ __forceinline__ int3 sh_sequence(const SharedParams& p, int b) {
  const int len = clamp_len(p.lengths, b, p.span);
  if (!p.cu_q) return make_int3(b, len > 0 ? 1 : 0, len);
  const int q0 = p.cu_q[b];
  int n = p.cu_q[b + 1] - q0;
  n = q0 < 0 || q0 >= p.num_tokens ? 0 : min(min(n, p.max_seqlen_q), p.num_tokens - q0);
  return make_int3(q0, max(n, 0), len);
}

// Exclusive scan over the workgroup of one number a thread; `total`: their sum.
__device__ __forceinline__ int sh_scan(int v, int* s_wave, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int upto = (int)wave_scan((uint32_t)v);
  __syncthreads();  // the last scan's sums have been read
  if (lane == 63) s_wave[wave] = upto;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < kShPlanWaves; ++i) {
    before += i < wave ? s_wave[i] : 0;
    total += s_wave[i];
  }
  return before + upto - v;
}
__device__ __forceinline__ long long sh_sum(long long v, long long* s_wave) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if (lane == 0) s_wave[wave] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int i = 0; i < kShPlanWaves; ++i) v += s_wave[i];
  return v;
}

__device__ __forceinline__ int sh_ceil(int a, int b) { return (a + b - 1) / b; }

// Workgroup 0 plans; the others (with cu_q) map tokens to sequences and kv
// positions, a token a thread.
__global__ void __launch_bounds__(kShPlanThreads)
shared_plan_kernel(SharedParams p) {
  const int tid = threadIdx.x;
  if (blockIdx.x > 0) {
    const int t = (blockIdx.x - 1) * kShPlanThreads + tid;
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
  __shared__ int s_wave[kShPlanWaves];
  __shared__ long long s_long[kShPlanWaves];
  const int lane = tid & 63, wave = tid >> 6;
  const int hkv = p.num_kv_heads;
  // ---- groups: a wave each
  for (int g = wave; g < p.groups; g += kShPlanWaves) {
    const int g0 = max(0, p.cu_groups[g]), g1 = min(p.batch, p.cu_groups[g + 1]);
    int active = 0, least = INT_MAX, first = INT_MAX;
    for (int b = g0 + lane; b < g1; b += 64) {
      const int3 s = sh_sequence(p, b);
      if (s.y > 0 && s.z > 0) {
        ++active;
        least = min(least, s.z);
        first = min(first, b);
      }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      active += __shfl_xor(active, o);
      least = min(least, __shfl_xor(least, o));
      first = min(first, __shfl_xor(first, o));
    }
    if (lane == 0) {
      ShGroup r = {0, 0, 0, 0};
      if (active > 1) {
        r.table = first;
        r.q0 = p.cu_q ? p.cu_q[g0] : g0;
        r.tokens = (p.cu_q ? p.cu_q[g1] : g1) - r.q0;
        // whole tiles, and no further than the shortest sequence
        r.shared = min(p.shared_lens[g], least) & ~(kTileN - 1);
        if (r.shared <= 0 || r.q0 < 0 || r.tokens <= 0 || r.tokens > p.num_tokens - r.q0) r = {0, 0, 0, 0};
      }
      p.group_info[g] = r;
    }
  }
  __syncthreads();
  auto group_pairs = [&](const ShGroup& r) { return r.shared ? sh_ceil(r.tokens, p.tile_tokens) : 0; };
  auto group_of = [&](int b) {
    int lo = 0, hi = p.groups;  // last g with cu_groups[g] <= b
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (p.cu_groups[mid] <= b) lo = mid;
      else hi = mid;
    }
    return p.groups > 0 && p.cu_groups[lo] <= b && b < p.cu_groups[lo + 1] ? lo : -1;
  };
  // kv tiles of q tile qt of sequence s behind `shared` tokens
  auto own_tiles = [&](const int3& s, int full, int shared, int qt) {
    const int hi = min(s.z, s.z - full + min((qt + 1) * p.tile_tokens, s.y));
    return hi <= shared ? 0 : sh_ceil(hi, kTileN) - shared / kTileN;
  };
  // ---- work in all
  long long tiles = 0, pairs = 0, own = 0;
  for (int g = tid; g < p.groups; g += kShPlanThreads) {
    const ShGroup r = p.group_info[g];
    const int n = group_pairs(r);
    pairs += n;
    tiles += (long long)n * (r.shared / kTileN);
  }
  for (int b = tid; b < p.batch; b += kShPlanThreads) {
    const int3 s = sh_sequence(p, b);
    const int g = group_of(b);
    const int shared = g >= 0 ? p.group_info[g].shared : 0;
    if (!p.cu_q) {
      own += max(0, s.z - shared);
    } else {
      const int full = p.cu_q[b + 1] - s.x, n = sh_ceil(s.y, p.tile_tokens);
      pairs += n;
      if (n) tiles += (long long)n * own_tiles(s, full, shared, n - 1);  // (its q tiles are cut alike)
    }
  }
  tiles = sh_sum(tiles, s_long);
  pairs = sh_sum(pairs, s_long);
  own = sh_sum(own, s_long);
  // Parts of at most `most` tiles: every pair rounds up, so where there are few
  // pairs an even share of the slots that they leave over makes one round;
  // else a share of all.
  const int slots = kShTileSlots / hkv;
  const long long left = slots - pairs;
  const long long share = (2 * left >= slots && left > 0) ? (tiles + left - 1) / left : (tiles + slots - 1) / max(1, slots);
  const int most = (int)max((long long)kShMinTiles, share);
  const long long chunk_share = (own * hkv * p.dec.hblocks + kShDecodeSlots - 1) / kShDecodeSlots;
  const int chunk = min(p.chunk_cap, max(kShMinChunk, (int)min(chunk_share, (long long)INT_MAX - 16) + 15 & ~15));
  // ---- the lists
  int n_tiles = 0, n_units = 0;  // before this round (units of one kv head)
  for (int g0 = 0; g0 < p.groups; g0 += kShPlanThreads) {
    const int g = g0 + tid;
    ShGroup r = {0, 0, 0, 0};
    if (g < p.groups) r = p.group_info[g];
    const int n = group_pairs(r), kv = r.shared / kTileN;
    const int parts = n ? sh_ceil(kv, most) : 0;
    const int step = n > 1 ? kWaves : min(kWaves, sh_ceil(r.tokens * p.group, 32));
    int all_t, all_u;
    const int at = n_tiles + sh_scan(n * parts, s_wave, all_t);
    const int unit = n_units + sh_scan(n * parts * step, s_wave, all_u);
    n_tiles += all_t;
    n_units += all_u;
    for (int i = 0; i < n * parts; ++i) {
      if (at + i >= p.cap_tiles) break;
      const int qt = i / parts, k = i - qt * parts;
      p.tiles[at + i] = ShTile{r.table, qt, r.q0, r.tokens, r.shared, (int)((long long)kv * k / parts),
                               (int)((long long)kv * (k + 1) / parts), (unit + i * step) * hkv, step, {0, 0, 0}};
    }
    if (g < p.groups) p.group_info[g].table = unit * hkv;  // (read below: the prefix's first unit)
    __syncthreads();
  }
  int n_chunks = 0;
  for (int b0 = 0; b0 < p.batch; b0 += kShPlanThreads) {
    const int b = b0 + tid;
    int3 s = make_int3(0, 0, 0);
    ShSeq q = {0, 0, 0, 0, 0, 0, 0, 0};
    int shared = 0;
    if (b < p.batch) {
      s = sh_sequence(p, b);
      const int g = s.y > 0 ? group_of(b) : -1;
      if (g >= 0) {
        const ShGroup r = p.group_info[g];
        const int n = group_pairs(r);
        if (n) {
          shared = r.shared;
          q.p_unit = r.table;
          q.p_parts = sh_ceil(r.shared / kTileN, most);
          q.p_step = n > 1 ? kWaves : min(kWaves, sh_ceil(r.tokens * p.group, 32));
          q.p_q0 = r.q0;
        }
      }
    }
    if (!p.cu_q) {
      const int tokens = max(0, s.z - shared);
      const int parts = sh_ceil(tokens, chunk), size = parts ? sh_ceil(tokens, parts) + 15 & ~15 : 0;
      int all;
      const int at = n_chunks + sh_scan(parts, s_wave, all);
      n_chunks += all;
      q.s_unit = at;
      q.s_parts = parts;
      const bool whole = parts == 1 && q.p_parts == 0;
      q.s_step = whole;
      for (int k = 0; k < parts && at + k < p.cap_chunks; ++k)
        p.chunks[at + k] = ShChunk{b, shared + k * size, min(shared + (k + 1) * size, s.z),
                                   (int)((uint32_t)(at + k) | (whole ? 0x80000000u : 0u))};
    } else {
      const int n = sh_ceil(s.y, p.tile_tokens);
      const int full = b < p.batch ? p.cu_q[b + 1] - s.x : 0;
      const int longest = n ? own_tiles(s, full, shared, n - 1) : 0;
      const int parts = sh_ceil(longest, most);
      const int step = n > 1 ? kWaves : min(kWaves, sh_ceil(s.y * p.group, 32));
      int all_t, all_u;
      const int at = n_tiles + sh_scan(n * parts, s_wave, all_t);
      const int unit = n_units + sh_scan(n * parts * step, s_wave, all_u);
      n_tiles += all_t;
      n_units += all_u;
      q.s_unit = unit * hkv;
      q.s_parts = parts;
      q.s_step = step;
      q.s_q0 = s.x;
      for (int i = 0; i < n * parts; ++i) {
        if (at + i >= p.cap_tiles) break;
        const int qt = i / parts, k = i - qt * parts;
        const int kv = own_tiles(s, full, shared, qt), lo = shared / kTileN;
        p.tiles[at + i] = ShTile{b, qt, s.x, s.y, s.z, lo + (int)((long long)kv * k / parts),
                                 lo + (int)((long long)kv * (k + 1) / parts), (unit + i * step) * hkv, step, {0, 0, 0}};
      }
    }
    if (b < p.batch) p.seqs[b] = q;
    __syncthreads();
  }
  // lists that do not fit (cu_groups that fall) are not run: every row is zero
  const bool fits = n_tiles <= p.cap_tiles && n_chunks <= p.cap_chunks && (long long)n_units * hkv <= p.cap_units;
  if (tid == 0) {
    p.header[0] = fits ? n_tiles : 0;
    p.header[1] = fits ? n_chunks : 0;
  }
  if (!fits)
    for (int b = tid; b < p.batch; b += kShPlanThreads) p.seqs[b] = ShSeq{0, 0, 0, 0, 0, 0, 0, 0};
}

// Parts of tile items: workgroup = (part, kv head).
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
  prefill_run<kSoftCap, kPaging, kPHeadDim, true>(p.pre, w, part);
}

// Chunks of own parts, one new token a sequence.  XCD x = bid % 8 takes chunks
// x, x + 8, ..., all kv heads of one in a row (they are adjacent in the pool).
template <bool kAligned, bool kSoftCap, bool kShared>
__global__ void __launch_bounds__(64 * kDecodeWaves, 2)
shared_decode_kernel(SharedParams p) {
  __shared__ DecodeLds red;
  const int vheads = p.num_kv_heads * p.dec.hblocks;
  const int k = blockIdx.x >> 3;
  const int kr = k / vheads;
  const int rank = 8 * kr + (blockIdx.x & 7);
  if (rank >= p.header[1]) return;  // uniform
  const ShChunk c = p.chunks[rank];
  DecodeWork w;
  w.b = __builtin_amdgcn_readfirstlane(c.b);
  w.vh = k - kr * vheads;
  w.t_begin = __builtin_amdgcn_readfirstlane(c.t0);
  w.t_end = __builtin_amdgcn_readfirstlane(c.t1);
  w.len = w.t_end;
  const int slot = __builtin_amdgcn_readfirstlane(c.slot);
  w.single = slot < 0;
  w.part = (int64_t)(slot & 0x7fffffff) * p.num_kv_heads + w.vh / p.dec.hblocks;
  decode_run<kDecodeWaves, kAligned, kSoftCap, false, kShared>(p.dec, w, &red.o[0][0][0], &red.m[0][0], &red.l[0][0]);
}

// One workgroup a (32 rows, kv head), one wave per 32 d: a lane has row n, d =
// 32 dt + 8 q4 + 4 h .. + 4, as prefill_run's accumulators.
__global__ void __launch_bounds__(256)
shared_merge_kernel(SharedParams p) {
  const int hkv = p.num_kv_heads;
  const int block = blockIdx.x / hkv, kvh = blockIdx.x - block * hkv;
  const int lane = threadIdx.x & 63, dt = threadIdx.x >> 6;
  const int n = lane & 31, h = lane >> 5;
  const int64_t row = (int64_t)32 * block + n;
  const int token = (int)(row / p.group), head = (int)(row - (int64_t)token * p.group);
  if (token >= p.num_tokens) return;
  const int b = p.cu_q ? p.owner[token] : token;
  if (b < 0 && !p.zero_rest) return;
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
    const int qt = at / p.tile_tokens;
    const int r = (at - qt * p.tile_tokens) * p.group + head;
    const float* src = p.pre.parts + ((int64_t)unit + ((int64_t)qt * parts * hkv + kvh) * step + (r >> 5)) *
                                         kPartFloats<kPHeadDim>;
    const float* po = src + 4 * (dt * 4 * 64 + 32 * h + (r & 31));
    const float* ml = src + kPartO<kPHeadDim> + 2 * (r & 31);
    const int64_t next = (int64_t)hkv * step * kPartFloats<kPHeadDim>;
#pragma unroll 4
    for (int k = 0; k < parts; ++k) {
      const f32x2 v = *reinterpret_cast<const f32x2*>(ml + k * next);
      add(po + k * next, 256, v[0], v[1]);
    }
  };
  if (b >= 0) {
    const ShSeq s = p.seqs[b];
    if (!p.cu_q && s.s_step) return;  // its one part wrote the row
    if (s.p_parts) add_tiles(s.p_unit, s.p_parts, s.p_step, s.p_q0);
    if (p.cu_q) {
      if (s.s_parts) add_tiles(s.s_unit, s.s_parts, s.s_step, s.s_q0);
    } else {
#pragma unroll 2
      for (int k = 0; k < s.s_parts; ++k) {
        const int64_t at = ((int64_t)(s.s_unit + k) * hkv + kvh) * p.group + head;
        const f32x2 v = *reinterpret_cast<const f32x2*>(p.dec.ws_ml + 2 * at);
        add(p.dec.ws_o + at * kHeadDim + 32 * dt + 4 * h, 8, v[0], v[1]);
      }
    }
  }
  const float inv = lsum > 0.f ? 1.f / lsum : 0.f;  // rows that see no key are zeros
  uint16_t* dst = p.pre.out + (int64_t)token * p.pre.o_ts + (int64_t)(kvh * p.group + head) * p.pre.o_hs + 32 * dt +
                  4 * h;
#pragma unroll
  for (int q4 = 0; q4 < 4; ++q4)
    *reinterpret_cast<u32x2*>(dst + 8 * q4) =
        u32x2{pack_bf16x2(o[q4][0] * inv, o[q4][1] * inv), pack_bf16x2(o[q4][2] * inv, o[q4][3] * inv)};
}

// What a launch of a shape needs: entries of the lists and bytes of the workspace.
struct ShSizes {
  int64_t tiles, units, chunks;
  int32_t chunk_cap;
  size_t header, groups, seqs, list, chunk_list, positions, owner, parts, dec_o, dec_ml, bytes;
};
size_t sh_up(size_t x) { return (x + 255) & ~(size_t)255; }

ShSizes shared_sizes(int64_t batch, int64_t groups, int64_t tokens, int64_t max_q, bool ragged, int64_t heads,
                     int64_t hkv, int64_t pages, int64_t page) {
  ShSizes z = {};
  const int64_t group = heads / hkv, tile = kRows / group;
  const int64_t span = pages * page;
  const int64_t extra = std::max<int64_t>(1, kShTileSlots / hkv);
  // q tiles of groups, and of sequences: a range of n tokens has ceil(n / tile)
  const int64_t prefix = std::min(groups, tokens) + tokens / tile;
  const int64_t mine = ragged ? std::min(batch, tokens) + tokens / tile : 0;
  const int64_t step = std::min<int64_t>(kWaves, (std::min(max_q, tokens) * group + 31) / 32);
  // parts of a share of the slots: one a pair and `extra` more
  z.tiles = prefix + mine + extra;
  z.units = hkv * (kWaves * (prefix + extra) + (max_q > tile ? kWaves : step) * mine);
  z.chunk_cap = (int32_t)std::max<int64_t>(16, std::min<int64_t>(2048, 62 * page) & ~(int64_t)15);
  if (!ragged) {
    const int64_t per = (span + z.chunk_cap - 1) / z.chunk_cap;  // of the longest sequence at the longest chunk
    const int64_t least = std::min<int64_t>(kShMinChunk, z.chunk_cap);
    z.chunks = std::min(batch * ((span + least - 1) / least),
                        batch + std::max(kShDecodeSlots / hkv + 1, batch * per));
  }
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t r = at;
    at += sh_up(bytes);
    return r;
  };
  z.header = take(kShHeader * sizeof(int32_t));
  z.groups = take(groups * sizeof(ShGroup));
  z.seqs = take(batch * sizeof(ShSeq));
  z.list = take(z.tiles * sizeof(ShTile));
  z.chunk_list = take((z.chunks + 8) * sizeof(ShChunk));
  z.positions = take(ragged ? tokens * sizeof(int32_t) : 0);
  z.owner = take(ragged ? tokens * sizeof(int32_t) : 0);
  z.parts = take((size_t)z.units * kPartFloats<kPHeadDim> * sizeof(float));
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
  p.tile_tokens = kRows / group;
  p.span = pages_per_seq * page_size;
  p.max_seqlen_q = max_seqlen_q;
  p.chunk_cap = z.chunk_cap;
  p.zero_rest = zero_rest;
  p.cap_tiles = (int32_t)z.tiles;
  p.cap_chunks = (int32_t)z.chunks;
  p.cap_units = (int32_t)z.units;
  p.header = (int32_t*)(ws + z.header);
  p.group_info = (ShGroup*)(ws + z.groups);
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
  if (z.tiles * num_kv_heads > kMaxGrid || (z.chunks + 7) / 8 * 8 * num_kv_heads * d.hblocks > 4 * kMaxGrid ||
      merges > 4 * kMaxGrid)
    return fail(PA_ERR_UNSUPPORTED, "%s: %lld parts of %lld rows", name, (long long)(z.tiles + z.chunks),
                (long long)merges * 32);
  const int64_t maps = ragged ? (num_tokens + kShPlanThreads - 1) / kShPlanThreads : 0;
  shared_plan_kernel<<<dim3((unsigned)(1 + maps)), dim3(kShPlanThreads), 0, s>>>(p);
  if (int rc = launch_status(name)) return rc;
  if (num_groups > 0 || ragged) {
    const dim3 grid((unsigned)(z.tiles * num_kv_heads)), blk(kThreads);
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
    const dim3 grid((unsigned)((z.chunks + 7) / 8 * 8 * num_kv_heads * d.hblocks)), blk(64 * kDecodeWaves);
    auto launch = [&](auto al, auto c, auto sh) {
      shared_decode_kernel<decltype(al)::value, decltype(c)::value, decltype(sh)::value><<<grid, blk, 0, s>>>(p);
    };
    auto by_cap = [&](auto al, auto sh) {
      if (cap) launch(al, std::true_type{}, sh);
      else launch(al, std::false_type{}, sh);
    };
    auto by_group = [&](auto al) {
      if (d.hblocks > 1) by_cap(al, std::true_type{});
      else by_cap(al, std::false_type{});
    };
    if (page_size % kDecodeStep == 0) by_group(std::true_type{});
    else by_group(std::false_type{});
    if (int rc = launch_status(name)) return rc;
  }
  shared_merge_kernel<<<dim3((unsigned)merges), dim3(256), 0, s>>>(p);
  return launch_status(name);
}
