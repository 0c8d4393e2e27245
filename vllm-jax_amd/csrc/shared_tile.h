// Rows against a range of one sequence's tokens, as a workgroup of four waves
// that shares its CU: 128 rows, a row being a (token, q head of the kv head) pair,
// by 32-token tiles, head size 128.
//
// Per tile and wave (32 rows, row n = lane % 32):
//   S^T[t][n] = K[t][:] . Q[n][:]       8 x v_mfma_f32_32x32x16_bf16
//   online softmax per row n            (the reference maximum moves only when a
//                                       row's exceeds it by 2^8)
//   O^T[d][n] += V^T[d][t] . P^T[t][n]  8 x v_mfma_f32_32x32x16_bf16
// K and V come through a ring of kLtStages tiles in LDS by direct loads, three
// tiles ahead; V is read transposed (ds_read_b64_tr_b16), P goes from the first
// product's accumulators into the second's operand in registers.  64 KiB of LDS
// and at most 256 registers a wave: two workgroups a CU, so that one's products
// run under the other's softmax, or, beside decode_run's workgroups, under their
// loads.  q is not scaled (and not rounded again): the scale is a factor of the
// exponent.  512 rows a kv head (32 / 8 heads), two workgroups a CU: 1 000 TFLOP/s
// from 16384 shared tokens to 65536 (61 to 164 us).  A wave and tile reads 16 KiB of
// operands from LDS (an operand feeds its 32 rows alone) for 16 matrix instructions
// of 32 cycles, so that at four waves a workgroup both need 512 cycles; by the
// counters the matrix cores are busy 39 % of the time and the waves wait 41 %.
#pragma once

#include <type_traits>

#include "lds_tiles.h"
#include "pa_common.h"

namespace pa {

constexpr int kLtWaves = 4;
constexpr int kLtRows = 32 * kLtWaves;
constexpr int kLtTile = 32;                       // tokens of a tile
constexpr int kLtStages = 4;
constexpr int kLtStageB = kLtTile * 256;          // bytes of a K (or V) tile
constexpr int kLtLdsB = 2 * kLtStages * kLtStageB;
constexpr float kLtSlack = 8.f;                   // lazy-rescale threshold (log2 units)
constexpr int kLtUnit = 32 * 128 + 2 * 32;        // floats of a 32-row partial: O, then (max, sum) a row

struct LtParams {
  const uint16_t* q;
  int64_t q_ts, q_hs;
  const uint16_t* k;
  const uint16_t* v;
  int32_t num_pages, page_size;  // page_size a multiple of 16
  int64_t page_stride, slot_stride, head_stride;
  const int32_t* block_tables;
  int64_t bt_stride;
  int32_t pages_per_seq, group;
  float logit_scale, soft_cap;   // as DecodeParams
  float* parts;
};

// One item: rows [row0, row0 + 128) of the kv head's rows (row r: token q0 + r /
// group, head r % group; `rows` of them in all) against tokens [t0, t1) of the
// sequence at `bt_row`, t0 a multiple of 32 and t1 at most lk.  A lane's row sees
// the tokens below `limit`.  Leaves a partial in units `unit` .. + 3; waves
// without a row write none.  `lds`: byte address of kLtLdsB bytes.
template <bool kSoftCap>
__device__ __forceinline__ void lt_run(const LtParams& p, const int32_t* bt_row, int kvh, int q0, int rows, int row0,
                                       int t0, int t1, int limit, int unit, uint32_t lds) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 31, h = lane >> 5;
  const uint32_t k_lds = lds, v_lds = lds + kLtStages * kLtStageB;
  const bool live = row0 + 32 * wave < rows;  // (uniform) the wave has a row

  // Q^T operand: lane (n, h)'s k-step ks is row n, d = 16 ks + 8 h ..; lanes
  // without a row repeat the last one (their columns are never stored)
  bf16x8 qt[8];
  {
    const int r = min(row0 + 32 * wave + n, rows - 1);
    const int tk = r / p.group;
    const uint16_t* src = p.q + (int64_t)(q0 + tk) * p.q_ts + (int64_t)(kvh * p.group + r - tk * p.group) * p.q_hs + 8 * h;
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) qt[ks] = as_bf16x8(ld16(src + 16 * ks));
  }
  // the exponent's factor is positive: q takes a negative scale's sign
  const float c = kSoftCap ? 1.f : fmaxf(fabsf(p.logit_scale), 1e-30f);  // (-inf times it stays -inf)
  if (!kSoftCap && p.logit_scale < 0.f) {
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) {
      const u32x4 w = as_u32x4(qt[ks]);
      qt[ks] = as_bf16x8(u32x4{w[0] ^ 0x80008000u, w[1] ^ 0x80008000u, w[2] ^ 0x80008000u, w[3] ^ 0x80008000u});
    }
  }
  const float cap_s2 = kSoftCap ? soft_cap_s2(p.logit_scale, p.soft_cap) : 0.f;
  const float cap_c = kSoftCap ? soft_cap_c(p.soft_cap) : 0.f;

  // tokens below `free` need no mask in this wave
  int free = min(limit, t1);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) free = min(free, __shfl_xor(free, o));
  free = __builtin_amdgcn_readfirstlane(free);

  // ---- tile loads.  Wave w fills 1 KiB blocks 2 w and 2 w + 1 (rows 8 w .. 8 w +
  // 7) of K and of V: lane l row l / 16 of a block, 16-byte chunk (l % 16) ^
  // swz(row).  Eight aligned rows lie in one page of a multiple of 16 tokens.
  const int64_t head_off = (int64_t)kvh * p.head_stride;
  const int last_tok = max(t1 - 1, 0);  // (a part without tokens reads the first, and weighs it nothing)
  auto page_of = [&](int lp) __attribute__((always_inline)) {
    return safe_page_scalar(bt_row, min(max(lp, 0), p.pages_per_seq - 1), p.num_pages);
  };
  // the wave's rows of the next tile to load: token, its table entry and offset there
  int nx_tok = t0 + 8 * wave;
  int nx_lp = nx_tok / p.page_size, nx_off = nx_tok - nx_lp * p.page_size;
  const int tail_lp = last_tok / p.page_size, tail_off = last_tok - tail_lp * p.page_size;
  int32_t nx_page = page_of(min(nx_lp, tail_lp));
  uint32_t sw[2], ro[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = 4 * i + (lane >> 4);  // row of the wave's eight
    sw[i] = (uint32_t)(16 * ((lane & 15) ^ swz256(8 * wave + r)));
    ro[i] = (uint32_t)(2 * r * (int32_t)p.slot_stride) + sw[i];
  }
  auto issue = [&](int stage) __attribute__((always_inline)) {
    const bool past = nx_tok > last_tok;  // uniform: all eight rows are behind the range
    const int off = past ? tail_off : nx_off;
    const int left = past ? 0 : min(last_tok - nx_tok, 7);  // rows of the eight behind the first, inside the range
    const int64_t base = (int64_t)nx_page * p.page_stride + (int64_t)off * p.slot_stride + head_off;
    const char* kb = (const char*)(p.k + base);
    const char* vb = (const char*)(p.v + base);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = 4 * i + (lane >> 4);
      const uint32_t vo = r <= left ? ro[i] : (uint32_t)(2 * left * (int32_t)p.slot_stride) + sw[i];
      const uint32_t at = (uint32_t)(stage * kLtStageB + (2 * wave + i) * 1024);
      lds_dma16v(vo, kb, k_lds + at);
      lds_dma16v(vo, vb, v_lds + at);
    }
    nx_tok += kLtTile;
    if (p.page_size == 16) {
      nx_lp += 2;
    } else {
      nx_off += kLtTile;
      while (nx_off >= p.page_size) {  // (a page of 48 holds one and a half tiles)
        nx_off -= p.page_size;
        ++nx_lp;
      }
    }
    nx_page = page_of(min(nx_lp, tail_lp));
  };
  constexpr int kDma = 4;  // loads of a tile a wave issues

  // ---- LDS operand addresses
  const int fn = swz256(n);
  uint32_t koff[8];
#pragma unroll
  for (int ks = 0; ks < 8; ++ks) koff[ks] = k_lds + n * 256 + 16 * ((2 * ks + h) ^ fn);
  const int tr_s = lane & 15, tr_g = (lane >> 4) & 1;
  const int tr_row = 4 * h + (tr_s >> 2);
  uint32_t voff0[4], voff1[4];
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) {
    const int ch = 4 * dt + 2 * tr_g + ((tr_s & 3) >> 1);
    voff0[dt] = v_lds + tr_row * 256 + 16 * (ch ^ swz256(tr_row)) + 8 * (tr_s & 1);
    voff1[dt] = v_lds + (tr_row + 8) * 256 + 16 * (ch ^ swz256(tr_row + 8)) + 8 * (tr_s & 1);
  }

  f32x16 acc[4];
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[dt][i] = 0.f;
  float m_ref = -1e30f, l0 = 0.f, l1 = 0.f;  // (finite: exp2(x - m) never sees inf - inf)

  auto tile = [&](int tok, auto st) __attribute__((always_inline)) {
    constexpr uint32_t so = decltype(st)::value * kLtStageB;
    wait_vm<2 * kDma>();  // this wave's share of the tile has landed
    lds_barrier();        // all shares have, and every wave is done with the tile before
    issue((decltype(st)::value + 3) % kLtStages);
    if (!live) return;
    f32x16 s = {};
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) s = mfma32(as_bf16x8(lds_ld16(koff[ks] + so)), qt[ks], s);
    // s[i] = S[row n][token tok + 8 (i / 4) + 4 h + i % 4]
    if constexpr (kSoftCap) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = soft_cap_log2(s[i], cap_s2, cap_c);
    }
    if (tok + kLtTile > free) {  // uniform
      const int lim = min(limit, t1) - tok - 4 * h;
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = 8 * (i >> 2) + (i & 3) < lim ? s[i] : -INFINITY;
    }
    float ma = fmaxf(fmaxf(s[0], s[1]), s[2]), mb = fmaxf(fmaxf(s[8], s[9]), s[10]);
#pragma unroll
    for (int i = 3; i < 8; ++i) {
      ma = fmaxf(ma, s[i]);
      mb = fmaxf(mb, s[8 + i]);
    }
    const float mx = max_xor32(fmaxf(ma, mb)) * c;
    if (__any(mx > m_ref + kLtSlack)) {
      const float m_new = fmaxf(m_ref, mx);
      const float corr = fast_exp2(m_ref - m_new);
      m_ref = m_new;
      l0 *= corr;
      l1 *= corr;
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) acc[dt] = acc[dt] * corr;
    }
    bf16x8 pt[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      u32x4 w;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float a = fast_exp2(__builtin_fmaf(s[8 * u + 2 * e], c, -m_ref));
        const float b = fast_exp2(__builtin_fmaf(s[8 * u + 2 * e + 1], c, -m_ref));
        w[e] = pack_bf16x2(a, b);
        if (u) l1 += a + b;
        else l0 += a + b;
      }
      pt[u] = as_bf16x8(w);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) {
        const u32x2 lo = lds_tr8(voff0[dt] + so + 16 * 256 * u), hi = lds_tr8(voff1[dt] + so + 16 * 256 * u);
        acc[dt] = mfma32(as_bf16x8(u32x4{lo[0], lo[1], hi[0], hi[1]}), pt[u], acc[dt]);
      }
  };
  // nothing that the compiler issued may still be in flight when the counted
  // loads start
#pragma unroll
  for (int ks = 0; ks < 8; ++ks) asm volatile("" : "+v"(qt[ks]));
  wait_vm<0>();
  asm volatile("" ::: "memory");
  issue(0);
  issue(1);
  issue(2);
  for (int tok = t0;;) {
    tile(tok, std::integral_constant<int, 0>{});
    if ((tok += kLtTile) >= t1) break;
    tile(tok, std::integral_constant<int, 1>{});
    if ((tok += kLtTile) >= t1) break;
    tile(tok, std::integral_constant<int, 2>{});
    if ((tok += kLtTile) >= t1) break;
    tile(tok, std::integral_constant<int, 3>{});
    if ((tok += kLtTile) >= t1) break;
  }
  wait_vm<0>();  // loads of tiles behind the range may still be in flight
  if (!live) return;
  const float l_run = sum_xor32(l0 + l1);
  float* dst = p.parts + (int64_t)(unit + wave) * kLtUnit;
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4)
      *reinterpret_cast<f32x4*>(dst + 4 * ((dt * 4 + q4) * 64 + lane)) =
          f32x4{acc[dt][4 * q4], acc[dt][4 * q4 + 1], acc[dt][4 * q4 + 2], acc[dt][4 * q4 + 3]};
  // a row that saw no key carries no weight, whatever its reference
  if (h == 0) *reinterpret_cast<f32x2*>(dst + 32 * 128 + 2 * n) = f32x2{l_run > 0.f ? m_ref : -INFINITY, l_run};
}

}  // namespace pa
