// Expanded-form latent attention for gfx950: ragged causal attention of new
// tokens over expanded K and V rows, key size DN + DR (the rotary part shared by
// all heads), value size DN.
//
// Workgroup = 256 query rows of one (sequence, head), eight waves of 32 rows.
// kv tiles of 64 tokens come by direct loads into three-stage LDS rings, K's
// unrotated part, K's rotary part and V apart, since K of a tile is read one
// half step before its V:
//   S^T[t][n] = K[t] . Q[n]     v_mfma_f32_32x32x16_bf16, K by 16-byte reads, Q^T
//                               in registers
//   O^T[d][n] += V^T P^T        V^T by transposing reads, P^T from the accumulators
// Waves 0-3 and 4-7 share the SIMDs pairwise and run the same sequence half a
// step apart, so that one wave's softmax runs under the other's products:
//   segment 2t:   A: PV(t-1), QK(t)   B: softmax(t-1)
//   segment 2t+1: A: softmax(t)       B: PV(t-1), QK(t)
// with a barrier behind every segment.  Of tile T, A issues its share of K(T)
// and V(T-1) behind its QK(T-2) and waits for it behind softmax(T-1); B issues
// half a step earlier, behind QK(T-3), and waits behind softmax(T-2).  K(T)
// overwrites K(T-3), last read by B in segment 2T-5; V(T-1) overwrites V(T-4),
// last read by B in segment 2T-5 as well; both are issued in 2T-4 or later.
//
// Rows: the softmax reference of a row moves only when its maximum grows by
// more than 2^8, so O is rarely rescaled; the exponent is one fused
// multiply-add (scores are float32 sums of unscaled bf16 products).  P is
// rounded to bf16 for the matrix cores (2^8 at most, so far from its range's
// ends); its sum, the statistics and O are float32.
//
// Bound by the power limit: two documents of 8-16 k tokens by 64 heads take 7.8 to
// 8.1 ms, 1 170 to 1 210 TFLOP/s issued, where a large library product reaches
// 1 230, with the matrix cores busy for 74 % of the time at 1.5 GHz and LDS reads
// for 37 %, without bank conflicts.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "latent_attend.h"
#include "lds_tiles.h"
#include "pa_errors.h"
#include "../../include/latent_attention.h"

namespace pa {
namespace {

constexpr int kRWaves = 8, kRThreads = 64 * kRWaves, kRRows = 32 * kRWaves;
constexpr int kRTile = 64, kRStages = 3;
constexpr float kRSlack = 8.f;

// Workgroups of a launch: a grid has fewer than 2^32 threads along x.
constexpr int64_t kRGrid = (1 << 22) - 1;  // and as many to zero rows

struct RaggedParams {
  LatentRagged r;
  float scale_log2;
  int32_t n_qtiles;
  int32_t level0;  // first level of this launch
};

template <int DN, int DR>
struct RDims {
  static constexpr int kKB = 2 * DN, kRB = 2 * DR;  // bytes of a K, V and a rotary row
  static constexpr int kKStage = kRTile * kKB, kRStage = kRTile * kRB;
  static constexpr int kKOff = 0, kROff = kRStages * kKStage, kVOff = kROff + kRStages * kRStage;
  static constexpr int kLds = kVOff + kRStages * kKStage;
  static constexpr int kKDma = kKStage / (1024 * kRWaves);  // loads of a wave per tile of K and of V
  static constexpr int kRowsK = 1024 / kKB;                 // rows of a load
  static constexpr int kDma = 2 * kKDma + 1;
  static constexpr int kKs = DN / 16, kRs = DR / 16;
  static constexpr int kDt = DN / 32;
};

// s_waitcnt vmcnt(N) lgkmcnt(0)
template <int N>
__device__ __forceinline__ void wait_vm_lgkm() {
  static_assert(N < 16);
  __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4));
}

template <int DN>
__device__ __forceinline__ int k_swz(int r) {
  return DN == 128 ? swz256(r) : swz128(r);
}
template <int DN>
__device__ __forceinline__ int v_swz(int r) {
  return DN == 128 ? swz256(r) : value_swz128(r);
}
template <int DR>
__device__ __forceinline__ int r_swz(int r) {
  return DR == 64 ? swz128(r) : swz64(r);
}

// Zeroes the rows of 512 tokens from t0 on that no sequence has: a lane looks
// one token up, the wave zeroes those that were not found (a token a wave at a
// time took 34 us for 512 tokens, longer than a short prompt's attention).
template <int DN>
__device__ __forceinline__ void zero_rows(const LatentRagged& p, int64_t t0) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t first = t0 + 64 * wave, own = first + lane;
  uint64_t rest = __ballot(own < p.num_tokens && !token_in_sequence(p.cu_q, p.batch, p.max_q, (int)own));
  for (; rest; rest &= rest - 1) {
    uint16_t* row = p.zero_out + (first + __builtin_ctzll(rest)) * p.o_ts;
    for (int c = lane; c < p.zero_heads * (DN / 8); c += 64)
      st16(row + (c / (DN / 8)) * p.o_hs + (c % (DN / 8)) * 8, u32x4{0, 0, 0, 0});
  }
}

template <int DN, int DR>
__global__ void __launch_bounds__(kRThreads) __attribute__((amdgpu_waves_per_eu(2, 2)))
latent_ragged_kernel(RaggedParams prm) {
  using D = RDims<DN, DR>;
  const LatentRagged& p = prm.r;
  __shared__ __attribute__((aligned(1024))) char smem[D::kLds];
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void)smem;
  // Items from the last query tile down (the longest rows first); within a
  // level (sequence, head) pairs in order, so that with a multiple of eight
  // heads all query tiles of a pair run on one XCD and share its L2.
  const int pairs = max(p.batch * p.heads, 1);  // no sequences: nothing but rows to zero
  int level = blockIdx.x / pairs;
  const int pair = blockIdx.x - level * pairs;
  level += prm.level0;
  if (level >= prm.n_qtiles) {
    zero_rows<DN>(p, ((int64_t)blockIdx.x - (int64_t)(prm.n_qtiles - prm.level0) * pairs) * kRThreads);
    return;
  }
  const int qt = prm.n_qtiles - 1 - level;
  const int b = pair / p.heads, head = pair - b * p.heads;
  const int q0 = p.cu_q[b];
  const int lq_all = p.cu_q[b + 1] - q0;
  const int lq = q0 < 0 || q0 >= p.num_tokens ? 0 : min(min(lq_all, p.max_q), p.num_tokens - q0);
  if (qt * kRRows >= lq) return;
  const int64_t kbase = flat_start(p.cu_k, b, p.span);
  const int lk_all = max(0, min(p.cu_k[b + 1] - p.cu_k[b], p.span));
  const int lk = kbase < 0 || kbase >= p.cap ? 0 : min(lk_all, p.cap - (int)kbase);
  const int first = lk_all - lq_all;  // row i sees first + i + 1 keys

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 31, h = lane >> 5;
  const int row = qt * kRRows + 32 * wave + n;
  const bool wave_live = qt * kRRows + 32 * wave < lq;
  // tokens this row sees (rows past the sequence's end compute on its last row
  // and store nothing)
  const int seen = min(lk, max(0, first + min(row, lq - 1) + 1));
  const int kv_hi = min(lk, max(0, first + min(lq, (qt + 1) * kRRows)));
  const int n_tiles = (kv_hi + kRTile - 1) / kRTile;
  const int n_free = min(lk, max(0, first + qt * kRRows + 1)) / kRTile;

  const uint16_t* kv = p.kv + ((int64_t)head * p.cap + kbase) * (2 * DN);
  const uint16_t* kr = p.k_rope + kbase * DR;

  // ---- tile loads: this wave's rows of a tile are 8 wave .. 8 wave + 7, each load
  // a scalar tile base and a lane offset kept in a register.  Piece i of kDma:
  // K's, the rotary parts', V's.  Rows past the kv length repeat the last one.
  constexpr int kRowChunks = D::kKB / 16, kRopeChunks = D::kRB / 16;
  uint32_t off_k[D::kKDma], off_v[D::kKDma], off_r;
#pragma unroll
  for (int i = 0; i < D::kKDma; ++i) {
    const int r = 8 * wave + i * D::kRowsK + lane / kRowChunks, c = lane & (kRowChunks - 1);
    off_k[i] = 2 * D::kKB * r + 16 * (c ^ k_swz<DN>(r));
    off_v[i] = 2 * D::kKB * r + D::kKB + 16 * (c ^ v_swz<DN>(r));
  }
  {
    const int r = 8 * wave + (lane / kRopeChunks & 7), c = lane & (kRopeChunks - 1);
    off_r = D::kRB * r + 16 * (c ^ r_swz<DR>(r));
  }
  auto issue = [&](int i, int tk, int ks, int tv, int vs) __attribute__((always_inline)) {
    const int t = i <= D::kKDma ? tk : tv;
    const int j0 = min(t * kRTile, max(lk - 1, 0)), last = max(lk - 1 - t * kRTile, 0);
    const int lrow = i == D::kKDma ? lane / kRopeChunks & 7
                                   : (i < D::kKDma ? i : i - D::kKDma - 1) * D::kRowsK + lane / kRowChunks;
    // rows of the tile past the last valid one
    const int past = last < kRTile - 1 ? max(8 * wave + lrow - last, 0) : 0;
    if (i < D::kKDma) {
      lds_dma16s(off_k[i] - 2 * D::kKB * past, kv + (int64_t)j0 * (2 * DN),
                 lds0 + (uint32_t)(D::kKOff + ks * D::kKStage + 8 * wave * D::kKB + 1024 * i));
    } else if (i > D::kKDma) {
      lds_dma16s(off_v[i - D::kKDma - 1] - 2 * D::kKB * past, kv + (int64_t)j0 * (2 * DN),
                 lds0 + (uint32_t)(D::kVOff + vs * D::kKStage + 8 * wave * D::kKB + 1024 * (i - D::kKDma - 1)));
    } else if (kRopeChunks == 8 || lane < 8 * kRopeChunks) {
      lds_dma16s(off_r - D::kRB * past, kr + (int64_t)j0 * DR,
                 lds0 + (uint32_t)(D::kROff + ks * D::kRStage + 8 * wave * D::kRB));
    }
  };
  auto issue_k = [&](int t, int st) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i <= D::kKDma; ++i) issue(i, t, st, 0, 0);
  };
  auto issue_v = [&](int t, int st) __attribute__((always_inline)) {
#pragma unroll
    for (int i = D::kKDma + 1; i < D::kDma; ++i) issue(i, 0, 0, t, st);
  };

  // ---- LDS read addresses
  constexpr int kKAddr = D::kKs < 8 ? D::kKs : 8;
  uint32_t koff[kKAddr], roff[D::kRs];
#pragma unroll
  for (int ks = 0; ks < kKAddr; ++ks)
    koff[ks] = lds0 + D::kKOff + n * D::kKB + 16 * ((2 * ks + h) ^ k_swz<DN>(n));
#pragma unroll
  for (int ks = 0; ks < D::kRs; ++ks)
    roff[ks] = lds0 + D::kROff + n * D::kRB + 16 * ((2 * ks + h) ^ r_swz<DR>(n));
  const int ts = lane & 15, gamma = lane >> 4, tr = 4 * h + (ts >> 2);
  uint32_t voff0[D::kDt], voff1[D::kDt];
#pragma unroll
  for (int dt = 0; dt < D::kDt; ++dt) {
    const int c = 4 * dt + 2 * (gamma & 1) + ((ts & 3) >> 1);
    voff0[dt] = lds0 + D::kVOff + tr * D::kKB + 16 * (c ^ v_swz<DN>(tr)) + 8 * (ts & 1);
    voff1[dt] = lds0 + D::kVOff + (tr + 8) * D::kKB + 16 * (c ^ v_swz<DN>(tr + 8)) + 8 * (ts & 1);
  }

  bf16x8 q[D::kKs + D::kRs];
  f32x16 acc[D::kDt] = {};
  float m_ref = 0.f;
  float l_part[4] = {};
  f32x16 s[2];
  bf16x8 pt[4];

  // Product i of a segment: those of O^T += V^T P^T of the previous tile (stage
  // `vst`), then those of S^T = K Q^T (stage `kst`).  Every operand is read
  // kAhead products before the one it feeds.
  constexpr int kPvN = 4 * D::kDt, kQkN = 2 * (D::kKs + D::kRs), kAhead = 6;
  auto products = [&](auto from_c, auto to_c, int vst, int kst) __attribute__((always_inline)) {
    constexpr int from = decltype(from_c)::value, to = decltype(to_c)::value;
    bf16x8 a[to];
    uint32_t ka[kKAddr], ra[D::kRs], va0[D::kDt], va1[D::kDt];
#pragma unroll
    for (int i = 0; i < kKAddr; ++i) ka[i] = koff[i] + kst * D::kKStage;
#pragma unroll
    for (int i = 0; i < D::kRs; ++i) ra[i] = roff[i] + kst * D::kRStage;
#pragma unroll
    for (int i = 0; i < D::kDt; ++i) {
      va0[i] = voff0[i] + vst * D::kKStage;
      va1[i] = voff1[i] + vst * D::kKStage;
    }
    auto fetch = [&](int i) __attribute__((always_inline)) {
      if (i < kPvN) {
        const int u = i / D::kDt, dt = i % D::kDt;
        const u32x2 lo = lds_tr8(va0[dt] + 16 * u * D::kKB), hi = lds_tr8(va1[dt] + 16 * u * D::kKB);
        a[i] = as_bf16x8(u32x4{lo[0], lo[1], hi[0], hi[1]});
      } else {
        const int ks = (i - kPvN) / 2, mt = (i - kPvN) % 2;
        a[i] = as_bf16x8(lds_ld16(ks < D::kKs ? ka[ks % kKAddr] + mt * (32 * D::kKB)
                                              : ra[(ks - D::kKs) % D::kRs] + mt * (32 * D::kRB)));
      }
    };
#pragma unroll
    for (int i = from; i < from + kAhead; ++i) fetch(i);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = from; i < to; ++i) {
      if (i < kPvN) {
        acc[i % D::kDt] = mfma32(a[i], pt[i / D::kDt], acc[i % D::kDt]);
      } else {
        const int ks = (i - kPvN) / 2, mt = (i - kPvN) % 2;
        s[mt] = mfma32(a[i], q[ks], ks == 0 ? f32x16{} : s[mt]);
      }
      if (i + kAhead < to) fetch(i + kAhead);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  using PvBegin = std::integral_constant<int, 0>;
  using QkBegin = std::integral_constant<int, kPvN>;
  using QkEnd = std::integral_constant<int, kPvN + kQkN>;
  const float scale = prm.scale_log2;
  auto softmax = [&](int t, auto&& between) __attribute__((always_inline)) {
    // s[mt][i] is token 64 t + 32 mt + 8 (i / 4) + 4 h + i % 4
    if (t >= n_free) {
      int lim = min(max(seen - t * kRTile - 4 * h, 0), kRTile);
      asm volatile("" : "+v"(lim));
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          s[mt][i] = 32 * mt + 8 * (i >> 2) + (i & 3) < lim ? s[mt][i] : -INFINITY;
    }
    float mq[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const f32x16& v = s[k >> 1];
      const int b0 = 8 * (k & 1);
      float m = __builtin_fmaxf(__builtin_fmaxf(v[b0], v[b0 + 1]), v[b0 + 2]);
      m = __builtin_fmaxf(__builtin_fmaxf(m, v[b0 + 3]), v[b0 + 4]);
      m = __builtin_fmaxf(__builtin_fmaxf(m, v[b0 + 5]), v[b0 + 6]);
      mq[k] = __builtin_fmaxf(m, v[b0 + 7]);
    }
    const float mx = max_xor32(__builtin_fmaxf(__builtin_fmaxf(mq[0], mq[1]), __builtin_fmaxf(mq[2], mq[3])));
    const float up = mx * scale - m_ref;  // the scale is positive
    if (t == 0 || __any(up > kRSlack)) {
      // the first tile sets the reference to the row's maximum (a row that
      // sees no key keeps 0)
      const float d = t == 0 ? (mx == -INFINITY ? 0.f : up) : __builtin_fmaxf(up, 0.f);
      if (t != 0) {
        const float corr = fast_exp2(-d);
#pragma unroll
        for (int u = 0; u < 4; ++u) l_part[u] *= corr;
#pragma unroll
        for (int dt = 0; dt < D::kDt; ++dt) acc[dt] = acc[dt] * corr;
      }
      m_ref += d;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      between(u);
      u32x4 w;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float a = fast_exp2(__builtin_fmaf(s[u >> 1][8 * (u & 1) + 2 * e], scale, -m_ref));
        const float c = fast_exp2(__builtin_fmaf(s[u >> 1][8 * (u & 1) + 2 * e + 1], scale, -m_ref));
        w[e] = pack_bf16x2(a, c);
        l_part[u] += a + c;
      }
      pt[u] = as_bf16x8(w);
      asm volatile("" : "+v"(pt[u]));  // made here, not in the next product segment
    }
    asm volatile("" : "+v"(l_part[0]), "+v"(l_part[1]), "+v"(l_part[2]), "+v"(l_part[3]));
  };

  const bool grp_b = wave >= kRWaves / 2;
  using T_ = std::true_type;
  using F_ = std::false_type;
  auto iteration = [&](int t, auto stc, auto has_pv) __attribute__((always_inline)) {
    constexpr int st = decltype(stc)::value;  // t % 3
    constexpr bool kPv = decltype(has_pv)::value;
    if (!kPv || wave_live) {
      if constexpr (kPv) products(PvBegin{}, QkEnd{}, (st + 2) % 3, st);
      else products(QkBegin{}, QkEnd{}, 0, st);
    }
    wait_lgkm0();
    lds_barrier();
    const int tk = t + (grp_b ? 3 : 2);  // K of tile tk, V of tile tk - 1
    const int ks = grp_b ? st : (st + 2) % 3, vs = grp_b ? (st + 2) % 3 : (st + 1) % 3;
    auto between = [&](int u) __attribute__((always_inline)) {
#pragma unroll
      for (int i = u * D::kDma / 4; i < (u + 1) * D::kDma / 4; ++i) issue(i, tk, ks, tk - 1, vs);
    };
    if (!kPv || wave_live) {
      softmax(t, between);
    } else {
#pragma unroll
      for (int u = 0; u < 4; ++u) between(u);
    }
    wait_vm_lgkm<D::kDma>();
    lds_barrier();
  };
  using S0 = std::integral_constant<int, 0>;
  using S1 = std::integral_constant<int, 1>;
  using S2 = std::integral_constant<int, 2>;

  // The first tiles' loads, then Q's, so that their latencies overlap.
  if (n_tiles > 0) {
    issue_k(0, 0);
    issue_k(1, 1);
    issue_v(0, 0);
    if (grp_b) {
      issue_k(2, 2);
      issue_v(1, 1);
    }
  }
  // ---- Q^T (waited for here, and with it all loads above: from now on vmcnt
  // counts the loop's tile loads)
  {
    const int64_t t = q0 + min(row, lq - 1);
    const uint16_t* qn = p.q_nope + t * p.qn_ts + head * p.qn_hs + 8 * h;
    const uint16_t* qr = p.q_rope + t * p.qr_ts + head * p.qr_hs + 8 * h;
#pragma unroll
    for (int ks = 0; ks < D::kKs; ++ks) q[ks] = as_bf16x8(ld16(qn + 16 * ks));
#pragma unroll
    for (int ks = 0; ks < D::kRs; ++ks) q[D::kKs + ks] = as_bf16x8(ld16(qr + 16 * ks));
  }
#pragma unroll
  for (int ks = 0; ks < D::kKs + D::kRs; ++ks) asm volatile("" : "+v"(q[ks]));
  wait_vm<0>();
  if (n_tiles > 0) {
    lds_barrier();
    if (grp_b) lds_barrier();
    iteration(0, S0{}, F_{});
    int last = 0;  // stage of the last tile
    for (int t = 1; t < n_tiles; ++t) {
      iteration(t, S1{}, T_{});
      last = 1;
      if (++t == n_tiles) break;
      iteration(t, S2{}, T_{});
      last = 2;
      if (++t == n_tiles) break;
      iteration(t, S0{}, T_{});
      last = 0;
    }
    // V of the last tile: A's share landed an iteration ago, B's before that
    products(PvBegin{}, QkBegin{}, last, 0);
    wait_vm_lgkm<0>();  // loads of tiles past the end may still be in flight
    if (!grp_b) lds_barrier();
  }

  const float l = sum_xor32((l_part[0] + l_part[1]) + (l_part[2] + l_part[3]));
  const float inv = l > 0.f ? 1.f / l : 0.f;
  if (row < lq) {
    uint16_t* o = p.out + (int64_t)(q0 + row) * p.o_ts + head * p.o_hs + 4 * h;
#pragma unroll
    for (int dt = 0; dt < D::kDt; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<u32x2*>(o + 32 * dt + 8 * i) =
            u32x2{pack_bf16x2(acc[dt][4 * i] * inv, acc[dt][4 * i + 1] * inv),
                  pack_bf16x2(acc[dt][4 * i + 2] * inv, acc[dt][4 * i + 3] * inv)};
  }
}

template <int DN, int DR>
int ragged_launch(const char* name, RaggedParams p, hipStream_t s) {
  const int64_t zero = p.r.zero_out ? ((int64_t)p.r.num_tokens + kRThreads - 1) / kRThreads : 0;
  const int64_t pairs = (int64_t)p.r.batch * p.r.heads;
  if (pairs > kRGrid) return fail(PA_ERR_UNSUPPORTED, "%s: %d sequences", name, p.r.batch);
  // as many levels at a time as a grid holds, the rows to zero behind the last
  int32_t left = pairs ? p.n_qtiles : 0;
  p.level0 = p.n_qtiles - left;
  for (bool rows = zero > 0; left > 0 || rows;) {
    const int64_t take = pairs ? std::min<int64_t>(left, kRGrid / pairs) : 0;
    int64_t blocks = take * pairs;
    if (take == left) {
      blocks += zero;
      rows = false;
    }
    latent_ragged_kernel<DN, DR><<<dim3((unsigned)blocks), kRThreads, 0, s>>>(p);
    if (int rc = launch_status(name)) return rc;
    p.level0 += (int32_t)take;
    left -= (int32_t)take;
  }
  return PA_OK;
}

}  // namespace

int latent_ragged_launch(const char* name, const LatentRagged& r, int nope, int rope, hipStream_t s) {
  RaggedParams p;
  p.r = r;
  p.scale_log2 = r.scale * kLog2e;
  p.n_qtiles = (int32_t)(((int64_t)r.max_q + kRRows - 1) / kRRows);
  p.level0 = 0;
  if (nope == 128) return rope == 64 ? ragged_launch<128, 64>(name, p, s) : ragged_launch<128, 32>(name, p, s);
  return rope == 64 ? ragged_launch<64, 64>(name, p, s) : ragged_launch<64, 32>(name, p, s);
}

// Exclusive sums of the sequences' kv lengths, one workgroup.
__global__ void __launch_bounds__(256) latent_sum_kernel(const int32_t* lens, int batch, int64_t span, int32_t* cu) {
  __shared__ int tmp[256];
  int base = 0;
  for (int c = 0; c < batch; c += 256) {
    const int b = c + threadIdx.x;
    const int v = b < batch ? (int)max((int64_t)0, min((int64_t)lens[b], span)) : 0;
    int total;
    const int before = block_exclusive_scan<256>(v, tmp, total);
    if (b < batch) cu[b] = base + before;
    base += total;
  }
  if (threadIdx.x == 0) cu[batch] = base;
}

int latent_sum_launch(const char* name, const int32_t* lens, int batch, int64_t span, int32_t* cu, hipStream_t s) {
  latent_sum_kernel<<<1, 256, 0, s>>>(lens, batch, span, cu);
  return launch_status(name);
}

}  // namespace pa

using namespace pa;

namespace {

constexpr size_t kGroupBytes = (size_t)2 << 30;  // K and V rows expanded at a time, one head's at least
// A bound of the kv lengths that makes one head's rows longer than this is the
// width of block tables rather than lengths (16.8 M tokens at Dn = 128 are 19 GB
// of cache a layer): the form with the smaller workspace runs.
constexpr size_t kHeadMost = (size_t)8 << 30;

size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

struct PrefillPlan {
  bool absorbed;
  size_t cu, q_lat, attn;  // bytes: running kv lengths, absorbed q (and as much of results), the attention's own
  size_t k_rope, kv;       // expanded rotary parts, K and V rows of `group` heads
  int32_t group;
  size_t need;
};

// Which form runs, by the operations of both with sequences of equal length:
// the absorbed form multiplies each (query, key) pair R + Dr and R wide, the
// expanded one Dn + Dr and Dn wide but expands every cached token first.
// Measured, absorbed against expanded, in us by the new tokens of a sequence:
// 8 sequences of 4 096 cached tokens by 32 heads (R = 512, Dn = 128; the rule
// changes behind 167 new tokens): 64: 196 / 447, 128: 373 / 463, 192: 559 / 484,
// 256: 751 / 495; 2 of 8 192 by 128 heads (168): 64: 341 / 820, 128: 682 / 851, 192:
// 988 / 873, 256: 1 310 / 936; 16 of 2 048 by 16 heads (R = 256, Dn = 64; 83): 64:
// 86 / 94, 128: 153 / 100.
bool absorbed_form(int32_t batch, int32_t num_tokens, int32_t max_q, int32_t total_kv, int32_t latent, int32_t rope,
                   int32_t nope) {
  const double tokens = std::min((double)num_tokens, (double)batch * max_q);
  const double kv = (double)total_kv / batch, q = std::min(tokens / batch, kv);
  const double pairs = tokens * (kv - q / 2);
  const double product = 2. * nope * latent;
  return pairs * (2 * latent + rope) + tokens * product < pairs * (2 * nope + rope) + total_kv * product;
}

int plan(const char* name, int32_t batch, int32_t num_tokens, int32_t max_q, int32_t total_kv, int32_t pages_per_seq,
         int32_t page_size, int32_t heads, int32_t latent, int32_t rope, int32_t nope, PrefillPlan& p) {
  p = PrefillPlan{};
  max_q = std::min(max_q, num_tokens);
  p.absorbed = absorbed_form(batch, num_tokens, max_q, total_kv, latent, rope, nope);
  p.cu = up256(4 * ((size_t)batch + 1));
  const size_t head = (size_t)total_kv * 2 * nope * 2;
  size_t g = head ? kGroupBytes / head : heads;
  if (g >= 8) g &= ~(size_t)7;
  g = std::min<size_t>(g, (size_t)std::max<int64_t>(1, kRGrid / batch));
  p.group = (int32_t)std::max<size_t>(1, std::min<size_t>(g, heads));
  p.k_rope = up256((size_t)total_kv * rope * 2);
  p.kv = up256(head * p.group);
  p.need = p.cu + p.k_rope + p.kv;
  if (!p.absorbed && head <= kHeadMost) return PA_OK;
  const char* why;
  p.attn = latent_attn_workspace(batch, max_q, heads, latent, (int64_t)pages_per_seq * page_size, &why);
  p.q_lat = up256((size_t)num_tokens * heads * latent * 2);
  const size_t need = 2 * p.q_lat + p.attn;
  if (!p.absorbed) p.absorbed = need < p.need;
  if (why) p.absorbed = false;  // sizes past the absorbed kernel's: the expanded form takes them
  if (p.absorbed) p.need = need;
  (void)name;
  return PA_OK;
}

bool prefill_sizes_ok(int32_t batch, int32_t num_tokens, int32_t max_q, int32_t total_kv, int32_t pages_per_seq,
                      int32_t page_size, int32_t heads, int32_t latent, int32_t rope, int32_t nope) {
  return batch > 0 && num_tokens >= 0 && max_q >= 0 && total_kv >= 0 && pages_per_seq >= 0 && page_size > 0 &&
         heads > 0 && latent_dims_ok(latent, rope) && latent_head_ok(nope, nope);
}

}  // namespace

extern "C" int pa_latent_prefill_route(int32_t batch, int32_t num_tokens, int32_t max_seqlen_q, int32_t total_kv,
                                       int32_t pages_per_seq, int32_t page_size, int32_t num_heads,
                                       int32_t latent_dim, int32_t rope_dim, int32_t nope_dim) {
  if (!prefill_sizes_ok(batch, num_tokens, max_seqlen_q, total_kv, pages_per_seq, page_size, num_heads, latent_dim,
                        rope_dim, nope_dim))
    return fail(PA_ERR_INVALID_ARGUMENT, "pa_latent_prefill_route: bad sizes");
  PrefillPlan p;
  plan("", batch, num_tokens, max_seqlen_q, total_kv, pages_per_seq, page_size, num_heads, latent_dim, rope_dim,
       nope_dim, p);
  return p.absorbed ? PA_LATENT_ABSORBED : PA_LATENT_EXPANDED;
}

extern "C" size_t pa_latent_prefill_workspace_size(int32_t batch, int32_t num_tokens, int32_t max_seqlen_q,
                                                   int32_t total_kv, int32_t pages_per_seq, int32_t page_size,
                                                   int32_t num_heads, int32_t latent_dim, int32_t rope_dim,
                                                   int32_t nope_dim) {
  if (!prefill_sizes_ok(batch, num_tokens, max_seqlen_q, total_kv, pages_per_seq, page_size, num_heads, latent_dim,
                        rope_dim, nope_dim))
    return 0;
  PrefillPlan p;
  plan("", batch, num_tokens, max_seqlen_q, total_kv, pages_per_seq, page_size, num_heads, latent_dim, rope_dim,
       nope_dim, p);
  return p.need;
}

extern "C" int pa_latent_prefill(const uint16_t* q_nope, int64_t qn_tok_stride, int64_t qn_head_stride,
                                 const uint16_t* q_rope, int64_t qr_tok_stride, int64_t qr_head_stride,
                                 const uint16_t* cache, int32_t num_pages, int32_t page_size, int64_t page_stride,
                                 int64_t slot_stride, const int32_t* block_tables, int64_t bt_stride,
                                 int32_t pages_per_seq, const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k,
                                 const int32_t* kv_lens, int32_t batch, int32_t num_tokens, int32_t max_seqlen_q,
                                 int32_t total_kv, int32_t num_heads, int32_t latent_dim, int32_t rope_dim,
                                 int32_t nope_dim, int32_t v_dim, const uint16_t* w_uk_t, const uint16_t* w_kv,
                                 float scale, int32_t zero_rest, uint16_t* out, int64_t out_tok_stride,
                                 int64_t out_head_stride, void* workspace, size_t workspace_bytes, void* stream) {
  const char* name = "pa_latent_prefill";
  if (batch < 0 || num_tokens < 0 || max_seqlen_q < 0 || total_kv < 0 || num_heads <= 0 || num_pages <= 0 ||
      page_size <= 0 || pages_per_seq < 0)
    return fail(PA_ERR_INVALID_ARGUMENT, "%s: bad sizes (batch=%d, num_tokens=%d, max_seqlen_q=%d, total_kv=%d, "
                "num_heads=%d, num_pages=%d, page_size=%d, pages_per_seq=%d)", name, batch, num_tokens, max_seqlen_q,
                total_kv, num_heads, num_pages, page_size, pages_per_seq);
  if (!latent_dims_ok(latent_dim, rope_dim) || !latent_head_ok(nope_dim, v_dim))
    return fail(PA_ERR_UNSUPPORTED, "%s: latent_dim %d, rope_dim %d, nope_dim %d, v_dim %d not supported", name,
                latent_dim, rope_dim, nope_dim, v_dim);
  if (num_heads > 65535) return fail(PA_ERR_UNSUPPORTED, "%s: %d heads", name, num_heads);
  if (!(scale > 0.f) || !(scale < INFINITY)) return fail(PA_ERR_INVALID_ARGUMENT, "%s: scale must be positive", name);
  if (batch > 0 && !!cu_seqlens_k == !!kv_lens)
    return fail(PA_ERR_INVALID_ARGUMENT, "%s: one of cu_seqlens_k and kv_lens", name);
  if (num_tokens == 0 || (batch == 0 && !zero_rest)) return PA_OK;
  if (!q_nope || !q_rope || !cache || !w_uk_t || !w_kv || !out ||
      (batch > 0 && (!cu_seqlens_q || (pages_per_seq && !block_tables))))
    return fail(PA_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
  const uintptr_t align = (uintptr_t)q_nope | (uintptr_t)q_rope | (uintptr_t)cache | (uintptr_t)w_uk_t |
                          (uintptr_t)w_kv | (uintptr_t)out | (uintptr_t)workspace;
  if ((align & 15u) || (qn_tok_stride | qn_head_stride | qr_tok_stride | qr_head_stride | page_stride | slot_stride |
                        out_tok_stride | out_head_stride) % 8)
    return fail(PA_ERR_UNSUPPORTED, "%s: operands must be 16-byte aligned with strides multiple of 8", name);
  hipStream_t s = (hipStream_t)stream;
  max_seqlen_q = std::min(max_seqlen_q, num_tokens);
  LatentRagged r;
  r.q_nope = q_nope;
  r.qn_ts = qn_tok_stride;
  r.qn_hs = qn_head_stride;
  r.q_rope = q_rope;
  r.qr_ts = qr_tok_stride;
  r.qr_hs = qr_head_stride;
  r.cu_q = cu_seqlens_q;
  r.batch = batch;
  r.num_tokens = num_tokens;
  r.max_q = max_seqlen_q;
  r.scale = scale;
  r.o_ts = out_tok_stride;
  r.o_hs = out_head_stride;
  r.zero_out = zero_rest ? out : nullptr;
  r.zero_heads = num_heads;
  const int64_t span = std::min<int64_t>((int64_t)pages_per_seq * page_size, 0x7fffffff);
  if (batch == 0 || max_seqlen_q == 0) {  // no rows but those to be zeroed
    r.batch = 0;
    r.heads = 1;
    r.max_q = 0;
    r.kv = r.k_rope = nullptr;
    r.cu_k = nullptr;
    r.cap = r.span = 0;
    r.out = out;
    return latent_ragged_launch(name, r, nope_dim, rope_dim, s);
  }
  PrefillPlan pl;
  if (int rc = plan(name, batch, num_tokens, max_seqlen_q, total_kv, pages_per_seq, page_size, num_heads, latent_dim,
                    rope_dim, nope_dim, pl))
    return rc;
  if (!workspace || workspace_bytes < pl.need)
    return fail(PA_ERR_WORKSPACE, "%s: workspace of %zu bytes given, %zu needed", name, workspace_bytes, pl.need);
  const LatentPool pool{cache, num_pages, magic_div((uint32_t)page_size), page_stride, slot_stride,
                        block_tables, bt_stride, pages_per_seq};
  char* ws = (char*)workspace;
  const int64_t head_w = (int64_t)(nope_dim + v_dim) * latent_dim;
  if (pl.absorbed) {
    uint16_t* q_lat = (uint16_t*)ws;
    uint16_t* o_lat = (uint16_t*)(ws + pl.q_lat);
    HeadProduct hp;
    hp.x = q_nope;
    hp.x_ts = qn_tok_stride;
    hp.x_hs = qn_head_stride;
    hp.w = w_uk_t;
    hp.w_hs = (int64_t)latent_dim * nope_dim;
    hp.y = q_lat;
    hp.y_ts = (int64_t)num_heads * latent_dim;
    hp.y_hs = latent_dim;
    hp.tokens = num_tokens;
    hp.heads = num_heads;
    hp.n = latent_dim;
    hp.k = nope_dim;
    if (int rc = head_product_launch(name, hp, s)) return rc;
    LatentAttn a;
    a.q_lat = q_lat;
    a.ql_ts = hp.y_ts;
    a.ql_hs = hp.y_hs;
    a.q_rope = q_rope;
    a.qr_ts = qr_tok_stride;
    a.qr_hs = qr_head_stride;
    a.pool = pool;
    a.cu_q = cu_seqlens_q;
    a.cu_k = cu_seqlens_k;
    a.kv_lens = kv_lens;
    a.batch = batch;
    a.num_tokens = num_tokens;
    a.heads = num_heads;
    a.max_q = max_seqlen_q;
    a.scale = scale;
    a.out = o_lat;
    a.o_ts = a.ql_ts;
    a.o_hs = a.ql_hs;
    if (int rc = latent_attn_launch(name, a, latent_dim, rope_dim, ws + 2 * pl.q_lat, s)) return rc;
    hp.x = o_lat;
    hp.x_ts = a.o_ts;
    hp.x_hs = a.o_hs;
    hp.w = w_kv + (int64_t)nope_dim * latent_dim;
    hp.w_hs = head_w;
    hp.y = out;
    hp.y_ts = out_tok_stride;
    hp.y_hs = out_head_stride;
    hp.n = v_dim;
    hp.k = latent_dim;
    hp.cu_q = cu_seqlens_q;
    hp.batch = batch;
    hp.max_q = max_seqlen_q;
    hp.zero_rest = zero_rest != 0;
    return head_product_launch(name, hp, s);
  }
  const int32_t* cu_k = cu_seqlens_k;
  if (!cu_k) {
    int32_t* cu = (int32_t*)ws;
    if (int rc = latent_sum_launch(name, kv_lens, batch, span, cu, s)) return rc;
    cu_k = cu;
  }
  LatentExpand x;
  x.pool = pool;
  x.cu_k = cu_k;
  x.batch = batch;
  x.cap = total_kv;
  x.w_kv = w_kv;
  x.k_rope = (uint16_t*)(ws + pl.cu);
  x.kv = (uint16_t*)(ws + pl.cu + pl.k_rope);
  r.cu_k = cu_k;
  r.cap = total_kv;
  r.span = (int32_t)span;
  r.kv = x.kv;
  r.k_rope = x.k_rope;
  for (int32_t h0 = 0; h0 < num_heads; h0 += pl.group) {
    x.head0 = h0;
    x.heads = r.heads = std::min(pl.group, num_heads - h0);
    if (total_kv > 0 && pages_per_seq > 0)
      if (int rc = latent_expand_launch(name, x, latent_dim, rope_dim, nope_dim, s)) return rc;
    r.q_nope = q_nope + h0 * qn_head_stride;
    r.q_rope = q_rope + h0 * qr_head_stride;
    r.out = out + h0 * out_head_stride;
    if (int rc = latent_ragged_launch(name, r, nope_dim, rope_dim, s)) return rc;
    x.k_rope = nullptr;  // the rotary parts and the zeroed rows are done once
    r.zero_out = nullptr;
  }
  return PA_OK;
}
