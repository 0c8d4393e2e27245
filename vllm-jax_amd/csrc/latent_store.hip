// Latent store for gfx950: RMSNorm of the new tokens' latent rows, rotation of
// their shared key part and of q's rotary part, and the paged write, in one
// pass over the new tokens.
//
//   cache[slot] = [ c * w / sqrt(mean(c^2) + eps) | rope(k) ],   q_out = rope(q)
//
// One workgroup per token.  Wave 0 owns the latent row, eight elements a lane
// (R <= 512), and sums its squares across the wave; the other threads
// rotate the key part and q's heads, whose cos and sin every workgroup
// evaluates once into LDS.  Everything is read once and written once; the
// squares' sum and the rotation are float32, each result rounded to bf16 once.
//
// HBM bound: 8 prompts of 1 024-3 000 tokens, 64 heads, R = 512, Dr = 64 (314 MB)
// take 70 us, 4.5 TB/s.  A workgroup a token keeps the angles' float64 products
// at one set a token; they pass under the rows' loads.  A decode step's four
// tokens take 4 us, 13 us with the host's part.
#include <algorithm>

#include "pa_errors.h"
#include "../../include/latent_attention.h"
#include "latent.h"
#include "rotary.h"

namespace pa {
namespace {

struct LatentStoreParams {
  const uint16_t* c;
  int64_t c_ts;
  const uint16_t* k;
  int64_t k_ts;
  const uint16_t* w;  // may be null: rows are stored as they come
  float eps;
  const double* inv_freq;
  float amp;
  const int32_t* positions;
  const int32_t* slots;
  int32_t heads;  // 0: no q
  const uint16_t* q;
  int64_t q_ts, q_hs;
  uint16_t* q_out;
  int64_t qo_ts, qo_hs;
  uint16_t* cache;
  int64_t num_slots;
  int32_t page_size;
  int64_t page_stride, slot_stride;
  int32_t latent;
};

template <int kRope, bool kInter>
__global__ void __launch_bounds__(256) latent_store_kernel(LatentStoreParams p) {
  constexpr int kPairs = kRope / 2;
  constexpr int kUnits = kInter ? kRope / 8 : kPairs / 8;  // pieces of a rotated row
  __shared__ float cs[kPairs], sn[kPairs];
  const int64_t t = blockIdx.x;
  const int tid = threadIdx.x, nthr = blockDim.x;
  const int total = (p.heads + 1) * kUnits;  // row 0: the key part
  const int64_t slot = p.slots[t];
  const bool store = slot >= 0 && slot < p.num_slots;
  uint16_t* row = p.cache;
  if (store) {
    const int64_t pg = slot / p.page_size;
    row += pg * p.page_stride + (slot - pg * p.page_size) * p.slot_stride;
  }
  auto src_of = [&](int u) -> const uint16_t* {
    const int h = u / kUnits - 1;
    return (h < 0 ? p.k + t * p.k_ts : p.q + t * p.q_ts + h * p.q_hs) + (u % kUnits) * 8;
  };
  auto dst_of = [&](int u) -> uint16_t* {
    const int h = u / kUnits - 1;
    return (h < 0 ? row + p.latent : p.q_out + t * p.qo_ts + h * p.qo_hs) + (u % kUnits) * 8;
  };
  // first pieces in flight before the angles are evaluated
  u32x4 a = {}, b = {};
  int u = tid;
  if (u < total) {
    a = ld16(src_of(u));
    if (!kInter) b = ld16(src_of(u) + kPairs);
  }
  const bool norm_wave = tid < 64;
  u32x4 cv = {}, wv = {};
  const int c8 = 8 * tid;
  if (norm_wave && c8 < p.latent) {
    cv = ld16(p.c + t * p.c_ts + c8);
    if (p.w) wv = ld16(p.w + c8);
  }
  for (int i = tid; i < kPairs; i += nthr) rot_angle(p.inv_freq[i], p.positions[t], p.amp, cs[i], sn[i]);
  __syncthreads();
  if (norm_wave && store) {
    if (p.w) {
      float x[8], w[8];
      RotVec<uint16_t>::load(cv, x);
      RotVec<uint16_t>::load(wv, w);
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = __builtin_fmaf(x[e], x[e], ss);
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) ss += __shfl_xor(ss, o);
      const float rs = 1.f / sqrtf(ss / (float)p.latent + p.eps);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = x[e] * rs * w[e];
      cv = RotVec<uint16_t>::store(x);
    }
    if (c8 < p.latent) st16(row + c8, cv);
  }
  while (u < total) {
    // the next piece's loads go out before this one is stored (its rows are
    // other rows, also in place)
    const int nu = u + nthr;
    u32x4 na = {}, nb = {};
    if (nu < total) {
      na = ld16(src_of(nu));
      if (!kInter) nb = ld16(src_of(nu) + kPairs);
    }
    if (u >= kUnits || store) {
      uint16_t* dst = dst_of(u);
      if constexpr (kInter) {
        a = rot_inter<uint16_t>(a, cs, sn, (u % kUnits) * 4);
      } else {
        rot_half<uint16_t>(a, b, cs, sn, (u % kUnits) * 8);
        st16(dst + kPairs, b);
      }
      st16(dst, a);
    }
    a = na;
    b = nb;
    u = nu;
  }
}

}  // namespace
}  // namespace pa

using namespace pa;

extern "C" int pa_latent_store(const uint16_t* latent, int64_t latent_tok_stride, const uint16_t* k_rope,
                               int64_t k_rope_tok_stride, const uint16_t* norm_weight, float eps,
                               const double* inv_freq, float amplitude, int32_t interleaved,
                               const int32_t* positions, const int32_t* slot_mapping, int32_t num_tokens,
                               int32_t latent_dim, int32_t rope_dim, const uint16_t* q_rope, int64_t q_tok_stride,
                               int64_t q_head_stride, int32_t num_heads, uint16_t* q_out, int64_t q_out_tok_stride,
                               int64_t q_out_head_stride, uint16_t* cache, int32_t num_pages, int32_t page_size,
                               int64_t page_stride, int64_t slot_stride, void* stream) {
  const char* name = "pa_latent_store";
  if (num_tokens < 0 || num_heads < 0 || num_pages <= 0 || page_size <= 0)
    return fail(PA_ERR_INVALID_ARGUMENT, "%s: bad sizes (num_tokens=%d, num_heads=%d, num_pages=%d, page_size=%d)",
                name, num_tokens, num_heads, num_pages, page_size);
  if (!latent_dims_ok(latent_dim, rope_dim))
    return fail(PA_ERR_UNSUPPORTED, "%s: latent_dim %d with rope_dim %d not supported (256 or 512 with 32 or 64)",
                name, latent_dim, rope_dim);
  if (!(eps >= 0.f)) return fail(PA_ERR_INVALID_ARGUMENT, "%s: bad eps", name);
  if (num_heads > (1 << 20)) return fail(PA_ERR_UNSUPPORTED, "%s: %d heads", name, num_heads);
  if (num_tokens == 0) return PA_OK;
  if (!latent || !k_rope || !inv_freq || !positions || !slot_mapping || !cache || (num_heads && (!q_rope || !q_out)))
    return fail(PA_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
  uintptr_t align = (uintptr_t)latent | (uintptr_t)k_rope | (uintptr_t)norm_weight | (uintptr_t)cache;
  int64_t strides = latent_tok_stride | k_rope_tok_stride | page_stride | slot_stride;
  if (num_heads) {
    align |= (uintptr_t)q_rope | (uintptr_t)q_out;
    strides |= q_tok_stride | q_head_stride | q_out_tok_stride | q_out_head_stride;
  }
  if ((align & 15u) || strides % 8)
    return fail(PA_ERR_UNSUPPORTED, "%s: operands must be 16-byte aligned with strides multiple of 8", name);
  // a row is read and written by one workgroup only where both lie alike
  if (num_heads && q_rope == q_out &&
      ((num_tokens > 1 && q_tok_stride != q_out_tok_stride) || (num_heads > 1 && q_head_stride != q_out_head_stride)))
    return fail(PA_ERR_INVALID_ARGUMENT, "%s: in place, q_rope and q_out must share strides", name);
  LatentStoreParams p;
  p.c = latent;
  p.c_ts = latent_tok_stride;
  p.k = k_rope;
  p.k_ts = k_rope_tok_stride;
  p.w = norm_weight;
  p.eps = eps;
  p.inv_freq = inv_freq;
  p.amp = amplitude;
  p.positions = positions;
  p.slots = slot_mapping;
  p.heads = num_heads;
  p.q = q_rope;
  p.q_ts = q_tok_stride;
  p.q_hs = q_head_stride;
  p.q_out = q_out;
  p.qo_ts = q_out_tok_stride;
  p.qo_hs = q_out_head_stride;
  p.cache = cache;
  p.num_slots = (int64_t)num_pages * page_size;
  p.page_size = page_size;
  p.page_stride = page_stride;
  p.slot_stride = slot_stride;
  p.latent = latent_dim;
  const bool inter = interleaved != 0;
  const int units = (num_heads + 1) * (inter ? rope_dim / 8 : rope_dim / 16);
  const unsigned threads = units <= 64 ? 64 : (units <= 128 ? 128 : 256);
  void (*kernel)(LatentStoreParams) = rope_dim == 64
      ? (inter ? latent_store_kernel<64, true> : latent_store_kernel<64, false>)
      : (inter ? latent_store_kernel<32, true> : latent_store_kernel<32, false>);
  // a grid has fewer than 2^32 threads along x
  constexpr int64_t kTokens = 1 << 23;
  for (int64_t t0 = 0; t0 < num_tokens; t0 += kTokens) {
    kernel<<<dim3((unsigned)std::min(num_tokens - t0, kTokens)), dim3(threads), 0, (hipStream_t)stream>>>(p);
    if (int rc = launch_status(name)) return rc;
    p.c += kTokens * p.c_ts;
    p.k += kTokens * p.k_ts;
    p.positions += kTokens;
    p.slots += kTokens;
    if (num_heads) {
      p.q += kTokens * p.q_ts;
      p.q_out += kTokens * p.qo_ts;
    }
  }
  return PA_OK;
}
