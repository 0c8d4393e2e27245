// rotary_embedding for gfx950: rotation of part of each head by the token's
// position, in interleaved pairs (2i, 2i + 1) or halves (i, i + r/2).
//
// A workgroup takes one token and a share of its heads: its threads put the
// cos and sin of the token's pairs into LDS (rot_angle: one float64 product a
// pair, once per workgroup and not per head) while their first rows are in
// flight, then rotate 16 bytes (halves: two times 16) each.  Everything is
// read once and written once; elements outside the rotated part are copied,
// and left alone in place.
//
// Rows whose 16-byte pieces would split a pair or be misaligned (odd head
// sizes, odd starts, odd strides) take the scalar kernel, one pair or element a
// thread: 403 us against 159 us for 16 384 tokens, 64 heads of 192 of which 64
// are rotated (bf16), so whatever can take 16-byte pieces does.
//
// HBM bound: those 159 us are 5.07 TB/s read and written, the rate of a large
// copy.  Small calls (64 tokens, 32 heads: 7.7 us) are the host's time.
#include <algorithm>

#include "magic_div.h"
#include "pa_errors.h"
#include "../../include/latent_attention.h"
#include "rotary.h"

namespace pa {
namespace {

struct RotaryParams {
  const void* x;
  int64_t x_ts, x_hs;
  void* out;
  int64_t o_ts, o_hs;
  const double* inv_freq;
  const int32_t* positions;
  int32_t heads, dim, start, pairs, units;  // units: pieces of a head a thread takes one at a time
  MagicDiv per_head;                        // by units
  float amp;
};

constexpr int kRotThreads = 256;
constexpr int kRotInFlight = 2;  // pieces a thread has in flight
constexpr int64_t kRotTokens = 1 << 23;  // tokens of a launch: a grid has fewer than 2^32 threads along x

__device__ __forceinline__ void rot_table(const RotaryParams& p, int64_t t, float* cs, float* sn) {
  const int32_t pos = p.positions[t];
  for (int i = threadIdx.x; i < p.pairs; i += kRotThreads) rot_angle(p.inv_freq[i], pos, p.amp, cs[i], sn[i]);
}

template <typename T, bool kInter>
__global__ void __launch_bounds__(kRotThreads) rotary_vec_kernel(RotaryParams p) {
  using V = RotVec<T>;
  __shared__ float cs[kRotMaxPairs], sn[kRotMaxPairs];
  const int64_t t = blockIdx.x;
  const T* xt = (const T*)p.x + t * p.x_ts;
  T* ot = (T*)p.out + t * p.o_ts;
  const int rot_units = kInter ? 2 * p.pairs / V::kN : p.pairs / V::kN;
  const int total = p.heads * p.units;
  const int first = blockIdx.y * (kRotThreads * kRotInFlight) + threadIdx.x;
  u32x4 a[kRotInFlight], b[kRotInFlight];
  int head[kRotInFlight], piece[kRotInFlight];
  // element offset of a piece inside its head; pieces past the rotated ones
  // are those before `start`, then those behind the rotated part
  auto offset = [&](int u) {
    if (u < rot_units) return p.start + u * V::kN;
    const int e = (u - rot_units) * V::kN;
    return e < p.start ? e : e + 2 * p.pairs;
  };
#pragma unroll
  for (int i = 0; i < kRotInFlight; ++i) {
    const int u = first + i * kRotThreads;
    if (u < total) {
      head[i] = (int)div_by((uint32_t)u, p.per_head);
      piece[i] = u - head[i] * p.units;
      const T* src = xt + head[i] * p.x_hs + offset(piece[i]);
      a[i] = ld16(src);
      if (!kInter && piece[i] < rot_units) b[i] = ld16(src + p.pairs);
    }
  }
  rot_table(p, t, cs, sn);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kRotInFlight; ++i) {
    const int u = first + i * kRotThreads;
    if (u >= total) continue;
    T* dst = ot + head[i] * p.o_hs + offset(piece[i]);
    if (piece[i] < rot_units) {
      if constexpr (kInter) {
        a[i] = rot_inter<T>(a[i], cs, sn, piece[i] * (V::kN / 2));
      } else {
        rot_half<T>(a[i], b[i], cs, sn, piece[i] * V::kN);
        st16(dst + p.pairs, b[i]);
      }
    }
    st16(dst, a[i]);
  }
}

// One pair, or one element outside the rotated part, a thread.
template <typename T, bool kInter>
__global__ void __launch_bounds__(kRotThreads) rotary_scalar_kernel(RotaryParams p) {
  using V = RotVec<T>;
  __shared__ float cs[kRotMaxPairs], sn[kRotMaxPairs];
  const int64_t t = blockIdx.x;
  const T* xt = (const T*)p.x + t * p.x_ts;
  T* ot = (T*)p.out + t * p.o_ts;
  rot_table(p, t, cs, sn);
  __syncthreads();
  const int total = p.heads * p.units;
  for (int u = blockIdx.y * kRotThreads + threadIdx.x; u < total; u += gridDim.y * kRotThreads) {
    const int h = u / p.units, i = u - h * p.units;
    const T* src = xt + h * p.x_hs;
    T* dst = ot + h * p.o_hs;
    if (i < p.pairs) {
      const int ia = p.start + (kInter ? 2 * i : i), ib = ia + (kInter ? 1 : p.pairs);
      const float x = V::get(src[ia]), y = V::get(src[ib]), c = cs[i], s = sn[i];
      dst[ia] = V::put(x * c - y * s);
      dst[ib] = V::put(x * s + y * c);
    } else {
      const int e = i - p.pairs < p.start ? i - p.pairs : i + p.pairs;
      dst[e] = src[e];
    }
  }
}

template <typename T>
int launch_tokens(RotaryParams p, int64_t tokens, int64_t parts, void (*kernel)(RotaryParams), hipStream_t s) {
  for (int64_t t0 = 0; t0 < tokens; t0 += kRotTokens) {
    const dim3 g((unsigned)std::min(tokens - t0, kRotTokens), (unsigned)parts);
    kernel<<<g, kRotThreads, 0, s>>>(p);
    if (int rc = launch_status("pa_rotary_embedding")) return rc;
    p.x = (const T*)p.x + kRotTokens * p.x_ts;
    p.out = (T*)p.out + kRotTokens * p.o_ts;
    p.positions += kRotTokens;
  }
  return PA_OK;
}

template <typename T>
int launch(const RotaryParams& prm, int64_t tokens, bool inter, bool in_place, hipStream_t s) {
  RotaryParams p = prm;
  constexpr int kN = RotVec<T>::kN;
  const int rot = 2 * p.pairs;
  const bool vec = (((uintptr_t)p.x | (uintptr_t)p.out) & 15) == 0 &&
                   (p.x_ts | p.x_hs | p.o_ts | p.o_hs | p.dim | p.start) % kN == 0 &&
                   (inter ? rot : p.pairs) % kN == 0;
  const int rest = in_place ? 0 : p.dim - rot;  // copied elements of a head
  if (vec) {
    p.units = (inter ? rot : p.pairs) / kN + rest / kN;
    p.per_head = magic_div((uint32_t)p.units);
    const int64_t parts = ((int64_t)p.heads * p.units + kRotThreads * kRotInFlight - 1) / (kRotThreads * kRotInFlight);
    return launch_tokens<T>(p, tokens, parts, inter ? rotary_vec_kernel<T, true> : rotary_vec_kernel<T, false>, s);
  } else {
    p.units = p.pairs + rest;
    const int64_t parts = ((int64_t)p.heads * p.units + kRotThreads * 8 - 1) / (kRotThreads * 8);
    return launch_tokens<T>(p, tokens, parts, inter ? rotary_scalar_kernel<T, true> : rotary_scalar_kernel<T, false>,
                            s);
  }
}

}  // namespace
}  // namespace pa

using namespace pa;

extern "C" int pa_rotary_embedding(int32_t dtype, const void* x, int64_t x_tok_stride, int64_t x_head_stride,
                                   const int32_t* positions, const double* inv_freq, float amplitude,
                                   int32_t num_tokens, int32_t num_heads, int32_t head_dim, int32_t start,
                                   int32_t rotary_dim, int32_t interleaved, void* out, int64_t out_tok_stride,
                                   int64_t out_head_stride, void* stream) {
  const char* name = "pa_rotary_embedding";
  if (num_tokens < 0 || num_heads <= 0 || head_dim <= 0)
    return fail(PA_ERR_INVALID_ARGUMENT, "%s: bad sizes (num_tokens=%d, num_heads=%d, head_dim=%d)", name, num_tokens,
                num_heads, head_dim);
  if (rotary_dim <= 0 || rotary_dim % 2 || start < 0 || (int64_t)start + rotary_dim > head_dim)
    return fail(PA_ERR_INVALID_ARGUMENT, "%s: rotated part [%d, %d + %d) is not an even part of a head of %d", name,
                start, start, rotary_dim, head_dim);
  if (rotary_dim > 2 * kRotMaxPairs)
    return fail(PA_ERR_UNSUPPORTED, "%s: rotary_dim %d is more than %d", name, rotary_dim, 2 * kRotMaxPairs);
  // a token's elements are counted in 32 bits, and the pieces in 16-bit grids
  if ((int64_t)num_heads * head_dim > (1 << 24))
    return fail(PA_ERR_UNSUPPORTED, "%s: %d heads of %d are more than 2^24 elements a token", name, num_heads,
                head_dim);
  if (dtype != PA_DTYPE_BF16 && dtype != PA_DTYPE_FP16 && dtype != PA_DTYPE_FP32)
    return fail(PA_ERR_UNSUPPORTED, "%s: dtype code %d", name, dtype);
  if (num_tokens == 0) return PA_OK;
  if (!x || !positions || !inv_freq || !out) return fail(PA_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
  const bool in_place = x == out;
  if (in_place && (x_tok_stride != out_tok_stride || x_head_stride != out_head_stride))
    return fail(PA_ERR_INVALID_ARGUMENT, "%s: in place, x and out must share strides", name);
  RotaryParams p;
  p.x = x;
  p.x_ts = x_tok_stride;
  p.x_hs = x_head_stride;
  p.out = out;
  p.o_ts = out_tok_stride;
  p.o_hs = out_head_stride;
  p.inv_freq = inv_freq;
  p.positions = positions;
  p.heads = num_heads;
  p.dim = head_dim;
  p.start = start;
  p.pairs = rotary_dim / 2;
  p.units = 0;
  p.per_head = MagicDiv{};
  p.amp = amplitude;
  const bool inter = interleaved != 0;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == PA_DTYPE_BF16) return launch<uint16_t>(p, num_tokens, inter, in_place, s);
  if (dtype == PA_DTYPE_FP16) return launch<_Float16>(p, num_tokens, inter, in_place, s);
  return launch<float>(p, num_tokens, inter, in_place, s);
}
