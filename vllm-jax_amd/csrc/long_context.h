// What the kernels over blocks of a long context share.
#pragma once

#include "pa_common.h"
#include "pa_errors.h"

namespace pa {

// Largest grid (x) of a launch, in workgroups of up to 1024 threads: a grid has
// fewer than 2^32 threads along x.
constexpr int64_t kMaxGrid = ((int64_t)1 << 22) - 1;

inline bool block_dim_ok(int32_t head_dim) { return head_dim == 64 || head_dim == 128 || head_dim == 256; }

// Tokens of a sequence: its length, inside the block table's span.
__device__ __forceinline__ int clamp_len(const int32_t* lengths, int b, int64_t span) {
  return (int)max((int64_t)0, min((int64_t)lengths[b], span));
}

// Maximum over the 16 lanes of a DPP row; every lane gets it.
template <int kCtrl>
__device__ __forceinline__ float max_dpp(float x) {
  return fmaxf(x, __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp((int)__float_as_uint(x),
                                                                        (int)__float_as_uint(x), kCtrl, 0xF, 0xF,
                                                                        false)));
}
__device__ __forceinline__ float max_row16(float x) {
  x = max_dpp<0xB1>(x);   // quad_perm(1, 0, 3, 2)
  x = max_dpp<0x4E>(x);   // quad_perm(2, 3, 0, 1)
  x = max_dpp<0x141>(x);  // row_half_mirror
  return max_dpp<0x140>(x);  // row_mirror
}

// Checks that the entries over blocks share; 0 or the failure's code.
inline int check_blocks(const char* name, int32_t num_pages, int32_t page_size, int32_t block, int32_t batch,
                        int32_t num_kv_heads, int32_t head_dim, int32_t pages_per_seq) {
  if (num_pages <= 0 || page_size <= 0 || batch < 0 || num_kv_heads <= 0 || pages_per_seq < 0)
    return fail(PA_ERR_INVALID_ARGUMENT, "%s: bad sizes (num_pages=%d, page_size=%d, batch=%d, num_kv_heads=%d, "
                "pages_per_seq=%d)", name, num_pages, page_size, batch, num_kv_heads, pages_per_seq);
  if (block <= 0 || block % 16 || page_size % block)
    return fail(PA_ERR_INVALID_ARGUMENT, "%s: block %d must be a multiple of 16 that divides the page size %d", name,
                block, page_size);
  if (!block_dim_ok(head_dim))
    return fail(PA_ERR_UNSUPPORTED, "%s: head_dim %d not supported (64, 128 or 256)", name, head_dim);
  if ((int64_t)pages_per_seq * page_size > 0x7fffffff)
    return fail(PA_ERR_UNSUPPORTED, "%s: block tables of %d pages span 2^31 tokens or more", name, pages_per_seq);
  return PA_OK;
}

}  // namespace pa
