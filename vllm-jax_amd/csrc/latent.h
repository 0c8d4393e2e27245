// What the kernels of the latent-attention path share: sizes, page lookup.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "magic_div.h"
#include "pa_common.h"

namespace pa {

// Latent and rotary sizes the kernels are built for.
inline bool latent_dims_ok(int latent, int rope) {
  return (latent == 256 || latent == 512) && (rope == 32 || rope == 64);
}
// Sizes of a head's unrotated key part and of its values (one size for both).
inline bool latent_head_ok(int nope, int v) { return (nope == 64 || nope == 128) && v == nope; }

// Pool of latent rows: row (page, slot) is `latent` normalised elements, then
// the rotated key part.
struct LatentPool {
  const uint16_t* cache;
  int32_t num_pages;
  MagicDiv page;  // page size
  int64_t page_stride, slot_stride;
  const int32_t* tables;
  int64_t bt_stride;
  int32_t pages_per_seq;
};

// kv length that a block-table row can hold, for a length read from the device.
__device__ __forceinline__ int latent_kv_len(const LatentPool& p, int len) {
  const int64_t span = (int64_t)p.pages_per_seq * p.page.d;
  return len < 0 ? 0 : (int)min((int64_t)len, span);
}

}  // namespace pa
