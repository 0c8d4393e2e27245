// Exact quotients by a divisor that the host knows.
//
// Numbers below 2^31 by a divisor of 1 .. 2^31 - 1: with l = ceil(log2 d) and
// m = ceil(2^(31 + l) / d) < 2^32 the quotient is (x * m) >> (31 + l), exactly
// (m d - 2^(31 + l) < d <= 2^l).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace pa {

struct MagicDiv {
  uint32_t d, m, shift;
};
inline MagicDiv magic_div(uint32_t d) {
  uint32_t l = 0;
  while ((1ull << l) < d) ++l;
  MagicDiv r;
  r.d = d;
  if (l == 0) {  // d == 1: (x * 2^31) >> 31
    r.m = 1u << 31;
    r.shift = 31;
    return r;
  }
  r.m = (uint32_t)(((1ull << (31 + l)) + d - 1) / d);
  r.shift = 31 + l;
  return r;
}
__host__ __device__ __forceinline__ uint32_t div_by(uint32_t x, const MagicDiv& v) {
  return (uint32_t)(((uint64_t)x * v.m) >> v.shift);
}

}  // namespace pa
