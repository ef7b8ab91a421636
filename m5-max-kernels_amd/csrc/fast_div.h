// Division by a number that the host knows.
#pragma once

#include "m5k_common.h"

namespace m5k {

// n / d of 0 <= n < 2^31 by one multiplication: magic = ceil(2^(31 + shift) / d), shift = ceil(log2 d).  The excess
// magic * d - 2^(31 + shift) is below d <= 2^shift, so n times it stays below 2^(31 + shift) and the quotient is exact.
__device__ __forceinline__ uint32_t fast_div(uint32_t n, uint32_t magic, uint32_t shift) {
  return __umulhi(2 * n, magic) >> shift;
}

inline void magic_of(uint32_t d, uint32_t& magic, uint32_t& shift) {
  shift = 0;
  while ((uint64_t{1} << shift) < d) ++shift;
  magic = static_cast<uint32_t>(((uint64_t{1} << (31 + shift)) + d - 1) / d);
}

}  // namespace m5k
