// n / d for 0 <= n < 2^31 by a multiplication: with 2^(shift-1) < d <= 2^shift and mul =
// floor(2^32 (2^shift - d) / d) + 1, n / d = (hi32(n mul) + n) >> shift.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace tia {

struct Divisor {
  uint32_t d, mul, shift;
};
inline Divisor divisor(uint32_t d) {
  uint32_t shift = 0;
  while ((uint64_t(1) << shift) < d) ++shift;
  return {d, uint32_t(((uint64_t(1) << 32) * ((uint64_t(1) << shift) - d)) / d + 1), shift};
}
__device__ __forceinline__ int div_by(int n, Divisor v) {
  return int((uint64_t(__umulhi(uint32_t(n), v.mul)) + uint32_t(n)) >> v.shift);
}

}  // namespace tia
