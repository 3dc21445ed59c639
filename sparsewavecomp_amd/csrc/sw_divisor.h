// Division by a number that the host knows.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace swd {

// Division of numbers below 2^31 by one that the host knows: n m / 2^(31 + s),
// m = 2^(31 + s) / d rounded up and s the logarithm of d rounded up.  m d passes
// 2^(31 + s) by less than d <= 2^s, which moves no quotient of such n.
struct Divisor {
  uint32_t by, factor, shift;
  Divisor() : by(1), factor(0), shift(0) {}
  explicit Divisor(uint32_t d) : by(d), factor(0), shift(0) {
    uint32_t s = 0;
    while (((uint64_t)1 << s) < d)
      ++s;
    if (s > 0) {
      factor = (uint32_t)((((uint64_t)1 << (31 + s)) + d - 1) / d);
      shift = s - 1;
    }
  }
  // (on the host too, where a test asks it)
  __host__ __device__ __forceinline__ uint32_t quotient(uint32_t n) const {
    return by == 1 ? n : (uint32_t)((uint64_t)n * factor >> 32) >> shift;
  }
};

} // namespace swd
