// Division of an int that is not negative by a number the host knows.
#pragma once

#include <stdint.h>

namespace b200 {

// n / d for n below 2^31, by a product: mul = floor(2^32 (2^shift - d) / d) + 1 with
// 2^shift >= d gives floor((n mul / 2^32 + n) / 2^shift) (Granlund and Montgomery).
struct Divisor {
  uint32_t mul;
  int d, shift;
  __device__ __forceinline__ int of(int n) const {
    return (int)((__umulhi(mul, (uint32_t)n) + (uint32_t)n) >> shift);
  }
};
inline Divisor divisor(int d) {
  Divisor r;
  r.d = d;
  r.shift = 0;
  while ((1ll << r.shift) < d) ++r.shift;
  r.mul = (uint32_t)(((1ull << 32) * ((1ull << r.shift) - (unsigned long long)d)) / d + 1);
  return r;
}

}  // namespace b200
