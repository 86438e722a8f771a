// Division by numbers that a launch knows: of x below 2^31 by one multiplication, where the compiler's takes
// some thirty dependent instructions. m = ceil(2^(32 + s) / d) with 2^s >= d (Granlund and Montgomery, division by
// invariant integers); m has 33 bits, of which the first is a plain add.
#pragma once

#include <stdint.h>

namespace h3sa {

struct Divisor {
  uint32_t d, m, s;
};
inline Divisor divisor(uint32_t d) {
  Divisor v;
  v.d = d;
  v.s = 0;
  while ((1ull << v.s) < d) ++v.s;
  v.m = static_cast<uint32_t>(((((1ull << v.s) - d) << 32) / d) + 1);
  return v;
}
__device__ __forceinline__ uint32_t quotient(uint32_t x, const Divisor& v) {
  return (__umulhi(x, v.m) + x) >> v.s;  // x below 2^31: the sum stays below 2^32
}
// x / d for x >= 0 and a power of two
__device__ __forceinline__ int over_pow2(int x, int d) { return x >> (31 - __clz(d)); }

}  // namespace h3sa
