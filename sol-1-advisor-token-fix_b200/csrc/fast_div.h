// fast_div.h — division by a number that the host knows.
#pragma once
#include <cstdint>

namespace attn_bwd {

// Division by a number known to the host, exact for 0 <= n < 2^31: with 2^shift >= d the
// multiplier ceil(2^(32 + shift) / d) has 33 bits, of which mul holds the lower 32.
struct FastDiv {
  uint32_t mul, shift, d;
  __device__ __forceinline__ int div(int n) const {
    if (d == 1) return n;
    const uint32_t h = __umulhi(uint32_t(n), mul);
    return int((h + ((uint32_t(n) - h) >> 1)) >> (shift - 1));
  }
};

inline FastDiv fast_div(int d) {   // d >= 1
  FastDiv f;
  f.d = uint32_t(d);
  f.shift = 1;
  while ((1u << f.shift) < uint32_t(d)) ++f.shift;
  f.mul = uint32_t((((1ull << f.shift) - uint64_t(d)) << 32) / uint64_t(d) + 1);
  return f;
}

}  // namespace attn_bwd
