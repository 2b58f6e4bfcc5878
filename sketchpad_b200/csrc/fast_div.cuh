// fast_div.cuh -- division by a launch's constant.
#pragma once
#include <stdint.h>

namespace sp {

// Division of a non-negative int32 by a fixed divisor d >= 1: n / d = (n * mul) >> 32 >> shift
// with mul = ceil(2^(32 + shift) / d), shift = ceil(log2 d) - 1 (exact for n < 2^31: the
// round-up method of Granlund and Montgomery); d = 1 has mul = 0.
struct FastDiv {
  uint32_t mul, shift;
  int32_t d;
  __device__ __forceinline__ int32_t div(int32_t n) const {
    return mul ? (int32_t)(__umulhi((uint32_t)n, mul) >> shift) : n;
  }
};
inline FastDiv make_fast_div(int32_t d) {
  FastDiv f{0, 0, d};
  if (d <= 1) return f;
  uint32_t l = 0;
  while ((1ll << l) < d) ++l;  // ceil(log2 d) >= 1
  f.shift = l - 1;
  f.mul = (uint32_t)(((1ull << (31 + l)) + (uint64_t)d - 1) / (uint64_t)d);
  return f;
}

}  // namespace sp
