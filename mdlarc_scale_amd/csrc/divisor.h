// Division of whole numbers by a divisor that a launch knows.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mdl {

// n / d for 0 <= n < 2^31 as (n m) >> s, m = ceil(2^s / d), s = 31 + ceil(log2 d): m d exceeds 2^s
// by less than d <= 2^(s - 31), so n of them by less than 2^s.  A block's place takes four
// divisions by numbers of the launch, some 200 cycles each the usual way.
struct Divisor {
  uint32_t m, s;
};

inline Divisor divisor(uint32_t d) {
  uint32_t s = 31;
  while ((uint64_t{1} << (s - 31)) < d) ++s;
  return {static_cast<uint32_t>(((uint64_t{1} << s) + d - 1) / d), s};
}

__device__ __forceinline__ int quotient(int n, Divisor d) {
  return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(n)) * d.m) >> d.s);
}

}  // namespace mdl
