// Division by a number that the host knows, as a multiplication and a shift.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace odit {

// n / d for n below 2^31: n * mul >> shift with mul = 2^shift / d rounded up, shift = 31 + log2(d) rounded up; what the rounding adds stays
// below 1 / d
struct Quotient {
  uint32_t mul;
  int shift;
  __device__ __forceinline__ int operator()(int n) const { return static_cast<int>(static_cast<uint64_t>(static_cast<uint32_t>(n)) * mul >> shift); }
};
inline Quotient quotient(int d) {
  Quotient q{0, 31};
  while ((1ll << (q.shift - 31)) < d) ++q.shift;
  q.mul = static_cast<uint32_t>(((1ull << q.shift) + d - 1) / d);
  return q;
}

}  // namespace odit
