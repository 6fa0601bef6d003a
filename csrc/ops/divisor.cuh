// Division by a number that the host knows, as one multiplication.
#pragma once

#include <cuda_runtime.h>

namespace mccl {
namespace ops {

// n / d for n < 2^31: with 2^s < d <= 2^(s + 1) and m = ceil(2^(32 + s) / d), m d exceeds 2^(32 + s) by less than 2^(s + 1).
struct Divisor {
  unsigned d, m, s;
  __host__ explicit Divisor(unsigned by = 1) : d(by), m(0), s(0) {
    while ((2ull << s) < by) ++s;
    if (by > 1) m = static_cast<unsigned>(((1ull << (32 + s)) + by - 1) / by);
  }
  __device__ __forceinline__ unsigned of(unsigned n) const { return m == 0 ? n : __umulhi(n, m) >> s; }
};

}  // namespace ops
}  // namespace mccl
