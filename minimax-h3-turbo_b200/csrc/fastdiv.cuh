// Division by a number that is the same for a whole launch.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace h3b {

// n / d and n % d for 0 <= n < 2^31 by one multiplication (a division by a number the compiler does not know takes some
// dozens of instructions, on the path of every warp at every unit): q = (hi(n m) + n) >> l with l = ceil(log2 d),
// m = floor(2^32 (2^l - d) / d) + 1.
struct FastDiv {
  uint32_t d, m, l;
  __host__ void set(uint32_t v) {
    d = v;
    for (l = 0; l < 31 && (1u << l) < v; ++l) {
    }
    m = static_cast<uint32_t>((static_cast<uint64_t>(1) << 32) * ((static_cast<uint64_t>(1) << l) - v) / v + 1);
  }
  __device__ __forceinline__ int div(int n) const {
    return static_cast<int>((__umulhi(static_cast<uint32_t>(n), m) + static_cast<uint32_t>(n)) >> l);
  }
  __device__ __forceinline__ int divmod(int n, int& rem) const {
    const int q = div(n);
    rem = n - q * static_cast<int>(d);
    return q;
  }
};

}  // namespace h3b
