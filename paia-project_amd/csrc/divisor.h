// Division of small numbers by one that the host knows.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace paia {

// n / d for n < 2^31 as one multiplication: with s = ceil(log2 d) and m = ceil(2^(31+s) / d), m d exceeds 2^(31+s) by less
// than d <= 2^s, so floor(n m / 2^(31+s)) is the quotient; 2 n m >> 32 >> s in 32-bit operations.
struct Divisor {
    uint32_t m, s, d;
    explicit Divisor(uint32_t by = 1) : s(0), d(by)
    {
        while ((1ull << s) < by) ++s;
        m = (uint32_t)(((1ull << (31 + s)) + by - 1) / by);
    }
    __device__ __forceinline__ uint32_t of(uint32_t n) const { return __umulhi(2u * n, m) >> s; }
};

}  // namespace paia
