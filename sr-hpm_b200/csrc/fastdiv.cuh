// Division of 32-bit numbers by a divisor that is fixed for a launch.
#pragma once
#include <cstdint>

namespace srhpm {

// n / d for 0 <= n < 2^31, d >= 1: one high product (d a power of two or not; the rounded-up reciprocal's error stays
// under 1 / d for every n < 2^31)
struct FastDiv {
    uint32_t mul, shr, d;
    static FastDiv of(uint32_t d) {
        FastDiv f{ 0, 0, d };
        while ((1ull << f.shr) < d) f.shr++;
        // 2^(31 + shr) / d rounded up: below 2^32, since 2^shr < 2 d
        f.mul = (uint32_t) (((1ull << (31 + f.shr)) + d - 1) / d);
        return f;
    }
    __device__ __forceinline__ int div(int n) const { return (int) (((uint64_t) (uint32_t) n * mul) >> (31 + shr)); }
};

}  // namespace srhpm
