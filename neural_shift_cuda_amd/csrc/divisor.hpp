// divisor.hpp -- division by a number that a launch knows.
#pragma once

#include "nsh_common.hpp"

namespace nsh {

// Division of a number below 2^31 by a fixed one, d: with 2^(s-1) < d <= 2^s and
// m = ceil(2^(31+s) / d), the excess m d - 2^(31+s) < d <= 2^s keeps the quotient
// n m / 2^(31+s) below the next whole number.
struct Divisor {
    uint32_t m, shift;
    static Divisor of(uint32_t d) {
        uint32_t s = 0;
        while ((uint64_t(1) << s) < d) ++s;
        if (s == 0) return Divisor{0, 0};
        return Divisor{static_cast<uint32_t>(((uint64_t(1) << (31 + s)) + d - 1) / d), s - 1};
    }
    __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return m ? __umulhi(n, m) >> shift : n; }
};

}  // namespace nsh
