// Division by a number that a launch has from its caller.  Plain C++, so that it can be checked without a GPU.
#pragma once
#include <stdint.h>

namespace hspmm {

// n / d for n < 2^31 by a multiplication: with l = ceil(log2 d) and m = floor(2^(31 + l) / d) + 1, n m >> (31 + l) is the
// quotient (Granlund and Montgomery, "Division by Invariant Integers using Multiplication", 1994).
struct Divisor {
    uint32_t d, m, shift;
    static Divisor of(uint32_t d)
    {
        uint32_t l = 0;
        while (l < 31u && (1u << l) < d) ++l;
        return Divisor{d, uint32_t((uint64_t(1) << (31u + l)) / d + 1u), 31u + l};
    }
    constexpr uint32_t quotient(uint32_t n) const { return uint32_t((uint64_t(n) * m) >> shift); }
};

}  // namespace hspmm
