// n / d by a product with a rounded-up 2^32 / d, of which the upper half counts. Off by d · (2^32 / d) − 2^32 = e in its place, the product finds the quotient for all n with n · e < 2^32.
#pragma once
#include <cstdint>
#include <stdexcept>
#include <string>

namespace oxk {

// The factor for quotients n / d, 0 ≤ n ≤ most; 0 stands for 1. A pair that the product does not serve is an error.
inline unsigned by_of(int64_t d, int64_t most) {
    if (d <= 1) return 0u;
    const int64_t two32 = (int64_t)1 << 32, by = (two32 + d - 1) / d, e = by * d - two32;
    if (d >= two32 / 2 || most >= two32 / 2 || most * e >= two32)
        throw std::runtime_error("packed keys and values: a quotient of " + std::to_string(most) + " by " + std::to_string(d) + " is beyond what a product finds");
    return (unsigned)by;
}

}  // namespace oxk
