// Division of 31-bit indexes by a divisor fixed per launch. Plain C++ and device code.
#pragma once

#include <cstdint>

#if defined(__HIPCC__)
#define TQT_HOST_DEVICE __host__ __device__
#else
#define TQT_HOST_DEVICE
#endif

namespace tqt {

// n / d for n < 2^31, 1 <= d < 2^31, as n * m >> (31 + l) with l = ceil(log2 d), m = floor(2^(31 + l) / d) + 1:
// m / 2^(31 + l) exceeds 1 / d by at most 2^-(31 + l), so the product exceeds n / d by less than 2^-l <= 1 / d,
// which reaches no next integer. m < 2^32, as d > 2^(l - 1) (d = 1: m = 2^31 + 1).
struct FastDiv
{
    uint32_t d, m, shift;
};

inline FastDiv make_fast_div(uint32_t d)
{
    uint32_t l = 0;
    while ((1ull << l) < d) {
        ++l;
    }
    return {d, static_cast<uint32_t>((1ull << (31 + l)) / d + 1), 31 + l};
}

TQT_HOST_DEVICE inline uint32_t fast_div(uint32_t n, FastDiv f)
{
    return static_cast<uint32_t>((static_cast<uint64_t>(n) * f.m) >> f.shift);
}

TQT_HOST_DEVICE inline uint32_t fast_div(uint32_t n, FastDiv f, uint32_t &rest)
{
    const uint32_t q = fast_div(n, f);
    rest = n - q * f.d;
    return q;
}

}  // namespace tqt
