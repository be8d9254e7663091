// Integer division by numbers that are fixed for a launch.
#pragma once
#include <cstdint>

namespace srt {

// Division of a number below 2^31 by a divisor fixed on the host: floor(n / d) = umulhi(n, mul) >> shr with
// mul = ceil(2^(31 + ceil(log2 d)) / d) (Granlund-Montgomery); d = 1 is passed through.  The tile walk divides by
// five such numbers per tile, and a 32-bit hardware-less division is some thirty dependent instructions: about
// 600 cycles per tile on each role's path, which is most of what a tile costs when it has one or two k-blocks.
struct FastDiv {
    uint32_t mul, shr, d;
};

inline FastDiv make_fast_div(uint32_t d)
{
    FastDiv f = {0u, 0u, d == 0 ? 1u : d};
    if (f.d == 1) return f;
    uint32_t lg = 0;
    while ((1ull << lg) < f.d) ++lg;                       // ceil(log2 d)
    const uint32_t pw = 31 + lg;
    f.mul = static_cast<uint32_t>(((1ull << pw) + f.d - 1) / f.d);
    f.shr = pw - 32;
    return f;
}

__device__ __forceinline__ uint32_t fast_div(uint32_t n, const FastDiv& f)
{
    return f.d == 1 ? n : (__umulhi(n, f.mul) >> f.shr);
}

}  // namespace srt
