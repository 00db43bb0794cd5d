// Random bits for dropout: Philox-4x32 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011) with 7 rounds, the fewest
// for which its authors report no failure in BigCrush.  Nothing is stored: the bits of element i of a tensor are a function of the key and of i, so
// the backward pass makes them again.
//
// An element takes 16 bits, so a call serves the eight elements that a lane loads at once.  With 32 bits an element (two calls) dropout of bf16 would be
// bound by the multiplications, which run at a quarter of the rate; what 16 cost is that p is a multiple of 2^-16, and kept values are
// multiplied with the reciprocal of what is then kept on average.
#pragma once
#include "mi8_common.h"

namespace mi8 {

struct Dropout {
    uint64_t seed, offset;
    const int64_t* seed_on_device;  // null: seed
    uint32_t threshold;             // an element is kept where its 16 bits are at least this: 0 keeps all, 65536 none
    float factor;                   // of kept elements
};

__device__ __forceinline__ uint4 philox(uint64_t index, uint64_t offset, uint64_t key)
{
    uint32_t c0 = (uint32_t)index, c1 = (uint32_t)(index >> 32), c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
    uint32_t k0 = (uint32_t)key, k1 = (uint32_t)(key >> 32);
#pragma unroll
    for (int r = 0; r < 7; ++r) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
}

// Which of the elements first .. first + 7 of a tensor are kept, a bit each.
__device__ __forceinline__ uint32_t kept8(int64_t first, uint64_t offset, uint64_t key, uint32_t threshold)
{
    const uint64_t call = (uint64_t)first >> 3;
    const int skip = (int)(first & 7);
    auto bits = [&](uint4 w) __attribute__((always_inline)) {
        const uint32_t v[4] = {w.x, w.y, w.z, w.w};
        uint32_t m = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) m |= (uint32_t)((v[e] & 0xFFFFu) >= threshold) << (2 * e) | (uint32_t)((v[e] >> 16) >= threshold) << (2 * e + 1);
        return m;
    };
    uint32_t m = bits(philox(call, offset, key));
    if (skip) m = (m | bits(philox(call + 1, offset, key)) << 8) >> skip & 0xFFu;  // (the elements straddle two calls')
    return m;
}

}  // namespace mi8
