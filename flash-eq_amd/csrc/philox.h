// Counter-based random numbers: Philox 4 x 32 with ten rounds (Salmon, Moraes, Dror and Shaw, "Parallel random
// numbers: as easy as 1, 2, 3", SC 2011).  The key is the seed; block b has the counter (b mod 2^32, b / 2^32, 0, 0), and
// its four words make eight numbers of 16 bits, the lower half of a word first.
//
// A unit of a tensor (an element, or an irrep of a channel) has number u mod 8 of block u / 8.  It is dropped where that is
// below limit = round(65536 p); what is kept is multiplied by 65536 / (65536 - limit), so the expectation is exact for the
// share that is dropped, which differs from p by at most 2^-17.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace feq {

// A dropout as the kernels take it.
struct Drop {
    const int64_t* seed;     // one number on the device
    uint32_t limit;          // 0: nothing is dropped, 65536: all
    float scale;
};

// p in [0, 1].
inline Drop make_drop(double p, const int64_t* seed) {
    const uint32_t limit = static_cast<uint32_t>(p * 65536.0 + 0.5);
    return Drop{seed, limit, limit < 65536 ? 65536.0f / static_cast<float>(65536 - limit) : 0.0f};
}

namespace {

__device__ __forceinline__ uint4 philox(uint64_t key, uint64_t block) {
    uint32_t c0 = static_cast<uint32_t>(block), c1 = static_cast<uint32_t>(block >> 32), c2 = 0, c3 = 0;
    uint32_t k0 = static_cast<uint32_t>(key), k1 = static_cast<uint32_t>(key >> 32);
#pragma unroll
    for (int i = 0; i < 10; ++i) {
        const uint64_t a = static_cast<uint64_t>(c0) * 0xD2511F53u, b = static_cast<uint64_t>(c2) * 0xCD9E8D57u;
        c0 = static_cast<uint32_t>(b >> 32) ^ c1 ^ k0;
        c1 = static_cast<uint32_t>(b);
        c2 = static_cast<uint32_t>(a >> 32) ^ c3 ^ k1;
        c3 = static_cast<uint32_t>(a);
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return uint4{c0, c1, c2, c3};
}

// Bit i: whether unit i of a block is kept.
__device__ __forceinline__ uint32_t kept_bits(uint64_t key, uint64_t block, uint32_t limit) {
    const uint4 w = philox(key, block);
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t v = i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w;
        bits |= ((v & 0xFFFFu) >= limit ? 1u : 0u) << (2 * i);
        bits |= ((v >> 16) >= limit ? 1u : 0u) << (2 * i + 1);
    }
    return bits;
}

// Whether unit u is kept.
__device__ __forceinline__ bool kept(uint64_t key, uint64_t u, uint32_t limit) {
    const uint4 w = philox(key, u >> 3);
    const uint32_t i = static_cast<uint32_t>(u) & 7u;
    const uint32_t v = i & 4 ? (i & 2 ? w.w : w.z) : (i & 2 ? w.y : w.x);
    return (i & 1 ? v >> 16 : v & 0xFFFFu) >= limit;
}

}  // namespace
}  // namespace feq
