// Philox4x32-10, shared by the random samplers and by dropout: block n is the counter [n, n >> 32, 0, 0] under the
// key [seed, seed >> 32] (ref: src/ops/random.rs:29-63).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace hmr {

struct Word4 {
    uint32_t v[4];
};

__device__ __forceinline__ Word4 philox_block(uint64_t n, uint64_t seed) {
    constexpr uint32_t M0 = 0xD2511F53u, M1 = 0xCD9E8D57u, W0 = 0x9E3779B9u, W1 = 0xBB67AE85u;
    uint32_t c0 = static_cast<uint32_t>(n), c1 = static_cast<uint32_t>(n >> 32), c2 = 0, c3 = 0;
    uint32_t k0 = static_cast<uint32_t>(seed), k1 = static_cast<uint32_t>(seed >> 32);
#pragma unroll
    for (int round = 0; round < 10; ++round) {
        if (round > 0) {
            k0 += W0;
            k1 += W1;
        }
        // One 32 x 32 -> 64 multiply each (v_mad_u64_u32) rather than a high and a low half.
        const uint64_t p0 = static_cast<uint64_t>(M0) * c0, p1 = static_cast<uint64_t>(M1) * c2;
        const uint32_t n0 = static_cast<uint32_t>(p1 >> 32) ^ c1 ^ k0, n2 = static_cast<uint32_t>(p0 >> 32) ^ c3 ^ k1;
        c0 = n0, c1 = static_cast<uint32_t>(p1), c2 = n2, c3 = static_cast<uint32_t>(p0);
    }
    return Word4{{c0, c1, c2, c3}};
}

}  // namespace hmr
