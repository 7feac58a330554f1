// The Philox4x32-10 counter of homura's generator (src/ops/random.rs:29-51, 75-83), shared by the samplers and dropout.
#pragma once

#include <cstdint>

namespace hmc {

struct Words4 {
    uint32_t w[4];
};

// Block n under the key [seed, seed >> 32]. src/ops/random.rs:29-51, 75-83.
__device__ __forceinline__ Words4 philox_block(uint64_t n, uint64_t seed) {
    constexpr uint32_t kM0 = 0xD2511F53u, kM1 = 0xCD9E8D57u;
    constexpr uint32_t kW0 = 0x9E3779B9u, kW1 = 0xBB67AE85u;
    uint32_t c0 = static_cast<uint32_t>(n), c1 = static_cast<uint32_t>(n >> 32), c2 = 0, c3 = 0;
    uint32_t k0 = static_cast<uint32_t>(seed), k1 = static_cast<uint32_t>(seed >> 32);
#pragma unroll
    for (int round = 0; round < 10; ++round) {
        if (round > 0) {
            k0 += kW0;
            k1 += kW1;
        }
        const uint64_t p0 = static_cast<uint64_t>(kM0) * c0;  // one wide multiplication each
        const uint64_t p1 = static_cast<uint64_t>(kM1) * c2;
        c0 = static_cast<uint32_t>(p1 >> 32) ^ c1 ^ k0;
        c1 = static_cast<uint32_t>(p1);
        c2 = static_cast<uint32_t>(p0 >> 32) ^ c3 ^ k1;
        c3 = static_cast<uint32_t>(p0);
    }
    return Words4{{c0, c1, c2, c3}};
}

// The keys of the ten rounds under `seed`, laid out on the host for kernels that spend their time on the rounds: a key is
// then an operand in the constant bank instead of two sums a round.
struct PhiloxKeys {
    uint32_t k0[10], k1[10];
};
inline PhiloxKeys philox_keys(uint64_t seed) {
    PhiloxKeys k;
    uint32_t a = static_cast<uint32_t>(seed), b = static_cast<uint32_t>(seed >> 32);
    for (int round = 0; round < 10; ++round) {
        k.k0[round] = a;
        k.k1[round] = b;
        a += 0x9E3779B9u;
        b += 0xBB67AE85u;
    }
    return k;
}
// philox_block(n, seed) from the seed's keys.
__device__ __forceinline__ Words4 philox_block(uint64_t n, const PhiloxKeys &keys) {
    uint32_t c0 = static_cast<uint32_t>(n), c1 = static_cast<uint32_t>(n >> 32), c2 = 0, c3 = 0;
#pragma unroll
    for (int round = 0; round < 10; ++round) {
        const uint64_t p0 = static_cast<uint64_t>(0xD2511F53u) * c0;
        const uint64_t p1 = static_cast<uint64_t>(0xCD9E8D57u) * c2;
        c0 = static_cast<uint32_t>(p1 >> 32) ^ c1 ^ keys.k0[round];
        c1 = static_cast<uint32_t>(p1);
        c2 = static_cast<uint32_t>(p0 >> 32) ^ c3 ^ keys.k1[round];
        c3 = static_cast<uint32_t>(p0);
    }
    return Words4{{c0, c1, c2, c3}};
}

}  // namespace hmc
