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
    uint32_t fixed_k1, fixed_c3;  // see philox_block_same_high
};
constexpr uint32_t kPhiloxM0 = 0xD2511F53u, kPhiloxM1 = 0xCD9E8D57u;
// `high`: the upper half of the block numbers, where it is the same for all blocks of a launch.
inline PhiloxKeys philox_keys(uint64_t seed, uint32_t high) {
    PhiloxKeys k;
    uint32_t a = static_cast<uint32_t>(seed), b = static_cast<uint32_t>(seed >> 32);
    for (int round = 0; round < 10; ++round) {
        k.k0[round] = a;
        k.k1[round] = b;
        a += 0x9E3779B9u;
        b += 0xBB67AE85u;
    }
    const uint64_t second = static_cast<uint64_t>(kPhiloxM0) * (high ^ k.k0[0]);
    k.fixed_k1 = static_cast<uint32_t>(second >> 32) ^ k.k1[1];
    k.fixed_c3 = static_cast<uint32_t>(second);
    return k;
}
// Rounds `from` to 9 of philox_block from the seed's keys.
template <int FROM> __device__ __forceinline__ Words4 philox_rounds(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, const PhiloxKeys &keys) {
#pragma unroll
    for (int round = FROM; round < 10; ++round) {
        const uint64_t p0 = static_cast<uint64_t>(kPhiloxM0) * c0;
        const uint64_t p1 = static_cast<uint64_t>(kPhiloxM1) * c2;
        c0 = static_cast<uint32_t>(p1 >> 32) ^ c1 ^ keys.k0[round];
        c1 = static_cast<uint32_t>(p1);
        c2 = static_cast<uint32_t>(p0 >> 32) ^ c3 ^ keys.k1[round];
        c3 = static_cast<uint32_t>(p0);
    }
    return Words4{{c0, c1, c2, c3}};
}
__device__ __forceinline__ Words4 philox_block(uint64_t n, const PhiloxKeys &keys) {
    return philox_rounds<0>(static_cast<uint32_t>(n), static_cast<uint32_t>(n >> 32), 0, 0, keys);
}
// The same for a block whose number has the upper half that the keys were made for, from the product of its lower half with
// the first multiplier. The counter begins as (low, high, 0, 0), so half of the first round and half of the second do not
// depend on the block and are in the keys: 17 wide multiplications instead of 20.
__device__ __forceinline__ Words4 philox_block_same_high(uint64_t first_product, const PhiloxKeys &keys) {
    const uint32_t c2 = static_cast<uint32_t>(first_product >> 32) ^ keys.k1[0], c3 = static_cast<uint32_t>(first_product);
    const uint64_t p1 = static_cast<uint64_t>(kPhiloxM1) * c2;
    return philox_rounds<2>(static_cast<uint32_t>(p1 >> 32) ^ keys.k0[1], static_cast<uint32_t>(p1), c3 ^ keys.fixed_k1, keys.fixed_c3, keys);
}

}  // namespace hmc
