// philox.cuh -- the counter-based generator behind dropout: Philox4x32-10
// (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2,
// 3", 2011), written from the paper: ten rounds of two 32 x 32 -> 64-bit
// products on a 128-bit counter under a 64-bit key that a Weyl sequence steps.
//
// A mask is a function of (seed, row, column) alone and is never stored:
//   counter = (column >> 3, 0, row's low 32 bits, row's high 32 bits), key = seed;
//   the four output words are eight 16-bit halves, half column & 7 decides:
//   kept iff half >= threshold, threshold = round(p * 2^16) in 0 .. 2^16.
// Sixteen bits a value: one generator call serves eight values, one 16-byte load
// of a 16-bit type.  The 20 wide products of a call are then a sixth of a bf16
// dropout's time (16384 x 4096: 60 us, with one round instead of ten 50 us); at 32
// bits a value there would be twice as many.  The scale uses the held probability
// threshold / 2^16, so the expectation is exact.  Rows count from row_offset: a
// token shard that passes its first row draws the same mask as the whole.
#pragma once

#include <stdint.h>

namespace act {

struct DropParams {
    uint64_t seed;             // used when seed_ptr is null
    const uint64_t *seed_ptr;  // device memory, read by the kernel
    uint64_t row_offset;
    uint32_t threshold;        // 0 .. 65536
    float scale;               // 65536 / (65536 - threshold), 0 if nothing is kept
};

__device__ __forceinline__ uint64_t drop_seed(const DropParams &d) {
    return d.seed_ptr ? *d.seed_ptr : d.seed;
}

__device__ __forceinline__ uint4 philox4x32_10(uint32_t c0, uint32_t c2, uint32_t c3, uint64_t key) {
    uint32_t c1 = 0, k0 = (uint32_t)key, k1 = (uint32_t)(key >> 32);
#pragma unroll
    for (int i = 0; i < 10; ++i) {
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

// Bit j of the result: whether value 8 * block + j of the row is kept.
__device__ __forceinline__ uint32_t drop_keep8(uint64_t row, uint32_t block, uint64_t key, uint32_t threshold) {
    const uint4 r = philox4x32_10(block, (uint32_t)row, (uint32_t)(row >> 32), key);
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
    uint32_t keep = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if ((w[j] & 0xffffu) >= threshold) keep |= 1u << (2 * j);
        if ((w[j] >> 16) >= threshold) keep |= 2u << (2 * j);
    }
    return keep;
}

}  // namespace act
