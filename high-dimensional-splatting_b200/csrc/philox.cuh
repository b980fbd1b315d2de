// philox.cuh -- the counter-based generator behind dropout: Philox4x32-10 (Salmon, Moraes, Dror and Shaw,
// "Parallel random numbers: as easy as 1, 2, 3", 2011), written from the paper's definition.
//
// The mask of a draw (seed, offset) is a function of the element's number alone, so the forward, the
// backward and every kernel variant form the same mask and none stores it.  Element e takes half e % 8
// (low half first) of the four words of counter (e / 8, offset) under key seed: 16 random bits an
// element, eight elements a generator call, because at one call per four elements (32 bits each) the
// integer pipes, not the memory, would bound the kernels.  An element is dropped when its 16 bits are
// below the threshold T = round(65536 p), and the kept ones are scaled by 65536 / (65536 - T), the
// reciprocal of exactly the probability that T gives, so the expectation is kept whatever p is.
#pragma once

#include "hds_common.cuh"

namespace hds {

constexpr int DROP_ONE = 65536;  // a threshold of 1.0: everything is dropped

// The draw: by value, or read from device memory when the kernel runs (so that a captured graph can
// advance it between replays).
struct Draw {
    uint64_t seed, offset;
    const int64_t* device;  // {seed, offset}, or NULL
};

// The draw as numbers that are the same in every lane: the reductions tell the compiler so, which then
// keeps the ten round keys and what the offset alone decides out of the lanes' integer work.  Every lane
// of the warp must call it.
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __reduce_or_sync(FULL_MASK, x); }

__device__ __forceinline__ Draw resolve(Draw d) {
    if (d.device != nullptr) {
        d.seed = (uint64_t)d.device[0];
        d.offset = (uint64_t)d.device[1];
    }
    d.seed = (uint64_t)uniform((uint32_t)(d.seed >> 32)) << 32 | uniform((uint32_t)d.seed);
    d.offset = (uint64_t)uniform((uint32_t)(d.offset >> 32)) << 32 | uniform((uint32_t)d.offset);
    return d;
}

// The eight 16-bit numbers of a group: number j is the low (j even) or high half of word j / 2.
struct Numbers8 {
    uint32_t w[4];
    // below_last = 65536 T - 1: a number is >= T when, moved to the upper half of a word, it is greater.
    __device__ __forceinline__ bool kept(int j, uint32_t below_last) const {
        return (j % 2 == 0 ? w[j / 2] << 16 : w[j / 2]) > below_last;
    }
    // Bit j: whether number j is kept.
    __device__ __forceinline__ uint32_t bits(uint32_t below_last) const {
        uint32_t b = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) b |= kept(j, below_last) ? 1u << j : 0u;
        return b;
    }
};

// The numbers of group 2^32 group_high + group_low.  A group_high that is the same in every lane (a constant,
// or made from blockIdx) takes two of the twenty products out of the lanes' work.
__device__ __forceinline__ Numbers8 philox4x32_10(uint32_t group_low, uint32_t group_high, const Draw& d) {
    uint32_t x0 = group_low, x1 = group_high;
    uint32_t x2 = (uint32_t)d.offset, x3 = (uint32_t)(d.offset >> 32);
    uint32_t k0 = (uint32_t)d.seed, k1 = (uint32_t)(d.seed >> 32);
#pragma unroll
    for (int r = 0; r < 10; r++) {
        const uint64_t p0 = (uint64_t)x0 * 0xD2511F53u, p1 = (uint64_t)x2 * 0xCD9E8D57u;
        x0 = (uint32_t)(p1 >> 32) ^ x1 ^ k0;
        x2 = (uint32_t)(p0 >> 32) ^ x3 ^ k1;
        x1 = (uint32_t)p1;
        x3 = (uint32_t)p0;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return Numbers8{{x0, x1, x2, x3}};
}

// For the kernels' below_last; thresholds from 1 to 65536 (modulo 2^32).
inline uint32_t below_last(int threshold) { return (uint32_t)((uint64_t)threshold * 65536u - 1u); }

// scale / (the kept share), rounded once to float; 0 when everything is dropped.
inline float keep_factor(double scale, int threshold) {
    return threshold >= DROP_ONE ? 0.0f : (float)(scale * ((double)DROP_ONE / (double)(DROP_ONE - threshold)));
}

}  // namespace hds
