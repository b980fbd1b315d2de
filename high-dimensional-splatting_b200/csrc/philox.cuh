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

__device__ __forceinline__ Draw resolve(Draw d) {
    if (d.device != nullptr) {
        d.seed = (uint64_t)d.device[0];
        d.offset = (uint64_t)d.device[1];
    }
    return d;
}

__device__ __forceinline__ uint4 philox4x32_10(uint64_t counter, const Draw& d) {
    uint32_t x0 = (uint32_t)counter, x1 = (uint32_t)(counter >> 32);
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
    return make_uint4(x0, x1, x2, x3);
}

// Bit j: whether element 8 group + j is kept.
__device__ __forceinline__ uint32_t keep8(uint64_t group, const Draw& d, uint32_t threshold) {
    const uint4 w = philox4x32_10(group, d);
    const uint32_t words[4] = {w.x, w.y, w.z, w.w};
    uint32_t bits = 0;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        bits |= ((words[k] & 0xffffu) >= threshold ? 1u : 0u) << (2 * k);
        bits |= ((words[k] >> 16) >= threshold ? 2u : 0u) << (2 * k);
    }
    return bits;
}

__device__ __forceinline__ bool keep_one(uint64_t e, const Draw& d, uint32_t threshold) {
    return (keep8(e >> 3, d, threshold) >> (e & 7)) & 1u;
}

// scale / (the kept share), rounded once to float; 0 when everything is dropped.
inline float keep_factor(double scale, int threshold) {
    return threshold >= DROP_ONE ? 0.0f : (float)(scale * ((double)DROP_ONE / (double)(DROP_ONE - threshold)));
}

}  // namespace hds
