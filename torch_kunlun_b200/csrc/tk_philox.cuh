// tk_philox.cuh -- the counter-based generator behind dropout: Philox4x32
// with 10 rounds (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as
// easy as 1, 2, 3", SC 2011).
//
// Element i of a tensor takes word i % 4 of the block with counter
// (i / 4, offset) and key `seed`, each a pair of 32-bit words, low word
// first.  The word depends on the element's index alone, not on the launch,
// so a backward pass recomputes the mask of its forward pass.
#pragma once

#include <cmath>
#include <cstdint>

namespace tk {

// The four words of the block (hi, lo).  Where hi is the same for the whole
// warp, so is half of the first two rounds, and the compiler computes it once
// per warp: 18 instead of 20 wide multiplies per thread, which bound dropout.
__device__ __forceinline__ void philox4x32_10(uint32_t lo, uint32_t hi, uint64_t offset, uint64_t seed,
                                              uint32_t (&out)[4]) {
    uint32_t c0 = lo, c1 = hi;
    uint32_t c2 = static_cast<uint32_t>(offset), c3 = static_cast<uint32_t>(offset >> 32);
    uint32_t k0 = static_cast<uint32_t>(seed), k1 = static_cast<uint32_t>(seed >> 32);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t a = static_cast<uint64_t>(0xD2511F53u) * c0;
        const uint64_t b = static_cast<uint64_t>(0xCD9E8D57u) * c2;
        c0 = static_cast<uint32_t>(b >> 32) ^ c1 ^ k0;
        c1 = static_cast<uint32_t>(b);
        c2 = static_cast<uint32_t>(a >> 32) ^ c3 ^ k1;
        c3 = static_cast<uint32_t>(a);
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    out[0] = c0;
    out[1] = c1;
    out[2] = c2;
    out[3] = c3;
}

// The dropout parameters a kernel takes.  An element is kept when its word is
// at least round(p * 2^32); a kept value is multiplied by 1 / (1 - p).
struct DropoutParams {
    uint64_t seed, offset;
    uint32_t threshold;
    float scale;
    bool none_kept;  // round(p * 2^32) == 2^32, which `threshold` cannot hold
};

inline DropoutParams dropout_params(double p, uint64_t seed, uint64_t offset) {
    const double t = std::nearbyint(p * 4294967296.0);
    DropoutParams d;
    d.seed = seed;
    d.offset = offset;
    d.none_kept = t >= 4294967296.0;
    d.threshold = d.none_kept ? 0xFFFFFFFFu : static_cast<uint32_t>(t);
    d.scale = d.none_kept ? 0.0f : static_cast<float>(1.0 / (1.0 - p));
    return d;
}

// Keep bits of the 8 elements [8 * octet, 8 * octet + 8), element j in bit j;
// indices below 2^34.
__device__ __forceinline__ uint32_t dropout_keep8(const DropoutParams& d, uint32_t octet) {
    uint32_t w[8];
    philox4x32_10(2 * octet, 0, d.offset, d.seed, reinterpret_cast<uint32_t(&)[4]>(w[0]));
    philox4x32_10(2 * octet + 1, 0, d.offset, d.seed, reinterpret_cast<uint32_t(&)[4]>(w[4]));
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m |= (w[j] >= d.threshold ? 1u : 0u) << j;
    return d.none_kept ? 0u : m;
}

// Keep bits of the 4 elements of one block, likewise.
__device__ __forceinline__ uint32_t dropout_keep4(const DropoutParams& d, uint32_t block) {
    uint32_t w[4];
    philox4x32_10(block, 0, d.offset, d.seed, w);
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) m |= (w[j] >= d.threshold ? 1u : 0u) << j;
    return d.none_kept ? 0u : m;
}

}  // namespace tk
