// Counter-based random bits: Philox 4x32 with ten rounds (Salmon, Moraes, Dror and Shaw, "Parallel
// random numbers: as easy as 1, 2, 3", SC 2011).  A block of 128 bits is a pure function of a 128-bit
// counter and a 64-bit key, so a dropout mask needs no storage: the backward pass computes it again.
//
// Element i of a tensor (its position in row-major order, whatever the strides) takes 16 bits: half
// i % 2 (the low one first) of word (i % 8) / 2 of the block with counter (i / 8, offset), each 64 bits,
// low word first, under the key `seed`.  It is kept iff those bits, as a number, reach `units`, the drop
// probability in units of 2^-16.  Sixteen bits per element rather than 32 halve the work of the generator,
// which at 32 bits would bound a 16-bit type's dropout on integer issue rather than on memory; the
// factor of the kept elements goes by the probability actually used, so the expectation is unchanged.
#pragma once
#include "common.cuh"

namespace tpb {

struct DropSpec {
    unsigned long long seed, offset;
    unsigned units;   // 0: nothing is dropped (no bits are drawn), 65536: everything is
    float factor;     // of a kept element: 65536 / (65536 - units)
};

__device__ __forceinline__ uint4 philox_block(unsigned long long index, const DropSpec& d) {
    uint32_t c0 = (uint32_t)index, c1 = (uint32_t)(index >> 32), c2 = (uint32_t)d.offset, c3 = (uint32_t)(d.offset >> 32);
    uint32_t k0 = (uint32_t)d.seed, k1 = (uint32_t)(d.seed >> 32);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const unsigned long long a = (unsigned long long)c0 * 0xD2511F53u, b = (unsigned long long)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c1 = (uint32_t)b;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
}

// factors (0 or d.factor) of the eight elements 8 * index .. 8 * index + 7
__device__ __forceinline__ void drop_factors8(unsigned long long index, const DropSpec& d, float* f) {
    const uint4 w = philox_block(index, d);
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        f[2 * j] = (v[j] & 0xffffu) >= d.units ? d.factor : 0.0f;
        f[2 * j + 1] = (v[j] >> 16) >= d.units ? d.factor : 0.0f;
    }
}

// factor of one element
__device__ __forceinline__ float drop_factor1(unsigned long long i, const DropSpec& d) {
    const uint4 w = philox_block(i >> 3, d);
    const int j = (int)(i & 7) >> 1;
    const uint32_t v = j == 0 ? w.x : (j == 1 ? w.y : (j == 2 ? w.z : w.w));
    return ((i & 1) ? v >> 16 : v & 0xffffu) >= d.units ? d.factor : 0.0f;
}

// p in [0, 1] -> units and factor; false if p is not a probability
inline bool make_drop(double p, unsigned long long seed, unsigned long long offset, DropSpec* d) {
    if (!(p >= 0.0 && p <= 1.0)) return false;
    d->seed = seed;
    d->offset = offset;
    d->units = (unsigned)(p * 65536.0 + 0.5);
    d->factor = d->units >= 65536u ? 0.0f : (float)(65536.0 / (double)(65536u - d->units));
    return true;
}

}  // namespace tpb
