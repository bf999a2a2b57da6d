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
    unsigned above;   // units * 2^16 - 1: an element is kept iff its bits, shifted to the top of a word, are above it
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

// the eight elements 8 * index .. 8 * index + 7: dropped ones (NaN and infinity too) become 0, kept ones are
// multiplied by the factor
__device__ __forceinline__ void drop8(unsigned long long index, const DropSpec& d, float* v) {
    const uint4 w = philox_block(index, d);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        v[2 * j] = (u[j] << 16) > d.above ? v[2 * j] * d.factor : 0.0f;
        v[2 * j + 1] = u[j] > d.above ? v[2 * j + 1] * d.factor : 0.0f;     // the lower half cannot decide
    }
}

// which of those eight are kept, one bit each
__device__ __forceinline__ unsigned keep_bits8(unsigned long long index, const DropSpec& d) {
    const uint4 w = philox_block(index, d);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
    unsigned bits = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) bits |= ((u[j] << 16) > d.above ? 1u : 0u) << (2 * j) | (u[j] > d.above ? 2u : 0u) << (2 * j);
    return bits;
}

// p in [0, 1] -> units and factor; false if p is not a probability
inline bool make_drop(double p, unsigned long long seed, unsigned long long offset, DropSpec* d) {
    if (!(p >= 0.0 && p <= 1.0)) return false;
    d->seed = seed;
    d->offset = offset;
    d->units = (unsigned)(p * 65536.0 + 0.5);
    d->above = (unsigned)(((unsigned long long)d->units << 16) - 1);
    d->factor = d->units >= 65536u ? 0.0f : (float)(65536.0 / (double)(65536u - d->units));
    return true;
}

}  // namespace tpb
