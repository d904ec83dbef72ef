// Philox-4x32 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", 2011): a bijection of a counter of four words under a
// key of two.  Seven rounds, the fewest that its authors found to pass every test of BigCrush; a round is two products of 32 x 32 bits, which
// v_mad_u64_u32 gives whole.  16 bits for each value: eight values from a counter, and probabilities in units of 2^-16.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

struct TdbKey {
    uint32_t lo, hi;
};

__device__ __forceinline__ TdbKey tdb_key(const int64_t* seed) {
    const uint64_t s = uint64_t(*seed);
    return {uint32_t(s), uint32_t(s >> 32)};
}

__device__ __forceinline__ uint4 tdb_philox(uint32_t a, uint32_t b, uint32_t c, uint32_t d, TdbKey key) {
#pragma unroll
    for (int r = 0; r < 7; ++r) {
        const uint64_t x = uint64_t(a) * 0xD2511F53u, y = uint64_t(c) * 0xCD9E8D57u;
        const uint32_t na = uint32_t(y >> 32) ^ b ^ (key.lo + uint32_t(r) * 0x9E3779B9u);
        const uint32_t nc = uint32_t(x >> 32) ^ d ^ (key.hi + uint32_t(r) * 0xBB67AE85u);
        b = uint32_t(y), d = uint32_t(x);
        a = na, c = nc;
    }
    return uint4{a, b, c, d};
}

// Number n of the eight, n a constant.
__device__ __forceinline__ uint32_t tdb_number(uint4 w, int n) {
    const uint32_t x = n < 2 ? w.x : n < 4 ? w.y : n < 6 ? w.z : w.w;
    return n & 1 ? x >> 16 : x & 0xffffu;
}

// Bit k: whether value k of the counter is kept.
__device__ __forceinline__ uint32_t tdb_kept(uint4 w, uint32_t threshold) {
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        bits |= (x[i] & 0xffffu) >= threshold ? 1u << (2 * i) : 0u;
        bits |= (x[i] >> 16) >= threshold ? 2u << (2 * i) : 0u;
    }
    return bits;
}

// What kept values are multiplied by; nothing is kept at 65536.
__host__ __device__ __forceinline__ float tdb_kept_factor(int threshold) {
    return threshold >= 65536 ? 0.f : 65536.f / float(65536 - threshold);
}
