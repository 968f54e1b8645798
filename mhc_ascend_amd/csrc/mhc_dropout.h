// Dropout from a counter: what is kept is computed where it is needed, in the
// forward and again in the backward, and never stored.
//
// The numbers are Philox4x32-10's (Salmon, Moraes, Dror and Shaw, "Parallel
// random numbers: as easy as 1, 2, 3", 2011): four 32-bit words from a 128-bit
// counter and a 64-bit key by ten rounds of two 32 x 32 -> 64 bit products.
// Channels 8 j .. 8 j + 7 of row i share one: counter = (i ceil(C / 8) + j,
// offset), two 64-bit numbers, key = seed; channel 8 j + e takes 16 bits, word
// e / 2, the low half for even e.  So a value's number depends on its row and
// channel alone, not on types, strides or the launch.
//
// A value is kept where its number is at least t = round(p 2^16), and then
// times 2^16 / (2^16 - t): the mean is exact for the p that t stands for, p to
// 2^-17.  16 bits a value and not 32 halve the products, which run beside the
// memory (two products a round at a quarter of the rate; 32768 x 4096 bf16, forward
// and backward: 174 us, with 32 bits a value 199; with the norm of 16384 x 4096 198
// and 206).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mhc_internal.h"

namespace mhc {

struct DropKey {
    uint32_t k0, k1, o0, o1;
    __device__ __forceinline__ DropKey(const DropArgs& d) {
        uint64_t seed = d.seed;
        if (d.seed_ptr) seed = *d.seed_ptr;
        k0 = (uint32_t)seed;
        k1 = (uint32_t)(seed >> 32);
        o0 = (uint32_t)d.offset;
        o1 = (uint32_t)(d.offset >> 32);
    }
    // The eight numbers of a block, two a word.
    __device__ __forceinline__ void words(uint64_t block, uint32_t (&c)[4]) const {
        c[0] = (uint32_t)block;
        c[1] = (uint32_t)(block >> 32);
        c[2] = o0;
        c[3] = o1;
        uint32_t a = k0, b = k1;
#pragma unroll
        for (int r = 0; r < 10; ++r) {
            const uint64_t m0 = (uint64_t)0xD2511F53u * c[0], m2 = (uint64_t)0xCD9E8D57u * c[2];
            c[0] = (uint32_t)(m2 >> 32) ^ c[1] ^ a;
            c[1] = (uint32_t)m2;
            c[2] = (uint32_t)(m0 >> 32) ^ c[3] ^ b;
            c[3] = (uint32_t)m0;
            a += 0x9E3779B9u;
            b += 0xBB67AE85u;
        }
    }
    // v where it is kept, times the scale, and zero elsewhere (whatever v is).
    // The product is rounded by itself: a sum behind it is not contracted, so
    // that dropout inside another operator gives its bits.
    __device__ __forceinline__ void apply(const DropArgs& d, uint64_t block, float (&v)[8]) const {
#pragma clang fp contract(off)
        uint32_t c[4];
        words(block, c);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t u = e & 1 ? c[e / 2] >> 16 : c[e / 2] & 0xffffu;
            v[e] = u >= d.threshold ? v[e] * d.scale : 0.f;
        }
    }
};

}  // namespace mhc
