// bf16 matrix-core pieces shared by the projection kernels (dynamic.hip,
// proj_ckpt.hip).
#pragma once

#include "mhc_device.h"

namespace mhc {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f32x4_t mfma16x16x32(u32x4_t a, u32x4_t b, f32x4_t c) {
    // A rows = lane % 16, B cols = lane % 16, k = 8 * (lane / 16) + 0..7;
    // D[4 * (lane / 16) + i][lane % 16] in element i.
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b),
                                                   c, 0, 0, 0);
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) { return pack_bf16x2(lo, hi); }

__device__ __forceinline__ void split_pack8(const float (&v)[8], u32x4_t& hi, u32x4_t& lo) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t h = pack_bf16(v[2 * e], v[2 * e + 1]);
        hi[e] = h;
        lo[e] = pack_bf16(v[2 * e] - __uint_as_float(h << 16), v[2 * e + 1] - __uint_as_float(h & 0xffff0000u));
    }
}

constexpr int kDpPitch = 40;  // bf16 per row of the split dP copies (32 + 8 pad)

}  // namespace mhc
