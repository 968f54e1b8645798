// Rows kept in 8 bits for the backward pass: the format and its device code.
//
// A row of C values is cut into blocks of 32 (the last may be shorter).  With
// a = max |x| of a block and M = 127 (int8) or 448 (e4m3), e is the least
// integer with a <= M 2^e, at least -100; the block holds x 2^-e rounded to
// nearest even in the format, and the byte e + 127.  The value it stands for,
// x^ = q 2^e, is exact in fp32 and in bf16 (at most 7 significant bits, no
// subnormal), so a backward pass may read x^ in either.
//   |x^ - x| <= 2^(e-1)                     (int8)
//   |x^ - x| <= max(2^-4 |x|, 2^(e-10))     (e4m3: half a step of 3 mantissa
//                                           bits, or of its subnormals)
// A power-of-two scale costs int8 at most one of its bits and makes every
// step exact but the one rounding; a block with a value that is not finite
// has the scale byte 255 and zero values, and comes back as NaN: 0 times the
// infinity that the byte's exponent field spells.  A value in the last binade
// may round to 2^128 and come back as infinity, as it does in bf16.
//
// Memory: values[rows][ck_stride(C)] (rows padded to 16 bytes, so every piece
// of up to 16 is aligned; padding is written as zeros), scales[rows][ck_blocks(C)].
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mhc_device.h"

namespace mhc {

enum CkFormat : int { kCkInt8 = 0, kCkE4M3 = 1 };

constexpr int kCkBlock = 32;
__host__ __device__ constexpr int64_t ck_blocks(int64_t C) { return (C + kCkBlock - 1) / kCkBlock; }
__host__ __device__ constexpr int64_t ck_stride(int64_t C) { return (C + 15) / 16 * 16; }

// Maximum over the aligned group of G lanes (G <= 16), in every lane of it.
template <int G>
__device__ __forceinline__ uint32_t ck_group_max(uint32_t a) {
    auto step = [&](uint32_t b) { a = a > b ? a : b; };
    if constexpr (G >= 2) step(__float_as_uint(dpp::mov<dpp::kQuadXor1>(__uint_as_float(a))));
    if constexpr (G >= 4) step(__float_as_uint(dpp::mov<dpp::kQuadXor2>(__uint_as_float(a))));
    if constexpr (G >= 8) step(__float_as_uint(dpp::mov<dpp::kRowHalfMirror>(__uint_as_float(a))));
    if constexpr (G >= 16) step(__float_as_uint(dpp::mov<dpp::kRowMirror>(__uint_as_float(a))));
    return a;
}

// Sum over the aligned group of 2^lg lanes (lg >= 2), in every lane of it.
__device__ __forceinline__ float lane_group_sum(float v, int lg) {
    v = group_sum<4>(v);
    if (lg >= 3) v += dpp::mov<dpp::kRowHalfMirror>(v);
    if (lg >= 4) v += dpp::mov<dpp::kRowMirror>(v);
    if (lg >= 5) v = xor16_add(v);
    if (lg >= 6) v = xor32_add(v);
    return v;
}

// The bits of |x| order as the values do, with infinity and NaN on top.
__device__ __forceinline__ uint32_t ck_abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

template <int FMT>
struct Ck {
    // M = 1.m 2^kTop with mantissa field kPast: 127 = 1.984375 2^6, 448 = 1.75 2^8
    static constexpr int kTop = FMT == kCkInt8 ? 6 : 8;
    static constexpr uint32_t kPast = FMT == kCkInt8 ? 0x7E0000u : 0x600000u;

    // The scale byte of a block whose largest |x| has the bits a: a mantissa
    // past M's carries into the exponent field.
    __device__ __forceinline__ static uint32_t scale(uint32_t a) {
        const int e = (int)((a + (0x7FFFFFu - kPast)) >> 23) - kTop;
        return a >= 0x7F800000u ? 255u : (uint32_t)(e > 27 ? e : 27);
    }
    // 2^-e of a scale byte in 27 .. 254 (of 255: zero)
    __device__ __forceinline__ static float up(uint32_t s) { return __uint_as_float(s == 255u ? 0u : (254u - s) << 23); }
    // 2^e, infinity for 255
    __device__ __forceinline__ static float down(uint32_t s) { return __uint_as_float(s << 23); }

    // Four values times `up` in one word, element 0 lowest.  `keep` is 0 for
    // a block that is not finite (its bytes are zero), all ones otherwise.
    __device__ __forceinline__ static uint32_t pack4(float a, float b, float c, float d, float up, uint32_t keep) {
        if constexpr (FMT == kCkInt8) {
            // 1.5 2^23 + q: the add rounds to the nearest integer, ties to
            // even, and leaves q in two's complement in the low byte
            constexpr float kMagic = 12582912.f;
            const uint32_t q0 = __float_as_uint(__builtin_fmaf(a, up, kMagic));
            const uint32_t q1 = __float_as_uint(__builtin_fmaf(b, up, kMagic));
            const uint32_t q2 = __float_as_uint(__builtin_fmaf(c, up, kMagic));
            const uint32_t q3 = __float_as_uint(__builtin_fmaf(d, up, kMagic));
            // v_perm_b32: selector bytes 0-3 take the second operand's bytes, 4-7 the first's
            const uint32_t lo = __builtin_amdgcn_perm(q1, q0, 0x0c0c0400u);
            const uint32_t hi = __builtin_amdgcn_perm(q3, q2, 0x04000c0cu);
            return (lo | hi) & keep;
        } else {
            // v_cvt_pk_fp8_f32 (OCP e4m3 on gfx950, nearest even); |x 2^-e| <= 448
            int w = __builtin_amdgcn_cvt_pk_fp8_f32(a * up, b * up, 0, false);
            w = __builtin_amdgcn_cvt_pk_fp8_f32(c * up, d * up, w, true);
            return (uint32_t)w & keep;
        }
    }

    __device__ __forceinline__ static void unpack4(uint32_t w, float down, float (&v)[4]) {
        if constexpr (FMT == kCkInt8) {
            v[0] = (float)(int8_t)w * down;
            v[1] = (float)(int8_t)(w >> 8) * down;
            v[2] = (float)(int8_t)(w >> 16) * down;
            v[3] = (float)(int8_t)(w >> 24) * down;
        } else {
            const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
            const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
            v[0] = lo[0] * down; v[1] = lo[1] * down;
            v[2] = hi[0] * down; v[3] = hi[1] * down;
        }
    }
};

// ---------------------------------------------------------------------------
// Pieces of 8 elements at element alignment.  Rows of any length start
// anywhere; global accesses of 16 bytes need no more than the element's own
// alignment, so a vector type of that alignment keeps them whole.
// ---------------------------------------------------------------------------
typedef uint32_t ck_u4_t __attribute__((ext_vector_type(4)));
typedef ck_u4_t ck_u4_a4_t __attribute__((aligned(4)));
typedef ck_u4_t ck_u4_a2_t __attribute__((aligned(2)));

template <typename T> struct CkPiece;  // 8 elements as raw words
template <> struct CkPiece<float> {
    ck_u4_t w[2];
    __device__ __forceinline__ void load(const float* p) {
        w[0] = __builtin_nontemporal_load(reinterpret_cast<const ck_u4_a4_t*>(p));
        w[1] = __builtin_nontemporal_load(reinterpret_cast<const ck_u4_a4_t*>(p + 4));
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(w[e / 4][e % 4]);
    }
};
template <> struct CkPiece<bf16_t> {
    ck_u4_t w;
    __device__ __forceinline__ void load(const bf16_t* p) {
        w = __builtin_nontemporal_load(reinterpret_cast<const ck_u4_a2_t*>(p));
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[2 * e] = __uint_as_float(w[e] << 16);
            v[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
        }
    }
};

__device__ __forceinline__ void ck_store8(float* p, const float (&v)[8]) {
    const ck_u4_t a = {__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
    const ck_u4_t b = {__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7])};
    __builtin_nontemporal_store(a, reinterpret_cast<ck_u4_a4_t*>(p));
    __builtin_nontemporal_store(b, reinterpret_cast<ck_u4_a4_t*>(p + 4));
}
__device__ __forceinline__ void ck_store8(bf16_t* p, const float (&v)[8]) {
    const ck_u4_t a = {pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                       pack_bf16x2(v[6], v[7])};
    __builtin_nontemporal_store(a, reinterpret_cast<ck_u4_a2_t*>(p));
}

// The same for the first `m` (0 .. 7) of 8 elements.
template <typename T>
__device__ __forceinline__ void ck_load_part(const T* p, int m, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < m ? VecIO<T>::scalar(p + e) : 0.f;
}
template <typename T>
__device__ __forceinline__ void ck_store_part(T* p, int m, const float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (e < m) VecIO<T>::put(p + e, v[e]);
}

// 8 values per lane, 4 lanes a block: the scale byte and the two words.
template <int FMT>
__device__ __forceinline__ uint32_t ck_pack8(const float (&v)[8], uint2& w) {
    uint32_t a = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const uint32_t b = ck_abs_bits(v[e]);
        a = a > b ? a : b;
    }
    const uint32_t s = Ck<FMT>::scale(ck_group_max<4>(a));
    const float up = Ck<FMT>::up(s);
    const uint32_t keep = s == 255u ? 0u : ~0u;
    w.x = Ck<FMT>::pack4(v[0], v[1], v[2], v[3], up, keep);
    w.y = Ck<FMT>::pack4(v[4], v[5], v[6], v[7], up, keep);
    return s;
}

template <int FMT>
__device__ __forceinline__ void ck_unpack8(uint2 w, uint32_t s, float (&v)[8]) {
    const float down = Ck<FMT>::down(s);
    float a[4], b[4];
    Ck<FMT>::unpack4(w.x, down, a);
    Ck<FMT>::unpack4(w.y, down, b);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        v[e] = a[e];
        v[4 + e] = b[e];
    }
}

}  // namespace mhc
