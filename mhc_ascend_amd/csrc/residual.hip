// Dropout of rows (mhc_dropout.h), and the RMSNorm of a residual's sum:
//   h = residual + dropout(x), rounded to residual's type
//   y = h / r * w,  r = sqrt(mean h^2 + eps), in x's type or in 8 bits (mhc_ckpt.h)
// Backward, for cotangents gy and gh (u = gy w):
//   dh = gh + u / r - h (sum_c u h) / (C r^3),  dx = dropout(dh),  dw = sum_rows gy h / r
// with h as it was stored, or the values of its 8-bit checkpoint (r from them
// as well).
#include <type_traits>

#include "mhc_ckpt.h"
#include "mhc_device.h"
#include "mhc_dropout.h"
#include "mhc_internal.h"

namespace mhc {

// ---------------------------------------------------------------------------
// Dropout.  A lane takes a piece of 8 channels, and the block of numbers that is
// theirs.  Rows of a multiple of 8 are one run of pieces; in other rows a piece's
// row is found by a 32-bit division.  Bound by bytes, its integer products beside
// them: 32768 x 4096 bf16 87 us, 6.2 TB/s (two pieces a lane 1 us more, four 3: many
// short waves spread the products best), 16384 x 4096 fp32 95 us, 5.7 TB/s; 7318 x
// 4673 bf16, rows on no boundary, 27 us, 5.1 TB/s.
// ---------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void dropout_flat_kernel(const T* __restrict__ x, T* __restrict__ y, DropArgs d,
                                                           int64_t first, int64_t pieces) {
    const int64_t p = first + (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (p >= pieces) return;
    CkPiece<T> in;
    in.load(x + p * 8);
    float v[8];
    in.get(v);
    DropKey(d).apply(d, (uint64_t)p, v);
    ck_store8(y + p * 8, v);
}

// rows * ceil(C / 8) < 2^31 pieces in a launch, from row `row0` on
template <typename T>
__global__ __launch_bounds__(256) void dropout_rows_kernel(const T* __restrict__ x, T* __restrict__ y, DropArgs d,
                                                           int64_t row0, uint32_t pieces, int C) {
    const DropKey key(d);
    const uint32_t per = ((uint32_t)C + 7u) / 8u;
    const uint32_t p = blockIdx.x * 256u + threadIdx.x;
    if (p >= pieces) return;
    const uint32_t r = p / per;
    const int c0 = (int)(p - r * per) * 8;
    const int m = C - c0;
    const int64_t at = (row0 + r) * C + c0;
    float v[8];
    if (m >= 8) {
        CkPiece<T> in;
        in.load(x + at);
        in.get(v);
    } else {
        ck_load_part(x + at, m, v);
    }
    key.apply(d, (uint64_t)row0 * per + p, v);
    if (m >= 8) ck_store8(y + at, v);
    else ck_store_part(y + at, m, v);
}

template <typename T>
static hipError_t dropout_run(const T* x, T* y, const DropArgs& d, int64_t rows, int64_t C, hipStream_t s) {
    if (C % 8 == 0) {
        const int64_t pieces = rows * (C / 8), most = (int64_t)1 << 31;  // lanes a launch
        for (int64_t p = 0; p < pieces; p += most) {
            const int64_t n = pieces - p < most ? pieces - p : most;
            MHC_LAUNCH_GGL((dropout_flat_kernel<T>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, x, y, d, p,
                           p + n);
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return e;
        }
        return hipSuccess;
    }
    const int64_t per = (C + 7) / 8, most = ((int64_t)1 << 30) / per;  // rows a launch
    for (int64_t r = 0; r < rows; r += most) {
        const int64_t n = (rows - r < most ? rows - r : most) * per;
        MHC_LAUNCH_GGL((dropout_rows_kernel<T>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, x, y, d, r,
                       (uint32_t)n, (int)C);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

hipError_t launch_dropout(int dt, const void* x, void* out, const DropArgs& d, int64_t rows, int64_t C,
                          hipStream_t s) {
    if (rows == 0) return hipSuccess;
    const int tok = timing_begin("dropout", s);
    const hipError_t e = dt == kBF16 ? dropout_run((const bf16_t*)x, (bf16_t*)out, d, rows, C, s)
                                     : dropout_run((const float*)x, (float*)out, d, rows, C, s);
    timing_end(tok, s);
    return e;
}

// ---------------------------------------------------------------------------
// Rows of any length, a workgroup a row at a time: h goes to memory in the first
// loop over the row and is read back by the lane that wrote it in the second.  A
// lane adds up to 2^20 values of a row one by one, so the row's sums are in 64 bits
// (fp32 sums of 2^14 equal ones a lane were off by 3000 roundings).  For rows that
// no workgroup's registers hold: 4096 x 20000 bf16 forward 182 us (3.6 TB/s of the
// four arrays; 179 with fp32 sums), backward 378 (370; 1.7 TB/s: every array is read
// twice, and dw's partial row read and written in fp32 once a row); 8192 x 16384 bf16
// with the rows in registers 182 and 217 us, 5.9 and 4.9 TB/s.
// ---------------------------------------------------------------------------
constexpr int kResAnyThreads = 1024;

template <typename T>
__device__ __forceinline__ void res_piece(const T* __restrict__ p, int m, float (&v)[8]) {
    if (m >= 8) {
        CkPiece<T> in;
        in.load(p);
        in.get(v);
    } else {
        ck_load_part(p, m < 0 ? 0 : m, v);
    }
}
template <typename T>
__device__ __forceinline__ void res_put(T* __restrict__ p, int m, const float (&v)[8]) {
    if (m >= 8) ck_store8(p, v);
    else ck_store_part(p, m < 0 ? 0 : m, v);
}
// Values as the storage type holds them.
template <typename T>
__device__ __forceinline__ void res_round(float (&v)[8]) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const uint32_t w = pack_bf16x2(v[e], v[e + 1]);
            v[e] = __uint_as_float(w << 16);
            v[e + 1] = __uint_as_float(w & 0xffff0000u);
        }
    }
}
__device__ __forceinline__ void res_weight(const ResidualArgs& a, int c0, float (&w)[8]) {
    if (a.w_dtype == kBF16) res_piece(static_cast<const bf16_t*>(a.w) + c0, a.C - c0, w);
    else res_piece(static_cast<const float*>(a.w) + c0, a.C - c0, w);
}
// A lane's 8 values of a row in 8 bits; every lane of a block of 32 takes part.
template <bool NT = true>
__device__ __forceinline__ void res_pack(int fmt, const float (&v)[8], uint8_t* __restrict__ q,
                                         uint8_t* __restrict__ sc, int64_t row, int C, int c0) {
    uint2 p;
    const uint32_t s = fmt == kCkInt8 ? ck_pack8<kCkInt8>(v, p) : ck_pack8<kCkE4M3>(v, p);
    if (c0 < (int)ck_stride(C)) {
        uint8_t* at = q + row * ck_stride(C) + c0;
        if (NT) st8_nt(at, p);
        else *reinterpret_cast<uint2*>(at) = p;
    }
    if ((c0 & 31) == 0 && c0 < C) sc[row * ck_blocks(C) + (c0 >> 5)] = (uint8_t)s;
}
__device__ __forceinline__ void res_unpack(int fmt, const uint8_t* __restrict__ q, const uint8_t* __restrict__ sc,
                                           int64_t row, int C, int c0, float (&v)[8]) {
    const uint2 p = ld8_nt(q + row * ck_stride(C) + c0);
    const uint32_t s = sc[row * ck_blocks(C) + (c0 >> 5)];
    if (fmt == kCkInt8) ck_unpack8<kCkInt8>(p, s, v);
    else ck_unpack8<kCkE4M3>(p, s, v);
}

// ---------------------------------------------------------------------------
// y in 8 bits is rounded once, from the norm's value: a number next to the middle
// of two 8-bit ones, or a block's largest next to where its exponent changes, would
// otherwise fall to one side or the other by the roundings before it (of 67 M e4m3
// numbers some tens, and a whole block of 32 now and then).  So there the mean
// square is summed in 64 bits, 1 / r and its product with h have two parts, and fp32
// y is rounded to odd: cut off, with the last bit set where something was lost,
// which the rounding to 8 bits takes for what it is.
// ---------------------------------------------------------------------------
// 1 / sqrt(s) = hi + lo: the instruction's own approximation (an ulp or so), the rest
// from the residual 1 - s hi^2; zero where that has no meaning (hi zero or
// infinite).  The instruction takes a subnormal s for zero, and under a large s the
// residual's terms are subnormal: past 2^-63 .. 2^65 both are formed for s of 1 / 4
// to 1 and its power of two put back (a branch that waves skip).  An s that is zero
// or infinite in fp32 is taken for that, as it is for y in fp32.
struct ResInv {
    float hi, lo;
    __device__ __forceinline__ explicit ResInv(double s) {
        const float f = (float)s;
        int k = 0;
        if (__float_as_uint(f) - 0x20000000u >= 0x40000000u) {
            k = (__builtin_amdgcn_frexp_expf(f) + 1) >> 1;
            s = __builtin_ldexp(s, -2 * k);
        }
        const float sh = (float)s, sl = (float)(s - (double)sh);
        hi = __builtin_amdgcn_rsqf(sh);
        const float sq = hi * hi, rest = __builtin_fmaf(hi, hi, -sq);
        const float res = __builtin_fmaf(-sl, sq, __builtin_fmaf(-sh, rest, __builtin_fmaf(-sh, sq, 1.f)));
        lo = fabsf(res) < 0x1p-10f ? 0.5f * hi * res : 0.f;
        hi = __builtin_ldexpf(hi, -k);
        lo = __builtin_ldexpf(lo, -k);
    }
    // v / r * w, rounded to odd: where something was lost (not where y is infinite),
    // one step towards zero if y was rounded away from it, then the last bit set
    __device__ __forceinline__ float odd(float v, float w) const {
        const float n = v * hi, nl = __builtin_fmaf(v, lo, __builtin_fmaf(v, hi, -n)), c = w * nl;
        const float y = __builtin_fmaf(w, n, c);
        const float rest = __builtin_fmaf(w, n, -y) + c;   // what y is off by
        constexpr int kLost = 0x198;                       // normal and subnormal numbers of either sign
        const uint32_t u = __float_as_uint(y), past = (u ^ __float_as_uint(rest)) >> 31;
        return __builtin_amdgcn_classf(rest, kLost) ? __uint_as_float((u - past) | 1u) : y;
    }
};

__device__ __forceinline__ double res_square(const float (&v)[8], double s) {
#pragma unroll
    for (int e = 0; e < 8; ++e) s = __builtin_fma((double)v[e], (double)v[e], s);
    return s;
}

// Sum over the aligned group of 2^lg lanes (lg >= 2), in every lane of it.
template <int CTRL>
__device__ __forceinline__ double res_dpp_add(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __float_as_uint(dpp::mov<CTRL>(__uint_as_float((uint32_t)u)));
    const uint32_t hi = __float_as_uint(dpp::mov<CTRL>(__uint_as_float((uint32_t)(u >> 32))));
    return v + __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double res_group_sum(double v, int lg) {
    const auto pair = [](auto lo, auto hi) {
        return __builtin_bit_cast(double, (uint64_t)hi[0] << 32 | lo[0]) +
               __builtin_bit_cast(double, (uint64_t)hi[1] << 32 | lo[1]);
    };
    v = res_dpp_add<dpp::kQuadXor1>(v);
    v = res_dpp_add<dpp::kQuadXor2>(v);
    if (lg >= 3) v = res_dpp_add<dpp::kRowHalfMirror>(v);
    if (lg >= 4) v = res_dpp_add<dpp::kRowMirror>(v);
    if (lg >= 5) {
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = (uint32_t)u, hi = (uint32_t)(u >> 32);
        v = pair(__builtin_amdgcn_permlane16_swap(lo, lo, false, false),
                 __builtin_amdgcn_permlane16_swap(hi, hi, false, false));
    }
    if (lg >= 6) {
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = (uint32_t)u, hi = (uint32_t)(u >> 32);
        v = pair(__builtin_amdgcn_permlane32_swap(lo, lo, false, false),
                 __builtin_amdgcn_permlane32_swap(hi, hi, false, false));
    }
    return v;
}
// Sum over the workgroup, in every lane; red: a double a wave.
__device__ __forceinline__ double res_block_sum(double v, double* red) {
    v = res_group_sum(v, 6);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0;
    for (unsigned w = 0; w < blockDim.x / 64; ++w) v += red[w];
    __syncthreads();
    return v;
}

template <typename TX, typename TR>
__global__ __launch_bounds__(kResAnyThreads) void residual_fwd_any_kernel(ResidualArgs a) {
    __shared__ double red[16];
    const DropKey key(a.drop);
    const int C = a.C;
    const double each = 1.0 / C;
    const int64_t per = ((int64_t)C + 7) / 8;
    // whole blocks of 32, so that the lanes of one pack it together
    const int64_t end = ck_blocks(C) * kCkBlock;
    for (int64_t b = blockIdx.x; b < a.B; b += gridDim.x) {
        const TX* x = static_cast<const TX*>(a.x) + b * C;
        const TR* res = static_cast<const TR*>(a.residual) + b * C;
        TR* h = static_cast<TR*>(a.h) + b * C;
        double t = 0.0;
        for (int64_t c = (int64_t)threadIdx.x * 8; c < end; c += kResAnyThreads * 8) {
            const int c0 = (int)c, m = c < C ? C - c0 : 0;
            float v[8], r[8];
            res_piece(x + (m > 0 ? c0 : 0), m, v);
            res_piece(res + (m > 0 ? c0 : 0), m, r);
            if (a.drop.threshold) key.apply(a.drop, (uint64_t)(b * per + c / 8), v);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += r[e];
            res_round<TR>(v);
            if (m > 0) res_put(h + c0, m, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = e < m ? v[e] : 0.f;
            t = res_square(v, t);
            if (a.h_fmt >= 0) res_pack(a.h_fmt, v, a.hq, a.hsc, b, C, c0);
        }
        t = res_block_sum(t, red) * each;
        if (a.y_fmt >= 0) {
            const ResInv inv(t + a.eps);
            for (int64_t c = (int64_t)threadIdx.x * 8; c < end; c += kResAnyThreads * 8) {
                const int c0 = (int)c, m = c < C ? C - c0 : 0;
                float v[8], w[8];
                res_piece(h + (m > 0 ? c0 : 0), m, v);
                if (m > 0) {
                    res_weight(a, c0, w);
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = e < m ? inv.odd(v[e], w[e]) : 0.f;
                }
                res_pack(a.y_fmt, v, a.yq, a.ysc, b, C, c0);
            }
            continue;
        }
        const float inv = 1.f / sqrtf((float)t + a.eps);
        for (int64_t c = (int64_t)threadIdx.x * 8; c < C; c += kResAnyThreads * 8) {
            const int c0 = (int)c, m = C - c0;
            float v[8], w[8];
            res_piece(h + c0, m, v);
            res_weight(a, c0, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = v[e] * inv * w[e];
            res_put(static_cast<TX*>(a.y) + b * C + c0, m, v);
        }
    }
}

// dw is summed in the workgroup's own partial row, each channel by one lane.
template <typename TX, typename TR>
__global__ __launch_bounds__(kResAnyThreads) void residual_bwd_any_kernel(ResidualArgs a) {
    __shared__ double red[16];
    const DropKey key(a.drop);
    const int C = a.C;
    const double each = 1.0 / C;
    const int64_t per = ((int64_t)C + 7) / 8;
    for (int64_t b = blockIdx.x; b < a.B; b += gridDim.x) {
        const TX* gy = static_cast<const TX*>(a.gy) + b * C;
        const auto row = [&](int c0, int m, float (&v)[8]) {
            if (a.h_fmt >= 0) res_unpack(a.h_fmt, a.hq, a.hsc, b, C, c0, v);
            else res_piece(static_cast<const TR*>(a.h) + b * C + c0, m, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = e < m ? v[e] : 0.f;
        };
        double ss = 0.0, dot = 0.0;
        for (int64_t c = (int64_t)threadIdx.x * 8; c < C; c += kResAnyThreads * 8) {
            const int c0 = (int)c, m = C - c0;
            float h[8], g[8], w[8];
            row(c0, m, h);
            res_piece(gy + c0, m, g);
            res_weight(a, c0, w);
            ss = res_square(h, ss);
#pragma unroll
            for (int e = 0; e < 8; ++e) dot = __builtin_fma((double)(g[e] * w[e]), (double)h[e], dot);
        }
        ss = res_block_sum(ss, red) * each;
        dot = res_block_sum(dot, red) * each;
        const float inv = 1.f / sqrtf((float)ss + a.eps);
        const float k2 = (float)dot * inv * inv * inv;
        float* dw = a.dw_part ? a.dw_part + (int64_t)blockIdx.x * C : nullptr;
        for (int64_t c = (int64_t)threadIdx.x * 8; c < C; c += kResAnyThreads * 8) {
            const int c0 = (int)c, m = C - c0;
            float h[8], g[8], w[8], d[8];
            row(c0, m, h);
            res_piece(gy + c0, m, g);
            res_weight(a, c0, w);
            if (a.gh) res_piece(static_cast<const TR*>(a.gh) + b * C + c0, m, d);
            else ck_load_part(static_cast<const TR*>(nullptr), 0, d);
            if (dw) {
                float p[8];
                if (b == blockIdx.x) ck_load_part(dw, 0, p);
                else res_piece(dw + c0, m, p);
#pragma unroll
                for (int e = 0; e < 8; ++e) p[e] += g[e] * h[e] * inv;
                res_put(dw + c0, m, p);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) d[e] += w[e] * g[e] * inv - h[e] * k2;
            if (a.gres) res_put(static_cast<TR*>(a.gres) + b * C + c0, m, d);
            if (a.gx) {
                if (a.drop.threshold) key.apply(a.drop, (uint64_t)(b * per + c / 8), d);
                res_put(static_cast<TX*>(a.gx) + b * C + c0, m, d);
            }
        }
    }
}

// ---------------------------------------------------------------------------
// Rows in registers (mhc_ckpt.h), up to kCkMaxRow channels: persistent
// workgroups, the weight in registers and the next row's loads in flight, so
// that every array is read or written once.  1024 lanes a CU: more add nothing in
// flight that the memory has not (16384 x 4096 bf16 forward 81 us, the same with 1536
// and 2048), and rows that share lines want fewer at once (20000 x 2733 fp32 forward
// 179 us, 240 with 1536).  The forward's outputs are stored to stay in the caches:
// what runs next reads them (16384 x 4096 bf16 with dropout, forward and backward,
// 198 us, 215 with streaming stores; forward alone 81 and 92).  The backward's
// stream, but for rows on no 16-byte boundary, whose neighbours' ends share lines
// (backward of 20000 x 2733 fp32 187 us, streamed 196; 400000 x 100 bf16 66 and 70; of
// 30000 x 4095 bf16 244 and 234).  Bound by bytes: 16384 x 4096 bf16 without dropout
// forward 81 us, 6.6 TB/s, backward 84, 6.4; with it 82 and 111, 6.5 and 6.0; 30000 x
// 4095 233 and 244 us, 4.2 and 4.0 TB/s: most of a row's pieces lie across lines.
// ---------------------------------------------------------------------------
template <int VPT, bool RAG>
__device__ __forceinline__ void res_weights(const ResidualArgs& a, float (&w)[VPT][8]) {
    if (a.w_dtype == kBF16) {
        CkPiece<bf16_t> p[VPT];
        ck_row_load<bf16_t, VPT, RAG>(static_cast<const bf16_t*>(a.w), a.C, p);
        ck_row_get<bf16_t, VPT, RAG>(static_cast<const bf16_t*>(a.w), a.C, p, w);
    } else {
        CkPiece<float> p[VPT];
        ck_row_load<float, VPT, RAG>(static_cast<const float*>(a.w), a.C, p);
        ck_row_get<float, VPT, RAG>(static_cast<const float*>(a.w), a.C, p, w);
    }
}

// ck_row_get without the zeros of lanes past the row.
template <typename T, int VPT, bool RAG>
__device__ __forceinline__ void res_row_get(const T* __restrict__ row, int C, const CkPiece<T> (&in)[VPT],
                                            float (&v)[VPT][8]) {
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        const int c0 = (k * blockDim.x + threadIdx.x) * 8;
        in[k].get(v[k]);
        if (RAG && c0 < C && c0 + 8 > C) {
            if (C >= 8) ck_shift_part(C - c0, v[k]);
            else ck_load_part(row, C, v[k]);
        }
    }
}

template <typename TX, typename TR, int VPT, bool RAG>
__global__ __launch_bounds__(1024) void residual_fwd_kernel(ResidualArgs a) {
    __shared__ float red[16];
    __shared__ double red64[16];
    const DropKey key(a.drop);
    const int C = a.C;
    const double each = 1.0 / C;
    const int64_t per = (C + 7) / 8;
    const TX* x = static_cast<const TX*>(a.x);
    const TR* res = static_cast<const TR*>(a.residual);
    const bool past = C < (int)blockDim.x * VPT * 8;  // some lane's piece is past the row
    CkPiece<TX> xn[VPT];
    CkPiece<TR> rn[VPT];
    int64_t b = blockIdx.x;
    ck_row_load<TX, VPT, RAG>(x + b * C, C, xn);
    ck_row_load<TR, VPT, RAG>(res + b * C, C, rn);
    float w[VPT][8];
    res_weights<VPT, RAG>(a, w);
    for (; b < a.B; b += gridDim.x) {
        float v[VPT][8];
        float t[1] = {0.f};
        {
            float r[VPT][8];
            res_row_get<TX, VPT, RAG>(x + b * C, C, xn, v);
            res_row_get<TR, VPT, RAG>(res + b * C, C, rn, r);
            const int64_t b1 = b + gridDim.x < a.B ? b + gridDim.x : b;
            ck_row_load<TX, VPT, RAG>(x + b1 * C, C, xn);
            ck_row_load<TR, VPT, RAG>(res + b1 * C, C, rn);
#pragma unroll
            for (int k = 0; k < VPT; ++k) {
                if (a.drop.threshold) key.apply(a.drop, (uint64_t)(b * per + k * blockDim.x + threadIdx.x), v[k]);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[k][e] += r[k][e];
                if (past && (k * blockDim.x + threadIdx.x) * 8 >= C) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[k][e] = 0.f;
                }
                res_round<TR>(v[k]);
            }
        }
        ck_row_put<TR, VPT, RAG, false>(static_cast<TR*>(a.h) + b * C, C, v);
        if (a.h_fmt >= 0) {
#pragma unroll
            for (int k = 0; k < VPT; ++k)
                res_pack(a.h_fmt, v[k], a.hq, a.hsc, b, C, (k * blockDim.x + threadIdx.x) * 8);
        }
        if (a.y_fmt >= 0) {
            double t64 = 0.0;
#pragma unroll
            for (int k = 0; k < VPT; ++k) t64 = res_square(v[k], t64);
            const ResInv inv(res_block_sum(t64, red64) * each + a.eps);
#pragma unroll
            for (int k = 0; k < VPT; ++k) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[k][e] = inv.odd(v[k][e], w[k][e]);
                res_pack<false>(a.y_fmt, v[k], a.yq, a.ysc, b, C, (k * blockDim.x + threadIdx.x) * 8);
            }
            continue;
        }
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
#pragma unroll
            for (int e = 0; e < 8; ++e) t[0] += v[k][e] * v[k][e];
        }
        block_sum<1>(t, red);
        const float inv = 1.f / sqrtf(t[0] / (float)C + a.eps);
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[k][e] = v[k][e] * inv * w[k][e];
        }
        ck_row_put<TX, VPT, RAG, false>(static_cast<TX*>(a.y) + b * C, C, v);
    }
}

// HELD: h from its checkpoint.  dw in registers, one partial row a workgroup.  With
// two pieces a lane a workgroup of 1024 has no registers left for the weight and
// the next row: those rows load when they are needed.  Of those 16 kernels only the
// two of whole pieces on a bf16 residual without a checkpoint spill nothing, the
// others 2 to 37 registers (8192 x 16384 bf16 217 us, 4.9 TB/s; 8192 x 12287 fp32 472
// and 8192 x 12288 bf16 on fp32 rows with dropout and an int8 checkpoint 391, 3.4).
template <typename TX, typename TR, int VPT, bool RAG, bool HELD>
__global__ __launch_bounds__(1024) void residual_bwd_kernel(ResidualArgs a) {
    __shared__ float red[32];
    constexpr bool kAhead = VPT == 1;
    const DropKey key(a.drop);
    const int C = a.C, nb = (int)ck_blocks(C), stride = (int)ck_stride(C);
    const int64_t per = (C + 7) / 8;
    const TX* gy = static_cast<const TX*>(a.gy);
    const TR* gh = static_cast<const TR*>(a.gh);
    const TR* h = static_cast<const TR*>(a.h);
    float w[VPT][8], dw[VPT][8];
    if (kAhead) res_weights<VPT, RAG>(a, w);
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
#pragma unroll
        for (int e = 0; e < 8; ++e) dw[k][e] = 0.f;
    }
    CkPiece<TX> gn[VPT];
    CkPiece<TR> dn[VPT], hn[VPT];
    uint2 qn[VPT];
    uint32_t sn[VPT];
    const auto load = [&](int64_t b) {
        ck_row_load<TX, VPT, RAG>(gy + b * C, C, gn);
        if (gh) ck_row_load<TR, VPT, RAG>(gh + b * C, C, dn);
        if constexpr (HELD) {
#pragma unroll
            for (int k = 0; k < VPT; ++k) {
                int c0 = (k * blockDim.x + threadIdx.x) * 8;
                c0 = c0 < C ? c0 : 0;
                qn[k] = ld8_nt(a.hq + b * stride + c0);
                sn[k] = a.hsc[b * nb + (c0 >> 5)];
            }
        } else {
            ck_row_load<TR, VPT, RAG>(h + b * C, C, hn);
        }
    };
    int64_t b = blockIdx.x;
    if (kAhead) load(b);
    for (; b < a.B; b += gridDim.x) {
        if (!kAhead) {
            load(b);
            res_weights<VPT, RAG>(a, w);
        }
        float hv[VPT][8], g[VPT][8], d[VPT][8];
        ck_row_get<TX, VPT, RAG>(gy + b * C, C, gn, g);
        if constexpr (HELD) {
#pragma unroll
            for (int k = 0; k < VPT; ++k) {
                if (a.h_fmt == kCkInt8) ck_unpack8<kCkInt8>(qn[k], sn[k], hv[k]);
                else ck_unpack8<kCkE4M3>(qn[k], sn[k], hv[k]);
                if ((k * blockDim.x + threadIdx.x) * 8 >= C) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) hv[k][e] = 0.f;
                }
            }
        } else {
            ck_row_get<TR, VPT, RAG>(h + b * C, C, hn, hv);
        }
        if (gh) {
            ck_row_get<TR, VPT, RAG>(gh + b * C, C, dn, d);
        } else {
#pragma unroll
            for (int k = 0; k < VPT; ++k) {
#pragma unroll
                for (int e = 0; e < 8; ++e) d[k][e] = 0.f;
            }
        }
        if (kAhead) load(b + gridDim.x < a.B ? b + gridDim.x : b);
        float t[2] = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                t[0] += hv[k][e] * hv[k][e];
                t[1] += g[k][e] * w[k][e] * hv[k][e];
            }
        }
        block_sum<2>(t, red);
        const float inv = 1.f / sqrtf(t[0] / (float)C + a.eps);
        const float k2 = t[1] * inv * inv * inv / (float)C;
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                dw[k][e] += g[k][e] * hv[k][e] * inv;
                d[k][e] += w[k][e] * g[k][e] * inv - hv[k][e] * k2;
            }
        }
        if (a.gres) ck_row_put<TR, VPT, RAG, !RAG>(static_cast<TR*>(a.gres) + b * C, C, d);
        if (a.gx) {
            if (a.drop.threshold) {
#pragma unroll
                for (int k = 0; k < VPT; ++k)
                    key.apply(a.drop, (uint64_t)(b * per + k * blockDim.x + threadIdx.x), d[k]);
            }
            ck_row_put<TX, VPT, RAG, !RAG>(static_cast<TX*>(a.gx) + b * C, C, d);
        }
    }
    if (a.dw_part) ck_row_put<float, VPT, RAG>(a.dw_part + (int64_t)blockIdx.x * C, C, dw);
}

// ---------------------------------------------------------------------------
// Narrow rows, several a wave (CkNarrow of mhc_ckpt.h): no LDS in the sums.  400000 x
// 96 bf16 forward 50 us, 6.2 TB/s, backward 52, 5.9; 400000 x 100, rows on no 16-byte
// boundary, 80 and 66 us, 4.0 and 4.8 TB/s (streamed backward 70).  Twice the lanes a
// CU: forward 50 and 78 us, backward 7% slower.
// ---------------------------------------------------------------------------
template <bool RAG>
__device__ __forceinline__ void res_narrow_weight(const ResidualArgs& a, const CkNarrow<float, RAG>& ln,
                                                  float (&w)[8]) {
    if (a.w_dtype == kBF16) {
        CkPiece<bf16_t> p;
        ln.load(static_cast<const bf16_t*>(a.w), p);
        ln.get(static_cast<const bf16_t*>(a.w), p, w);
    } else {
        CkPiece<float> p;
        ln.load(static_cast<const float*>(a.w), p);
        ln.get(static_cast<const float*>(a.w), p, w);
    }
}

template <typename TX, typename TR, bool RAG>
__global__ __launch_bounds__(256) void residual_fwd_narrow_kernel(ResidualArgs a, int lg) {
    const DropKey key(a.drop);
    const int C = a.C;
    const double each = 1.0 / C;
    const CkNarrow<float, RAG> ln(C, lg);
    const CkNarrow<TX, RAG> lx(C, lg);
    const CkNarrow<TR, RAG> lr(C, lg);
    const int64_t per = (C + 7) / 8;
    const int lane = threadIdx.x & 63, rows = 64 >> lg, sub = lane >> lg;
    const int nb = (int)ck_blocks(C), stride = (int)ck_stride(C);
    float w[8];
    res_narrow_weight<RAG>(a, ln, w);
    const TX* x = static_cast<const TX*>(a.x);
    const TR* res = static_cast<const TR*>(a.residual);
    const int64_t step = (int64_t)gridDim.x * 4 * rows;
    int64_t b0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * rows;  // the wave's first row
    const auto at = [&](int64_t b) { return b + sub < a.B ? b + sub : a.B - 1; };
    const auto pack = [&](int fmt, const float (&v)[8], uint8_t* q, uint8_t* sc, int64_t row, bool on) {
        uint2 p;
        const uint32_t s = fmt == kCkInt8 ? ck_pack8<kCkInt8>(v, p) : ck_pack8<kCkE4M3>(v, p);
        if (on && ln.c0 < stride) st8_nt(q + row * stride + ln.c0, p);
        if (on && ln.in() && (lane & 3) == 0) sc[row * nb + (ln.c0 >> 5)] = (uint8_t)s;
    };
    CkPiece<TX> xn;
    CkPiece<TR> rn;
    ln.load(x + at(b0) * C, xn);
    ln.load(res + at(b0) * C, rn);
    for (; b0 < a.B; b0 += step) {
        const bool on = b0 + sub < a.B;
        const int64_t b = at(b0);
        float v[8], r[8];
        ln.get(x + b * C, xn, v);
        ln.get(res + b * C, rn, r);
        const int64_t b1 = at(b0 + step);
        ln.load(x + b1 * C, xn);
        ln.load(res + b1 * C, rn);
        if (a.drop.threshold) key.apply(a.drop, (uint64_t)(b * per + (ln.c0 >> 3)), v);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += r[e];
        res_round<TR>(v);
        if (on) lr.template put<false>(static_cast<TR*>(a.h) + b * C, v);
        if (a.h_fmt >= 0) pack(a.h_fmt, v, a.hq, a.hsc, b, on);
        if (a.y_fmt >= 0) {
            const ResInv inv(res_group_sum(res_square(v, 0.0), lg) * each + a.eps);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = inv.odd(v[e], w[e]);
            pack(a.y_fmt, v, a.yq, a.ysc, b, on);
            continue;
        }
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += v[e] * v[e];
        ss = lane_group_sum(ss, lg);
        const float inv = 1.f / sqrtf(ss / (float)C + a.eps);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = v[e] * inv * w[e];
        if (on) lx.template put<false>(static_cast<TX*>(a.y) + b * C, v);
    }
}

template <typename TX, typename TR, bool RAG, bool HELD>
__global__ __launch_bounds__(512) void residual_bwd_narrow_kernel(ResidualArgs a, int lg) {
    __shared__ float red[8 * kCkNarrow];
    const DropKey key(a.drop);
    const int C = a.C;
    const CkNarrow<float, RAG> ln(C, lg);
    const CkNarrow<TX, RAG> lx(C, lg);
    const CkNarrow<TR, RAG> lr(C, lg);
    const int64_t per = (C + 7) / 8;
    const int nb = (int)ck_blocks(C), stride = (int)ck_stride(C);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, rows = 64 >> lg, sub = lane >> lg;
    const TX* gy = static_cast<const TX*>(a.gy);
    const TR* gh = static_cast<const TR*>(a.gh);
    const TR* h = static_cast<const TR*>(a.h);
    float w[8], dw[8];
    res_narrow_weight<RAG>(a, ln, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[e] = 0.f;
    const int64_t step = (int64_t)gridDim.x * 8 * rows;
    int64_t b0 = ((int64_t)blockIdx.x * 8 + wave) * rows;
    const auto at = [&](int64_t b) { return b + sub < a.B ? b + sub : a.B - 1; };
    CkPiece<TX> gn;
    CkPiece<TR> dn, hn;
    uint2 qn;
    uint32_t sn;
    const auto load = [&](int64_t row) {
        ln.load(gy + row * C, gn);
        if (gh) ln.load(gh + row * C, dn);
        if constexpr (HELD) {
            const int c0 = ln.in() ? ln.c0 : 0;
            qn = ld8_nt(a.hq + row * stride + c0);
            sn = a.hsc[row * nb + (c0 >> 5)];
        } else {
            ln.load(h + row * C, hn);
        }
    };
    load(at(b0));
    for (; b0 < a.B; b0 += step) {
        const bool on = b0 + sub < a.B;
        const int64_t b = at(b0);
        float hv[8], g[8], d[8];
        ln.get(gy + b * C, gn, g);
        if constexpr (HELD) {
            if (a.h_fmt == kCkInt8) ck_unpack8<kCkInt8>(qn, sn, hv);
            else ck_unpack8<kCkE4M3>(qn, sn, hv);
#pragma unroll
            for (int e = 0; e < 8; ++e) hv[e] = ln.in() ? hv[e] : 0.f;
        } else {
            ln.get(h + b * C, hn, hv);
        }
        if (gh) {
            ln.get(gh + b * C, dn, d);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) d[e] = 0.f;
        }
        load(at(b0 + step));
        float ss = 0.f, dot = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            ss += hv[e] * hv[e];
            dot += g[e] * w[e] * hv[e];
        }
        ss = lane_group_sum(ss, lg);
        dot = lane_group_sum(dot, lg);
        const float inv = 1.f / sqrtf(ss / (float)C + a.eps);
        const float k2 = dot * inv * inv * inv / (float)C;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            dw[e] += on ? g[e] * hv[e] * inv : 0.f;
            d[e] += w[e] * g[e] * inv - hv[e] * k2;
        }
        if (a.gres && on) lr.template put<!RAG>(static_cast<TR*>(a.gres) + b * C, d);
        if (a.gx) {
            if (a.drop.threshold) key.apply(a.drop, (uint64_t)(b * per + (ln.c0 >> 3)), d);
            if (on) lx.template put<!RAG>(static_cast<TX*>(a.gx) + b * C, d);
        }
    }
    if (!a.dw_part) return;  // the whole grid
    // the wave's groups, the workgroup's waves
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        float v = dw[e];
        for (int k = 1 << lg; k < 64; k <<= 1) v += __shfl_xor(v, k);
        if (sub == 0 && ln.c0 + e < C) red[wave * C + ln.c0 + e] = v;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < C; i += 512) {
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) v += red[k * C + i];
        a.dw_part[(int64_t)blockIdx.x * C + i] = v;
    }
}

#define MHC_RES_TYPED(x_dt, r_dt, ...)                                                        \
    do {                                                                                      \
        auto typed = [&](auto x_, auto r_) {                                                  \
            using X_ = decltype(x_);                                                          \
            using R_ = decltype(r_);                                                          \
            __VA_ARGS__;                                                                      \
        };                                                                                    \
        if ((x_dt) == kBF16 && (r_dt) == kBF16) typed(bf16_t{}, bf16_t{});                    \
        else if ((x_dt) == kBF16) typed(bf16_t{}, float{});                                   \
        else if ((r_dt) == kBF16) typed(float{}, bf16_t{});                                   \
        else typed(float{}, float{});                                                         \
    } while (0)

// Calls f(integral_constant of the pieces a lane, true_type where rows end inside a piece).
template <typename F>
static void res_rows(int vpt, bool rag, F f) {
    const auto go = [&](auto v) {
        if (rag) f(v, std::true_type{});
        else f(v, std::false_type{});
    };
    if (vpt == 1) go(std::integral_constant<int, 1>{});
    else go(std::integral_constant<int, 2>{});
}
// The fewest pieces a lane that a workgroup of `most` lanes covers the row with, or
// two a lane of more.
static CkRowTiling res_tiling(int64_t C, int most) {
    const int64_t pieces = (C + 7) / 8;
    const int vpt = pieces <= most ? 1 : 2;
    return CkRowTiling{vpt, (int)(((pieces + vpt - 1) / vpt + 63) / 64 * 64)};
}
constexpr int kResFwdLanes = 512, kResBwdLanes = 1024;
template <typename F>
static void res_flag(bool on, F f) {
    if (on) f(std::true_type{});
    else f(std::false_type{});
}

// Workgroups of 1024 lanes a CU together, or as many as fit; 1536 where y leaves in
// 8 bits, which is bound by its instructions (16384 x 4096 bf16 to e4m3: 83 us with
// 1024, 79.5 with 1536, 80 with 2048; rows that share lines, 20000 x 2733 fp32, would
// rather have 1024: 141 us for 190).
static unsigned res_grid(const void* fn, int threads, int64_t most, int y_fmt) {
    int64_t per_cu = occupancy_per_cu(fn, threads, 0);
    const int lanes = y_fmt >= 0 ? 1536 : 1024;
    if (per_cu > lanes / threads) per_cu = lanes / threads;
    const int64_t g = (int64_t)device_cu_count() * per_cu;
    return (unsigned)(g < most ? g : most);
}

hipError_t launch_rmsnorm_residual_fwd(int x_dt, int r_dt, const ResidualArgs& a, hipStream_t s) {
    if (a.B == 0) return hipSuccess;
    const CkRowTiling t = res_tiling(a.C, kResFwdLanes);
    const bool rag = a.C % 8 != 0;
    const int tok = timing_begin("rmsnorm_residual_fwd", s);
    MHC_RES_TYPED(x_dt, r_dt, {
        if (a.C > kCkMaxRow) {
            const int64_t most = 2 * (int64_t)device_cu_count();
            MHC_LAUNCH_GGL((residual_fwd_any_kernel<X_, R_>), dim3((unsigned)(a.B < most ? a.B : most)),
                           dim3(kResAnyThreads), 0, s, a);
        } else if (a.C <= kCkNarrow) {
            const int lg = ck_narrow_lg(a.C);
            const int64_t each = 4 * (64 >> lg);
            res_flag(rag, [&](auto g) {
                constexpr bool G_ = decltype(g)::value;
                const void* fn = reinterpret_cast<const void*>(&residual_fwd_narrow_kernel<X_, R_, G_>);
                MHC_LAUNCH_GGL((residual_fwd_narrow_kernel<X_, R_, G_>),
                               dim3(res_grid(fn, 256, (a.B + each - 1) / each, a.y_fmt)), dim3(256), 0, s, a, lg);
            });
        } else {
            res_rows(t.vpt, rag, [&](auto v, auto g) {
                constexpr int V_ = decltype(v)::value;
                constexpr bool G_ = decltype(g)::value;
                const void* fn = reinterpret_cast<const void*>(&residual_fwd_kernel<X_, R_, V_, G_>);
                MHC_LAUNCH_GGL((residual_fwd_kernel<X_, R_, V_, G_>), dim3(res_grid(fn, t.threads, a.B, a.y_fmt)),
                               dim3(t.threads), 0, s, a);
            });
        }
    });
    timing_end(tok, s);
    return hipGetLastError();
}

int rmsnorm_residual_bwd_grid(int x_dt, int r_dt, int64_t B, int64_t C) {
    const int64_t cus = device_cu_count();
    int64_t g = 2 * cus, most = B;
    if (C <= kCkNarrow) {
        const int64_t each = 8 * (64 >> ck_narrow_lg(C));
        most = (B + each - 1) / each;
    } else if (C <= kCkMaxRow) {
        // as many workgroups as 1024 lanes a CU, where each has 16 rows: a partial
        // row of dw costs as many bytes as a row (two a CU at least)
        const int threads = res_tiling(C, kResBwdLanes).threads;
        int64_t per_cu = B / (16 * cus);
        if (per_cu > 1024 / threads) per_cu = 1024 / threads;
        if (per_cu > 2) g = per_cu * cus;
    }
    return (int)(g < most ? g : (most < 1 ? 1 : most));
}

hipError_t launch_rmsnorm_residual_bwd(int x_dt, int r_dt, const ResidualArgs& a, int grid, hipStream_t s) {
    if (a.B == 0) return hipSuccess;
    const CkRowTiling t = res_tiling(a.C, kResBwdLanes);
    const bool rag = a.C % 8 != 0;
    const int tok = timing_begin("rmsnorm_residual_bwd", s);
    MHC_RES_TYPED(x_dt, r_dt, {
        res_flag(a.h_fmt >= 0, [&](auto held) {
            constexpr bool H_ = decltype(held)::value;
            if (a.C > kCkMaxRow) {
                MHC_LAUNCH_GGL((residual_bwd_any_kernel<X_, R_>), dim3(grid), dim3(kResAnyThreads), 0, s, a);
            } else if (a.C <= kCkNarrow) {
                res_flag(rag, [&](auto g) {
                    MHC_LAUNCH_GGL((residual_bwd_narrow_kernel<X_, R_, decltype(g)::value, H_>), dim3(grid), dim3(512),
                                   0, s, a, ck_narrow_lg(a.C));
                });
            } else {
                res_rows(t.vpt, rag, [&](auto v, auto g) {
                    MHC_LAUNCH_GGL((residual_bwd_kernel<X_, R_, decltype(v)::value, decltype(g)::value, H_>),
                                   dim3(grid), dim3(t.threads), 0, s, a);
                });
            }
        });
    });
    timing_end(tok, s);
    return hipGetLastError();
}

}  // namespace mhc
