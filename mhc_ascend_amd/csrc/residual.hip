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
// Dropout.  A lane takes pieces of 8 channels, a block of numbers each.  Rows
// of a multiple of 8 are one run of pieces, U a lane; other rows go piece by
// piece with the row found by a 32-bit division.
// ---------------------------------------------------------------------------
constexpr int kDropU = 4;

template <typename T>
__global__ __launch_bounds__(256) void dropout_flat_kernel(const T* __restrict__ x, T* __restrict__ y, DropArgs d,
                                                           int64_t first, int64_t pieces) {
    const DropKey key(d);
    const int64_t p0 = first + (int64_t)blockIdx.x * (256 * kDropU) + threadIdx.x;
    CkPiece<T> in[kDropU];
#pragma unroll
    for (int u = 0; u < kDropU; ++u) {
        const int64_t p = p0 + u * 256;
        in[u].load(x + (p < pieces ? p : first) * 8);
    }
#pragma unroll
    for (int u = 0; u < kDropU; ++u) {
        const int64_t p = p0 + u * 256;
        float v[8];
        in[u].get(v);
        key.apply(d, (uint64_t)p, v);
        if (p < pieces) ck_store8(y + p * 8, v);
    }
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
        const int64_t pieces = rows * (C / 8), most = ((int64_t)1 << 23) * (256 * kDropU);  // 2^31 lanes a launch
        for (int64_t p = 0; p < pieces; p += most) {
            const int64_t n = pieces - p < most ? pieces - p : most;
            MHC_LAUNCH_GGL((dropout_flat_kernel<T>), dim3((unsigned)((n + 256 * kDropU - 1) / (256 * kDropU))),
                           dim3(256), 0, s, x, y, d, p, p + n);
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
// loop over the row and is read back by the lane that wrote it in the second.
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
        for (int e = 0; e < 8; ++e) v[e] = bf16_to_f32(f32_to_bf16(v[e]));
    }
}
__device__ __forceinline__ void res_weight(const ResidualArgs& a, int c0, float (&w)[8]) {
    if (a.w_dtype == kBF16) res_piece(static_cast<const bf16_t*>(a.w) + c0, a.C - c0, w);
    else res_piece(static_cast<const float*>(a.w) + c0, a.C - c0, w);
}
// A lane's 8 values of a row in 8 bits; every lane of a block of 32 takes part.
__device__ __forceinline__ void res_pack(int fmt, const float (&v)[8], uint8_t* __restrict__ q,
                                         uint8_t* __restrict__ sc, int64_t row, int C, int c0) {
    uint2 p;
    const uint32_t s = fmt == kCkInt8 ? ck_pack8<kCkInt8>(v, p) : ck_pack8<kCkE4M3>(v, p);
    if (c0 < (int)ck_stride(C)) st8_nt(q + row * ck_stride(C) + c0, p);
    if ((c0 & 31) == 0 && c0 < C) sc[row * ck_blocks(C) + (c0 >> 5)] = (uint8_t)s;
}
__device__ __forceinline__ void res_unpack(int fmt, const uint8_t* __restrict__ q, const uint8_t* __restrict__ sc,
                                           int64_t row, int C, int c0, float (&v)[8]) {
    const uint2 p = ld8_nt(q + row * ck_stride(C) + c0);
    const uint32_t s = sc[row * ck_blocks(C) + (c0 >> 5)];
    if (fmt == kCkInt8) ck_unpack8<kCkInt8>(p, s, v);
    else ck_unpack8<kCkE4M3>(p, s, v);
}

template <typename TX, typename TR>
__global__ __launch_bounds__(kResAnyThreads) void residual_fwd_any_kernel(ResidualArgs a) {
    __shared__ float red[16];
    const DropKey key(a.drop);
    const int C = a.C;
    const int64_t per = ((int64_t)C + 7) / 8;
    // whole blocks of 32, so that the lanes of one pack it together
    const int64_t end = ck_blocks(C) * kCkBlock;
    for (int64_t b = blockIdx.x; b < a.B; b += gridDim.x) {
        const TX* x = static_cast<const TX*>(a.x) + b * C;
        const TR* res = static_cast<const TR*>(a.residual) + b * C;
        TR* h = static_cast<TR*>(a.h) + b * C;
        float t[1] = {0.f};
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
            for (int e = 0; e < 8; ++e) {
                v[e] = e < m ? v[e] : 0.f;
                t[0] += v[e] * v[e];
            }
            if (a.h_fmt >= 0) res_pack(a.h_fmt, v, a.hq, a.hsc, b, C, c0);
        }
        block_sum<1>(t, red);
        const float inv = 1.f / sqrtf(t[0] / (float)C + a.eps);
        for (int64_t c = (int64_t)threadIdx.x * 8; c < end; c += kResAnyThreads * 8) {
            const int c0 = (int)c, m = c < C ? C - c0 : 0;
            float v[8], w[8];
            res_piece(h + (m > 0 ? c0 : 0), m, v);
            if (m > 0) {
                res_weight(a, c0, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = e < m ? v[e] * inv * w[e] : 0.f;
            }
            if (a.y_fmt >= 0) res_pack(a.y_fmt, v, a.yq, a.ysc, b, C, c0);
            else if (m > 0) res_put(static_cast<TX*>(a.y) + b * C + c0, m, v);
        }
    }
}

// dw is summed in the workgroup's own partial row, each channel by one lane.
template <typename TX, typename TR>
__global__ __launch_bounds__(kResAnyThreads) void residual_bwd_any_kernel(ResidualArgs a) {
    __shared__ float red[32];
    const DropKey key(a.drop);
    const int C = a.C;
    const int64_t per = ((int64_t)C + 7) / 8;
    for (int64_t b = blockIdx.x; b < a.B; b += gridDim.x) {
        const TX* gy = static_cast<const TX*>(a.gy) + b * C;
        const auto row = [&](int c0, int m, float (&v)[8]) {
            if (a.h_fmt >= 0) res_unpack(a.h_fmt, a.hq, a.hsc, b, C, c0, v);
            else res_piece(static_cast<const TR*>(a.h) + b * C + c0, m, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = e < m ? v[e] : 0.f;
        };
        float t[2] = {0.f, 0.f};
        for (int64_t c = (int64_t)threadIdx.x * 8; c < C; c += kResAnyThreads * 8) {
            const int c0 = (int)c, m = C - c0;
            float h[8], g[8], w[8];
            row(c0, m, h);
            res_piece(gy + c0, m, g);
            res_weight(a, c0, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                t[0] += h[e] * h[e];
                t[1] += g[e] * w[e] * h[e];
            }
        }
        block_sum<2>(t, red);
        const float inv = 1.f / sqrtf(t[0] / (float)C + a.eps);
        const float k2 = t[1] * inv * inv * inv / (float)C;
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

hipError_t launch_rmsnorm_residual_fwd(int x_dt, int r_dt, const ResidualArgs& a, hipStream_t s) {
    if (a.B == 0) return hipSuccess;
    const int tok = timing_begin("rmsnorm_residual_fwd", s);
    const int64_t most = 2 * (int64_t)device_cu_count();
    MHC_RES_TYPED(x_dt, r_dt,
                  MHC_LAUNCH_GGL((residual_fwd_any_kernel<X_, R_>), dim3((unsigned)(a.B < most ? a.B : most)),
                                 dim3(kResAnyThreads), 0, s, a));
    timing_end(tok, s);
    return hipGetLastError();
}

int rmsnorm_residual_bwd_grid(int x_dt, int r_dt, int64_t B, int64_t C) {
    const int64_t most = 2 * (int64_t)device_cu_count();
    return (int)(B < 1 ? 1 : (B < most ? B : most));
}

hipError_t launch_rmsnorm_residual_bwd(int x_dt, int r_dt, const ResidualArgs& a, int grid, hipStream_t s) {
    if (a.B == 0) return hipSuccess;
    const int tok = timing_begin("rmsnorm_residual_bwd", s);
    MHC_RES_TYPED(x_dt, r_dt,
                  MHC_LAUNCH_GGL((residual_bwd_any_kernel<X_, R_>), dim3(grid), dim3(kResAnyThreads), 0, s, a));
    timing_end(tok, s);
    return hipGetLastError();
}

}  // namespace mhc
