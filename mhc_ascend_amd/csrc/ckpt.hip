// 8-bit checkpoints of rows (the format of mhc_ckpt.h) and RMSNorm over them.
//
// RMSNorm with a checkpoint writes it in the pass that has the row in
// registers, and its backward reads it in place of the row:
//   forward   y = x / r * w,  r = sqrt(mean x^2 + eps);  x^ out
//   backward  the gradients of that at x^, r recomputed from x^:
//             dx = w g / r - x^ (sum_c g w x^) / (C r^3),  dw = sum_rows g x^ / r
#include <type_traits>

#include "mhc_ckpt.h"
#include "mhc_device.h"
#include "mhc_internal.h"

namespace mhc {

// ---------------------------------------------------------------------------
// Pack and unpack.  A lane takes pieces of 8 elements, 4 lanes a block of 32.
// Rows of a multiple of 32 are one run of blocks (the padded layout is then
// the plain one): U pieces a lane, all loads first.  Other rows go piece by
// piece with the row found by a 32-bit division.
// Both are bound by their bytes: 32768 x 4096 bf16, 65-66 us each way, 6.2 TB/s.
// ---------------------------------------------------------------------------
constexpr int kCkU = 4;

template <typename T, int FMT>
__global__ __launch_bounds__(256) void ckpt_pack_flat_kernel(const T* __restrict__ x, uint8_t* __restrict__ q,
                                                             uint8_t* __restrict__ sc, int64_t pieces) {
    const int64_t p0 = (int64_t)blockIdx.x * (256 * kCkU) + threadIdx.x;
    CkPiece<T> in[kCkU];
#pragma unroll
    for (int u = 0; u < kCkU; ++u) {
        const int64_t p = p0 + u * 256;
        in[u].load(x + (p < pieces ? p : 0) * 8);
    }
#pragma unroll
    for (int u = 0; u < kCkU; ++u) {
        const int64_t p = p0 + u * 256;
        float v[8];
        in[u].get(v);
        uint2 w;
        const uint32_t s = ck_pack8<FMT>(v, w);  // a block's four lanes are in or past the end together
        if (p < pieces) {
            st8_nt(q + p * 8, w);
            if ((threadIdx.x & 3) == 0) sc[p >> 2] = (uint8_t)s;
        }
    }
}

template <typename T, int FMT>
__global__ __launch_bounds__(256) void ckpt_unpack_flat_kernel(const uint8_t* __restrict__ q,
                                                               const uint8_t* __restrict__ sc, T* __restrict__ out,
                                                               int64_t pieces) {
    const int64_t p0 = (int64_t)blockIdx.x * (256 * kCkU) + threadIdx.x;
    uint2 w[kCkU];
    uint32_t s[kCkU];
#pragma unroll
    for (int u = 0; u < kCkU; ++u) {
        const int64_t p = p0 + u * 256;
        const int64_t pp = p < pieces ? p : 0;
        w[u] = ld8_nt(q + pp * 8);
        s[u] = sc[pp >> 2];
    }
#pragma unroll
    for (int u = 0; u < kCkU; ++u) {
        const int64_t p = p0 + u * 256;
        float v[8];
        ck_unpack8<FMT>(w[u], s[u], v);
        if (p < pieces) ck_store8(out + p * 8, v);
    }
}

// rows * 4 ck_blocks(C) < 2^31 pieces in a launch
template <typename T, int FMT>
__global__ __launch_bounds__(256) void ckpt_pack_rows_kernel(const T* __restrict__ x, uint8_t* __restrict__ q,
                                                             uint8_t* __restrict__ sc, uint32_t pieces, int C) {
    const uint32_t per = (uint32_t)ck_blocks(C) * 4u;
    const int64_t stride = ck_stride(C);
    const uint32_t p = blockIdx.x * 256u + threadIdx.x;
    const bool on = p < pieces;
    const uint32_t row = on ? p / per : 0u;
    const int c0 = (int)(on ? p - row * per : 0u) * 8;
    const int m = C - c0;
    float v[8];
    const T* xp = x + (int64_t)row * C + c0;
    if (m >= 8) {
        CkPiece<T> in;
        in.load(xp);
        in.get(v);
    } else {
        ck_load_part(xp, m, v);
    }
    uint2 w;
    const uint32_t s = ck_pack8<FMT>(v, w);
    if (on) {
        if (c0 < stride) st8_nt(q + row * stride + c0, w);
        if ((c0 & 31) == 0) sc[(int64_t)row * (per >> 2) + (c0 >> 5)] = (uint8_t)s;
    }
}

template <typename T, int FMT>
__global__ __launch_bounds__(256) void ckpt_unpack_rows_kernel(const uint8_t* __restrict__ q,
                                                               const uint8_t* __restrict__ sc, T* __restrict__ out,
                                                               uint32_t pieces, int C) {
    const uint32_t per = (uint32_t)ck_blocks(C) * 4u;
    const int64_t stride = ck_stride(C);
    const uint32_t p = blockIdx.x * 256u + threadIdx.x;
    if (p >= pieces) return;
    const uint32_t row = p / per;
    const int c0 = (int)(p - row * per) * 8;
    const int m = C - c0;
    if (m <= 0) return;
    float v[8];
    ck_unpack8<FMT>(ld8_nt(q + row * stride + c0), sc[(int64_t)row * (per >> 2) + (c0 >> 5)], v);
    T* op = out + (int64_t)row * C + c0;
    if (m >= 8) {
        ck_store8(op, v);
    } else {
        ck_store_part(op, m, v);
    }
}

// Calls f.template operator()<T, FMT>() of a storage type and a format.
#define MHC_CK_TYPED(dt, fmt, ...)                                                                      \
    do {                                                                                                \
        if ((dt) == kBF16) {                                                                            \
            using T_ = bf16_t;                                                                          \
            if ((fmt) == kCkInt8) { constexpr int F_ = kCkInt8; __VA_ARGS__; }                          \
            else { constexpr int F_ = kCkE4M3; __VA_ARGS__; }                                           \
        } else {                                                                                        \
            using T_ = float;                                                                           \
            if ((fmt) == kCkInt8) { constexpr int F_ = kCkInt8; __VA_ARGS__; }                          \
            else { constexpr int F_ = kCkE4M3; __VA_ARGS__; }                                           \
        }                                                                                               \
    } while (0)

template <typename Flat, typename Rows>
static hipError_t ckpt_run(int64_t rows, int64_t C, Flat flat, Rows ragged) {
    if (rows == 0) return hipSuccess;
    if (C % kCkBlock == 0) {
        // whole blocks: at most 2^23 workgroups (2^31 lanes) a launch
        const int64_t pieces = rows * (C / 8), most = ((int64_t)1 << 23) * (256 * kCkU);
        for (int64_t p = 0; p < pieces; p += most) {
            const int64_t n = pieces - p < most ? pieces - p : most;
            flat(p, n, (unsigned)((n + 256 * kCkU - 1) / (256 * kCkU)));
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return e;
        }
        return hipSuccess;
    }
    const int64_t per = ck_blocks(C) * 4;
    const int64_t most = ((int64_t)1 << 30) / per;  // rows a launch
    for (int64_t r = 0; r < rows; r += most) {
        const int64_t n = (rows - r < most ? rows - r : most) * per;
        ragged(r, (uint32_t)n, (unsigned)((n + 255) / 256));
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

hipError_t launch_ckpt_pack(int dt, int fmt, const void* x, void* values, void* scales, int64_t rows, int64_t C,
                            hipStream_t s) {
    uint8_t* q = (uint8_t*)values;
    uint8_t* sc = (uint8_t*)scales;
    const int tok = timing_begin("ckpt_pack", s);
    hipError_t e = hipSuccess;
    MHC_CK_TYPED(dt, fmt, {
        const T_* xs = (const T_*)x;
        e = ckpt_run(
            rows, C,
            [&](int64_t p, int64_t n, unsigned grid) {
                MHC_LAUNCH_GGL((ckpt_pack_flat_kernel<T_, F_>), dim3(grid), dim3(256), 0, s, xs + p * 8, q + p * 8,
                               sc + p / 4, n);
            },
            [&](int64_t r, uint32_t n, unsigned grid) {
                MHC_LAUNCH_GGL((ckpt_pack_rows_kernel<T_, F_>), dim3(grid), dim3(256), 0, s, xs + r * C,
                               q + r * ck_stride(C), sc + r * ck_blocks(C), n, (int)C);
            });
    });
    timing_end(tok, s);
    return e;
}

hipError_t launch_ckpt_unpack(int dt, int fmt, const void* values, const void* scales, void* out, int64_t rows,
                              int64_t C, hipStream_t s) {
    const uint8_t* q = (const uint8_t*)values;
    const uint8_t* sc = (const uint8_t*)scales;
    const int tok = timing_begin("ckpt_unpack", s);
    hipError_t e = hipSuccess;
    MHC_CK_TYPED(dt, fmt, {
        T_* os = (T_*)out;
        e = ckpt_run(
            rows, C,
            [&](int64_t p, int64_t n, unsigned grid) {
                MHC_LAUNCH_GGL((ckpt_unpack_flat_kernel<T_, F_>), dim3(grid), dim3(256), 0, s, q + p * 8, sc + p / 4,
                               os + p * 8, n);
            },
            [&](int64_t r, uint32_t n, unsigned grid) {
                MHC_LAUNCH_GGL((ckpt_unpack_rows_kernel<T_, F_>), dim3(grid), dim3(256), 0, s, q + r * ck_stride(C),
                               sc + r * ck_blocks(C), os + r * C, n, (int)C);
            });
    });
    timing_end(tok, s);
    return e;
}

// Persistent workgroups over rows, the weight in registers and the next row's
// loads in flight.  Bound by its bytes: 16384 x 4096 bf16 in 64 us, 5.3 TB/s
// (forward and backward 130 us, 155 with one workgroup a row).
template <typename T, int FMT, int VPT, bool RAG>
__global__ __launch_bounds__(512) void rmsnorm_ckpt_fwd_kernel(const T* __restrict__ x, const float* __restrict__ w,
                                                               T* __restrict__ y, uint8_t* __restrict__ q,
                                                               uint8_t* __restrict__ sc, int64_t B, int C, float eps) {
    __shared__ float red[8];
    const int nb = (int)ck_blocks(C), stride = (int)ck_stride(C);
    float wv[VPT][8];
    CkPiece<T> in[VPT];
    int64_t b = blockIdx.x;
    ck_row_load<T, VPT, RAG>(x + b * C, C, in);
    {
        CkPiece<float> wr[VPT];
        ck_row_load<float, VPT, RAG>(w, C, wr);
        ck_row_get<float, VPT, RAG>(w, C, wr, wv);
    }
    for (; b < B; b += gridDim.x) {
        float v[VPT][8];
        ck_row_get<T, VPT, RAG>(x + b * C, C, in, v);
        const int64_t b1 = b + gridDim.x;
        ck_row_load<T, VPT, RAG>(x + (b1 < B ? b1 : b) * C, C, in);
        float t[1] = {0.f};
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
#pragma unroll
            for (int e = 0; e < 8; ++e) t[0] += v[k][e] * v[k][e];
        }
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            const int c0 = (k * blockDim.x + threadIdx.x) * 8;
            uint2 p;
            const uint32_t s = ck_pack8<FMT>(v[k], p);
            if (c0 < stride) st8_nt(q + b * stride + c0, p);
            if ((threadIdx.x & 3) == 0 && c0 < C) sc[b * nb + (c0 >> 5)] = (uint8_t)s;
        }
        block_sum<1>(t, red);
        const float inv = 1.f / sqrtf(t[0] / (float)C + eps);
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[k][e] = v[k][e] * inv * wv[k][e];
        }
        ck_row_put<T, VPT, RAG>(y + b * C, C, v);
    }
}

// Persistent workgroups over rows, the next row's loads in flight; dw in
// registers, one partial row a workgroup.  Bound by its bytes: 16384 x 4096 bf16
// in 65 us, 5.2 TB/s.
template <typename T, int FMT, int VPT, bool RAG>
__global__ __launch_bounds__(512) void rmsnorm_ckpt_bwd_kernel(const T* __restrict__ g,
                                                               const uint8_t* __restrict__ q,
                                                               const uint8_t* __restrict__ sc,
                                                               const float* __restrict__ w, T* __restrict__ gx,
                                                               float* __restrict__ dw_part, int64_t B, int C,
                                                               float eps) {
    __shared__ float red[16];
    const int nb = (int)ck_blocks(C), stride = (int)ck_stride(C);
    float wv[VPT][8], dw[VPT][8];
    {
        CkPiece<float> wr[VPT];
        ck_row_load<float, VPT, RAG>(w, C, wr);
        ck_row_get<float, VPT, RAG>(w, C, wr, wv);
    }
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
#pragma unroll
        for (int e = 0; e < 8; ++e) dw[k][e] = 0.f;
    }
    uint2 qn[VPT];
    uint32_t sn[VPT];
    CkPiece<T> gn[VPT];
    auto load = [&](int64_t b) {
        ck_row_load<T, VPT, RAG>(g + b * C, C, gn);
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            int c0 = (k * blockDim.x + threadIdx.x) * 8;
            c0 = c0 < C ? c0 : 0;
            qn[k] = ld8_nt(q + b * stride + c0);
            sn[k] = sc[b * nb + (c0 >> 5)];
        }
    };
    int64_t b = blockIdx.x;
    load(b);
    for (; b < B; b += gridDim.x) {
        float xv[VPT][8], gv[VPT][8];
        ck_row_get<T, VPT, RAG>(g + b * C, C, gn, gv);
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            const int c0 = (k * blockDim.x + threadIdx.x) * 8;
            ck_unpack8<FMT>(qn[k], sn[k], xv[k]);
            if (c0 >= C) {
#pragma unroll
                for (int e = 0; e < 8; ++e) xv[k][e] = 0.f;
            }
        }
        const int64_t b1 = b + gridDim.x;
        load(b1 < B ? b1 : b);
        float t[2] = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                t[0] += xv[k][e] * xv[k][e];
                t[1] += gv[k][e] * wv[k][e] * xv[k][e];
            }
        }
        block_sum<2>(t, red);
        const float inv = 1.f / sqrtf(t[0] / (float)C + eps);
        const float k2 = t[1] * inv * inv * inv / (float)C;
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                dw[k][e] += gv[k][e] * xv[k][e] * inv;
                gv[k][e] = wv[k][e] * gv[k][e] * inv - xv[k][e] * k2;
            }
        }
        ck_row_put<T, VPT, RAG>(gx + b * C, C, gv);
    }
    ck_row_put<float, VPT, RAG>(dw_part + (int64_t)blockIdx.x * C, C, dw);
}

// ---------------------------------------------------------------------------
// Narrow rows, several a wave (CkNarrow).  Forward and backward, against a
// workgroup a row: 35334 x 104 bf16 23 us for 44, 65536 x 256 bf16 45 for 63,
// 65536 x 512 bf16 75 for 86, 30000 x 500 fp32 78 for 88; 1000 x 400 bf16 17 for
// 17.  Bound by bytes from 256 channels on.
// ---------------------------------------------------------------------------
template <typename T, int FMT, bool RAG>
__global__ __launch_bounds__(256) void rmsnorm_ckpt_fwd_narrow_kernel(const T* __restrict__ x,
                                                                      const float* __restrict__ w, T* __restrict__ y,
                                                                      uint8_t* __restrict__ q, uint8_t* __restrict__ sc,
                                                                      int64_t B, int C, int lg, float eps) {
    const CkNarrow<T, RAG> ln(C, lg);
    const int nb = (int)ck_blocks(C), stride = (int)ck_stride(C);
    const int lane = threadIdx.x & 63, rows = 64 >> lg, sub = lane >> lg;
    float wv[8];
    {
        CkPiece<float> p;
        ln.load(w, p);
        ln.get(w, p, wv);
    }
    const int64_t step = (int64_t)gridDim.x * 4 * rows;
    int64_t b0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * rows;  // the wave's first row
    const auto at = [&](int64_t b) { return b + sub < B ? b + sub : B - 1; };
    CkPiece<T> in;
    ln.load(x + at(b0) * C, in);
    for (; b0 < B; b0 += step) {
        const int64_t b = b0 + sub;
        float v[8];
        ln.get(x + at(b0) * C, in, v);
        ln.load(x + at(b0 + step) * C, in);
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += v[e] * v[e];
        uint2 p;
        const uint32_t s = ck_pack8<FMT>(v, p);
        if (b < B && ln.c0 < stride) st8_nt(q + b * stride + ln.c0, p);
        if (b < B && ln.in() && (lane & 3) == 0) sc[b * nb + (ln.c0 >> 5)] = (uint8_t)s;
        ss = lane_group_sum(ss, lg);
        const float inv = 1.f / sqrtf(ss / (float)C + eps);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = v[e] * inv * wv[e];
        if (b < B) ln.put(y + b * C, v);
    }
}

template <typename T, int FMT, bool RAG>
__global__ __launch_bounds__(512) void rmsnorm_ckpt_bwd_narrow_kernel(const T* __restrict__ g,
                                                                      const uint8_t* __restrict__ q,
                                                                      const uint8_t* __restrict__ sc,
                                                                      const float* __restrict__ w, T* __restrict__ gx,
                                                                      float* __restrict__ dw_part, int64_t B, int C,
                                                                      int lg, float eps) {
    __shared__ float red[8 * kCkNarrow];
    const CkNarrow<T, RAG> ln(C, lg);
    const int nb = (int)ck_blocks(C), stride = (int)ck_stride(C);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, rows = 64 >> lg, sub = lane >> lg;
    float wv[8], dw[8];
    {
        CkPiece<float> p;
        ln.load(w, p);
        ln.get(w, p, wv);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[e] = 0.f;
    const int64_t step = (int64_t)gridDim.x * 8 * rows;
    int64_t b0 = ((int64_t)blockIdx.x * 8 + wave) * rows;
    const auto at = [&](int64_t b) { return b + sub < B ? b + sub : B - 1; };
    CkPiece<T> gn;
    uint2 qn;
    uint32_t sn;
    const auto load = [&](int64_t row) {
        ln.load(g + row * C, gn);
        const int c0 = ln.in() ? ln.c0 : 0;
        qn = ld8_nt(q + row * stride + c0);
        sn = sc[row * nb + (c0 >> 5)];
    };
    load(at(b0));
    for (; b0 < B; b0 += step) {
        const bool on = b0 + sub < B;
        const int64_t b = at(b0);
        float xv[8], gv[8];
        ln.get(g + b * C, gn, gv);
        ck_unpack8<FMT>(qn, sn, xv);
        load(at(b0 + step));
        float ss = 0.f, dot = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            xv[e] = ln.in() ? xv[e] : 0.f;
            ss += xv[e] * xv[e];
            dot += gv[e] * wv[e] * xv[e];
        }
        ss = lane_group_sum(ss, lg);
        dot = lane_group_sum(dot, lg);
        const float inv = 1.f / sqrtf(ss / (float)C + eps);
        const float k2 = dot * inv * inv * inv / (float)C;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            dw[e] += on ? gv[e] * xv[e] * inv : 0.f;
            gv[e] = wv[e] * gv[e] * inv - xv[e] * k2;
        }
        if (on) ln.put(gx + b * C, gv);
    }
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
        dw_part[(int64_t)blockIdx.x * C + i] = v;
    }
}

// ---------------------------------------------------------------------------
// Sums of a weight gradient's partials part[rows][cols] over rows, 32 columns a
// workgroup in 32 phases of rows (each in order, then the phases in order):
// 512 rows take two rounds of eight loads a lane and one LDS sum.  Bound by the
// latency of those: 256 columns 4 us, with 256 lanes on 64 columns 9.6.
// ---------------------------------------------------------------------------
template <typename TW>
__global__ __launch_bounds__(1024) void weight_grad_sum_kernel(const float* __restrict__ part, int rows, int cols,
                                                     TW* __restrict__ dw) {
    __shared__ float red[32][33];
    const int cl = threadIdx.x & 31, ph = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + cl;
    float s = 0.f;
    if (c < cols) {
        int r = ph;
        for (; r + 7 * 32 < rows; r += 8 * 32) {
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = part[(int64_t)(r + u * 32) * cols + c];
#pragma unroll
            for (int u = 0; u < 8; ++u) s += v[u];
        }
        for (; r < rows; r += 32) s += part[(int64_t)r * cols + c];
    }
    red[ph][cl] = s;
    __syncthreads();
    if (ph == 0 && c < cols) {
        float t = 0.f;
#pragma unroll
        for (int k = 0; k < 32; ++k) t += red[k][cl];
        VecIO<TW>::put(dw + c, t);
    }
}

hipError_t launch_weight_grad_sum(int w_dtype, const float* part, int rows, int64_t cols, void* dw, hipStream_t s) {
    if (cols < 1 || cols > 0x7fffffff) return hipErrorInvalidValue;
    const dim3 grid((unsigned)((cols + 31) / 32));
    if (w_dtype == kBF16) {
        MHC_LAUNCH_GGL((weight_grad_sum_kernel<bf16_t>), grid, dim3(1024), 0, s, part, rows, (int)cols, (bf16_t*)dw);
    } else {
        MHC_LAUNCH_GGL((weight_grad_sum_kernel<float>), grid, dim3(1024), 0, s, part, rows, (int)cols, (float*)dw);
    }
    return hipGetLastError();
}

bool rmsnorm_ckpt_supported(int64_t C) { return C >= 1 && C <= kCkMaxRow; }

#define MHC_CK_NARROW(dt, fmt, rag, ...)                                                 \
    MHC_CK_TYPED(dt, fmt, {                                                              \
        if (rag) { constexpr bool R_ = true; __VA_ARGS__; }                              \
        else { constexpr bool R_ = false; __VA_ARGS__; }                                 \
    })

#define MHC_CK_ROWS(dt, fmt, vpt, rag, ...)                                              \
    MHC_CK_TYPED(dt, fmt, {                                                              \
        auto pick = [&](auto v_) {                                                       \
            constexpr int V_ = decltype(v_)::value;                                      \
            if (rag) { constexpr bool R_ = true; __VA_ARGS__; }                          \
            else { constexpr bool R_ = false; __VA_ARGS__; }                             \
        };                                                                               \
        if ((vpt) == 1) pick(std::integral_constant<int, 1>{});                          \
        else if ((vpt) == 2) pick(std::integral_constant<int, 2>{});                     \
        else pick(std::integral_constant<int, 4>{});                                     \
    })

hipError_t launch_rmsnorm_ckpt_fwd(int dt, int fmt, const void* x, const float* w, void* y, void* values,
                                   void* scales, int64_t B, int64_t C, float eps, hipStream_t s) {
    if (B == 0) return hipSuccess;
    if (!rmsnorm_ckpt_supported(C) || B > 0x7fffffff) return hipErrorInvalidValue;
    const CkRowTiling t = ck_row_tiling(C);
    const bool rag = C % 8 != 0;
    const int tok = timing_begin("rmsnorm_ckpt_fwd", s);
    if (C <= kCkNarrow) {
        const int lg = ck_narrow_lg(C);
        const int64_t each = 4 * (64 >> lg), most = (B + each - 1) / each;
        MHC_CK_NARROW(dt, fmt, rag, {
            const void* fn = reinterpret_cast<const void*>(&rmsnorm_ckpt_fwd_narrow_kernel<T_, F_, R_>);
            const int64_t g = (int64_t)device_cu_count() * occupancy_per_cu(fn, 256, 0);
            MHC_LAUNCH_GGL((rmsnorm_ckpt_fwd_narrow_kernel<T_, F_, R_>), dim3((unsigned)(g < most ? g : most)),
                           dim3(256), 0, s, (const T_*)x, w, (T_*)y, (uint8_t*)values, (uint8_t*)scales, B, (int)C, lg,
                           eps);
        });
        timing_end(tok, s);
        return hipGetLastError();
    }
    MHC_CK_ROWS(dt, fmt, t.vpt, rag, {
        const void* fn = reinterpret_cast<const void*>(&rmsnorm_ckpt_fwd_kernel<T_, F_, V_, R_>);
        const int64_t g = (int64_t)device_cu_count() * occupancy_per_cu(fn, t.threads, 0);
        MHC_LAUNCH_GGL((rmsnorm_ckpt_fwd_kernel<T_, F_, V_, R_>), dim3((unsigned)(g < B ? g : B)), dim3(t.threads), 0,
                       s, (const T_*)x, w, (T_*)y, (uint8_t*)values, (uint8_t*)scales, B, (int)C, eps);
    });
    timing_end(tok, s);
    return hipGetLastError();
}

int rmsnorm_ckpt_bwd_grid(int dt, int fmt, int64_t B, int64_t C) {
    if (C <= kCkNarrow) {
        const int64_t each = 8 * (64 >> ck_narrow_lg(C)), most = (B + each - 1) / each;
        const int64_t g = 2 * (int64_t)device_cu_count();
        return (int)(g < most ? g : (most < 1 ? 1 : most));
    }
    const CkRowTiling t = ck_row_tiling(C);
    const bool rag = C % 8 != 0;
    const void* fn = nullptr;
    MHC_CK_ROWS(dt, fmt, t.vpt, rag, fn = reinterpret_cast<const void*>(&rmsnorm_ckpt_bwd_kernel<T_, F_, V_, R_>));
    // at most two workgroups a CU, or as many of 1024 lanes together where each
    // still has 16 rows: their partial rows of dw cost as many bytes as rows of x
    // (2999 x 1001 fp32: 2560 workgroups 20.7 us and 8.8 for their partials, 512
    // of them 14.4 and 3.6)
    int64_t per_cu = occupancy_per_cu(fn, t.threads, 0), most = B / (16 * (int64_t)device_cu_count());
    if (most > 1024 / t.threads) most = 1024 / t.threads;
    if (most < 2) most = 2;
    if (per_cu > most) per_cu = most;
    const int64_t g = (int64_t)device_cu_count() * per_cu;
    return (int)(g < B ? g : (B < 1 ? 1 : B));
}

hipError_t launch_rmsnorm_ckpt_bwd(int dt, int fmt, const void* g, const void* values, const void* scales,
                                   const float* w, void* gx, float* dw_part, int grid, int64_t B, int64_t C,
                                   float eps, hipStream_t s) {
    if (B == 0) return hipSuccess;
    if (!rmsnorm_ckpt_supported(C)) return hipErrorInvalidValue;
    const CkRowTiling t = ck_row_tiling(C);
    const bool rag = C % 8 != 0;
    const int tok = timing_begin("rmsnorm_ckpt_bwd", s);
    if (C <= kCkNarrow) {
        MHC_CK_NARROW(dt, fmt, rag,
                      MHC_LAUNCH_GGL((rmsnorm_ckpt_bwd_narrow_kernel<T_, F_, R_>), dim3(grid), dim3(512), 0, s,
                                     (const T_*)g, (const uint8_t*)values, (const uint8_t*)scales, w, (T_*)gx, dw_part,
                                     B, (int)C, ck_narrow_lg(C), eps));
        timing_end(tok, s);
        return hipGetLastError();
    }
    MHC_CK_ROWS(dt, fmt, t.vpt, rag,
                MHC_LAUNCH_GGL((rmsnorm_ckpt_bwd_kernel<T_, F_, V_, R_>), dim3(grid), dim3(t.threads), 0, s,
                               (const T_*)g, (const uint8_t*)values, (const uint8_t*)scales, w, (T_*)gx, dw_part, B,
                               (int)C, eps));
    timing_end(tok, s);
    return hipGetLastError();
}

}  // namespace mhc
