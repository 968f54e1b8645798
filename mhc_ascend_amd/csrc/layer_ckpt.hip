// The fused layer's register-row passes with the token rows in 8 bits
// (mhc_ckpt.h): the forward writes the checkpoint of the row it holds, the
// backward reads the row x^ from it.  Arithmetic per token as the kernels of
// layer.hip (mhc_layer_rows.h), n = 2..8 on rows those take, 16-byte aligned
// arrays; other shapes run layer.hip / wide.hip / generic.hip with a pack or
// unpack pass.
//
// A lane holds 4 channels of a chunk, so 8 lanes a block of 32: the block's
// maximum is three DPP steps.  Both passes are bound by their bytes; the
// pack pass (a second read of x) and the unpack pass (x^ written and read)
// are what they save.  8192 x 4 x 4096: fp32 forward 201-209 us (5.8-6.0 TB/s),
// backward 205-227 (5.3-5.9); bf16 forward 160 (5.9), backward of the dynamic
// layer 165-178 (5.3-5.7).  With a pack and an unpack pass the fp32 step took 780 us,
// with these 413.
#include "mhc_ckpt.h"
#include "mhc_device.h"
#include "mhc_internal.h"
#include "mhc_layer_rows.h"
#include "mhc_rows.h"

namespace mhc {

// ---------------------------------------------------------------------------
// Rows to and from the checkpoint, through buffer resources over one token's
// values [N][stride] and scales [N][nb] (no access behind a branch).
// ---------------------------------------------------------------------------
__device__ __forceinline__ uint32_t held_ld4(buf_rsrc_t r, uint32_t off) {
    return (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(r, (int)off, 0, 2);
}
__device__ __forceinline__ uint32_t held_ld1(buf_rsrc_t r, uint32_t off) {
    return (uint32_t)(uint8_t)__builtin_amdgcn_raw_buffer_load_b8(r, (int)off, 0, 0);
}

template <int N, int VPT>
struct HeldRows {
    uint32_t q[N][VPT];  // 4 values
    uint32_t s[N][VPT];  // their block's scale byte
};

// Lanes past the row read zeros, and a token past the end (no bytes) too:
// zeros stand for 0.
template <int N, int VPT>
__device__ __forceinline__ void held_load(const uint8_t* __restrict__ q, const uint8_t* __restrict__ sc, int64_t b,
                                          int64_t B, int C, HeldRows<N, VPT>& r) {
    const int stride = (int)ck_stride(C), nb = (int)ck_blocks(C);
    const int64_t bb = b < B ? b : 0;
    const buf_rsrc_t rq = make_buf_rsrc(q + bb * N * stride, b < B ? (uint32_t)(N * stride) : 0u);
    const buf_rsrc_t rs = make_buf_rsrc(sc + bb * N * nb, b < B ? (uint32_t)(N * nb) : 0u);
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        const int c0 = (k * blockDim.x + threadIdx.x) * kLayerWC;
        const uint32_t oq = c0 < C ? (uint32_t)c0 : kBufOff, os = c0 < C ? (uint32_t)(c0 >> 5) : kBufOff;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            r.q[i][k] = held_ld4(rq, oq + (uint32_t)(i * stride));
            r.s[i][k] = held_ld1(rs, os + (uint32_t)(i * nb));
        }
    }
}

template <int FMT, int N, int VPT>
__device__ __forceinline__ void held_get_as(const HeldRows<N, VPT>& r, float (&v)[N][VPT][kLayerWC]) {
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
#pragma unroll
        for (int i = 0; i < N; ++i) Ck<FMT>::unpack4(r.q[i][k], Ck<FMT>::down(r.s[i][k]), v[i][k]);
    }
}
// The format is an argument (a scalar branch once a token): half the kernels.
template <int N, int VPT>
__device__ __forceinline__ void held_get(int fmt, const HeldRows<N, VPT>& r, float (&v)[N][VPT][kLayerWC]) {
    if (fmt == kCkInt8) held_get_as<kCkInt8, N, VPT>(r, v);
    else held_get_as<kCkE4M3, N, VPT>(r, v);
}

template <int FMT, int N, int VPT>
__device__ __forceinline__ void held_put_as(const float (&v)[N][VPT][kLayerWC], uint8_t* __restrict__ q,
                                         uint8_t* __restrict__ sc, int64_t b, int C) {
    const int stride = (int)ck_stride(C), nb = (int)ck_blocks(C);
    const buf_rsrc_t rq = make_buf_rsrc(q + b * N * stride, (uint32_t)(N * stride));
    const buf_rsrc_t rs = make_buf_rsrc(sc + b * N * nb, (uint32_t)(N * nb));
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        const int c0 = (k * blockDim.x + threadIdx.x) * kLayerWC;
        const uint32_t oq = c0 < stride ? (uint32_t)c0 : kBufOff;  // the padding too
        const uint32_t os = c0 < C && (threadIdx.x & 7) == 0 ? (uint32_t)(c0 >> 5) : kBufOff;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float(&f)[kLayerWC] = v[i][k];
            uint32_t a = ck_abs_bits(f[0]);
#pragma unroll
            for (int e = 1; e < kLayerWC; ++e) a = a > ck_abs_bits(f[e]) ? a : ck_abs_bits(f[e]);
            const uint32_t s = Ck<FMT>::scale(ck_group_max<8>(a));
            const uint32_t w = Ck<FMT>::pack4(f[0], f[1], f[2], f[3], Ck<FMT>::up(s), s == 255u ? 0u : ~0u);
            __builtin_amdgcn_raw_buffer_store_b32(w, rq, (int)(oq + (uint32_t)(i * stride)), 0, 2);
            __builtin_amdgcn_raw_buffer_store_b8((uint8_t)s, rs, (int)(os + (uint32_t)(i * nb)), 0, 0);
        }
    }
}

template <int N, int VPT>
__device__ __forceinline__ void held_put(int fmt, const float (&v)[N][VPT][kLayerWC], uint8_t* __restrict__ q,
                                         uint8_t* __restrict__ sc, int64_t b, int C) {
    if (fmt == kCkInt8) held_put_as<kCkInt8, N, VPT>(v, q, sc, b, C);
    else held_put_as<kCkE4M3, N, VPT>(v, q, sc, b, C);
}

template <typename TX, int N, int VPT>
__global__ MHC_ROW_BOUNDS(false) void layer_ckpt_fwd_kernel(int fmt, const TX* __restrict__ x, const float* __restrict__ w,
                                                            const float* __restrict__ coef, int64_t coef_stride,
                                                            float* __restrict__ out, uint8_t* __restrict__ q,
                                                            uint8_t* __restrict__ sc, int C, float eps) {
    constexpr int WC = kLayerWC;
    __shared__ float red[8];
    const int64_t b = blockIdx.x;  // one token per workgroup
    RawRows<TX, N, VPT, WC> xr;
    load_rows_raw<TX, N, VPT, WC, true>(x + b * (int64_t)N * C, C, xr);
    float wv[VPT][WC];
    load_weight<VPT, WC>(w, C, wv);
    float xv[N][VPT][WC];
    unpack_rows<TX, N, VPT, WC>(xr, C, xv);
    held_put<N, VPT>(fmt, xv, q, sc, b, C);
    fwd_token<TX, float, N, VPT>(b, coef, coef_stride, wv, xv, out, nullptr, C, eps, red);
}

// Static H's saved state in a launch of its own: workgroup 0 the coefficients,
// by the code of the kernel below (so the same bits at any number of tokens),
// the others the weight in fp32, 4 a lane.
template <int N>
__global__ __launch_bounds__(256) void layer_ckpt_coef_kernel(const void* __restrict__ weight, int w_bf16,
                                                              const float* __restrict__ h_pre,
                                                              const float* __restrict__ h_post,
                                                              const float* __restrict__ h_res,
                                                              float* __restrict__ saved, int w_off, int iters,
                                                              float sk_eps, int C) {
    __shared__ float cf[coef_size<N>()];
    if (blockIdx.x == 0) {
        if (threadIdx.x < kWave) static_coefs_wave<N>(h_pre, h_post, h_res, iters, sk_eps, cf, saved);
        return;
    }
    const int c0 = ((blockIdx.x - 1) * 256 + threadIdx.x) * 4;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (c0 + e < C)
            saved[w_off + c0 + e] = w_bf16 ? VecIO<bf16_t>::scalar(static_cast<const bf16_t*>(weight) + c0 + e)
                                           : static_cast<const float*>(weight)[c0 + e];
}

// Static H in one launch, as layer_static_fwd_kernel: every workgroup forms the
// shared coefficients while its row loads are in flight, workgroup 0 writes the
// saved state.  For few tokens.
template <typename TX, int N, int VPT>
__global__ MHC_ROW_BOUNDS(false) void layer_ckpt_static_fwd_kernel(
    int fmt, const TX* __restrict__ x, const void* __restrict__ weight, int w_bf16, const float* __restrict__ h_pre,
    const float* __restrict__ h_post, const float* __restrict__ h_res, float* __restrict__ saved, int w_off, int iters,
    float sk_eps, float* __restrict__ out, uint8_t* __restrict__ q, uint8_t* __restrict__ sc, int C, float eps) {
    constexpr int WC = kLayerWC;
    __shared__ float red[8];
    __shared__ float cf[coef_size<N>()];
    const int64_t b = blockIdx.x;
    RawRows<TX, N, VPT, WC> xr;
    load_rows_raw<TX, N, VPT, WC, true>(x + b * (int64_t)N * C, C, xr);
    if (threadIdx.x < kWave) static_coefs_wave<N>(h_pre, h_post, h_res, iters, sk_eps, cf, b == 0 ? saved : nullptr);
    float wv[VPT][WC];
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        const int c0 = (k * blockDim.x + threadIdx.x) * WC;
#pragma unroll
        for (int e = 0; e < WC; ++e) {
            wv[k][e] = 0.f;
            if (c0 < C)
                wv[k][e] = w_bf16 ? VecIO<bf16_t>::scalar(static_cast<const bf16_t*>(weight) + c0 + e)
                                  : static_cast<const float*>(weight)[c0 + e];
        }
        if (b == 0 && c0 < C) store_run<float, WC>(saved + w_off + c0, wv[k]);
    }
    __syncthreads();
    float xv[N][VPT][WC];
    unpack_rows<TX, N, VPT, WC>(xr, C, xv);
    held_put<N, VPT>(fmt, xv, q, sc, b, C);
    fwd_token<TX, float, N, VPT>(b, cf, 0, wv, xv, out, nullptr, C, eps, red);
}

// As layer_bwd_kernel: persistent workgroups over tokens, with PF the next
// token's rows in flight.  TX is dx's storage type.
template <typename TX, int N, int VPT, int MODE, bool PF>
__global__ MHC_ROW_BOUNDS((PF && N * VPT > 8)) void layer_ckpt_bwd_kernel(int fmt, const float* __restrict__ g, const uint8_t* __restrict__ q,
                                                         const uint8_t* __restrict__ sc, const float* __restrict__ w,
                                                         const float* __restrict__ coef, int64_t coef_stride,
                                                         BwdDx<TX, MODE>* __restrict__ dx,
                                                         float* __restrict__ dw_part, float* __restrict__ scal_out,
                                                         int32_t* __restrict__ dx_scale, int64_t B, int C, float eps) {
    constexpr int WC = kLayerWC;
    constexpr int NS = N * N + 2 * N;
    constexpr int NR = 2 + N * N + 3 * N;
    __shared__ float red[9 * NR];  // 8 wave partials + totals
    float wv[VPT][WC];
    load_weight<VPT, WC>(w, C, wv);
    float dwacc[VPT][WC];
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
#pragma unroll
        for (int e = 0; e < WC; ++e) dwacc[k][e] = 0.f;
    }
    float sacc = 0.f;
    const int64_t G = gridDim.x;
    int64_t b = blockIdx.x;
    float xv[N][VPT][WC], gv[N][VPT][WC];
    const auto token = [&](int64_t t, const HeldRows<N, VPT>& xr, const RawRows<float, N, VPT, WC>& gr) {
        held_get<N, VPT>(fmt, xr, xv);
        unpack_rows<float, N, VPT, WC>(gr, C, gv);
        bwd_token<TX, N, VPT, MODE, true>(t, coef, coef_stride, wv, xv, gv, dwacc, sacc, dx, scal_out, dx_scale, C, eps, red);
    };
    if constexpr (PF) {
        HeldRows<N, VPT> xA, xB;
        RawRows<float, N, VPT, WC> gA, gB;
        held_load<N, VPT>(q, sc, b, B, C, xA);
        load_rows_raw_rs<float, N, VPT, WC, true>(token_rows_rsrc(g, b, B, N, C), C, gA);
        while (b < B) {
            const int64_t b1 = b + G;
            held_load<N, VPT>(q, sc, b1, B, C, xB);
            load_rows_raw_rs<float, N, VPT, WC, true>(token_rows_rsrc(g, b1, B, N, C), C, gB);
            token(b, xA, gA);
            if (b1 >= B) break;
            const int64_t b2 = b1 + G;
            held_load<N, VPT>(q, sc, b2, B, C, xA);
            load_rows_raw_rs<float, N, VPT, WC, true>(token_rows_rsrc(g, b2, B, N, C), C, gA);
            token(b1, xB, gB);
            b = b2;
        }
    } else {
        for (; b < B; b += G) {
            HeldRows<N, VPT> xr;
            RawRows<float, N, VPT, WC> gr;
            held_load<N, VPT>(q, sc, b, B, C, xr);
            load_rows_raw<float, N, VPT, WC, true>(g + b * (int64_t)N * C, C, gr);
            token(b, xr, gr);
        }
    }
    float* dwp = dw_part + (int64_t)blockIdx.x * C;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        const int c0 = (k * blockDim.x + threadIdx.x) * WC;
        if (c0 < C) store_run<float, WC>(dwp + c0, dwacc[k]);
    }
    if (MODE == 0 && threadIdx.x < NS) scal_out[(int64_t)blockIdx.x * NS + threadIdx.x] = sacc;
}

// ---------------------------------------------------------------------------
// Host launchers
// ---------------------------------------------------------------------------
#define MHC_CL_VPT(v, ...)                                       \
    switch (v) {                                                 \
        case 1: { constexpr int V_ = 1; __VA_ARGS__; break; }    \
        case 2: { constexpr int V_ = 2; __VA_ARGS__; break; }    \
        case 4: { constexpr int V_ = 4; __VA_ARGS__; break; }    \
        case 8: { constexpr int V_ = 8; __VA_ARGS__; break; }    \
        default: break;                                          \
    }
#define MHC_CL_N(n, ...)                                         \
    switch (n) {                                                 \
        case 2: { constexpr int N_ = 2; __VA_ARGS__; break; }    \
        case 3: { constexpr int N_ = 3; __VA_ARGS__; break; }    \
        case 4: { constexpr int N_ = 4; __VA_ARGS__; break; }    \
        case 5: { constexpr int N_ = 5; __VA_ARGS__; break; }    \
        case 6: { constexpr int N_ = 6; __VA_ARGS__; break; }    \
        case 7: { constexpr int N_ = 7; __VA_ARGS__; break; }    \
        case 8: { constexpr int N_ = 8; __VA_ARGS__; break; }    \
        default: break;                                          \
    }

template <typename TX, int N, int V>
static const void* ck_fwd_fn() {
    if constexpr (layer_row_fits(N, V)) return reinterpret_cast<const void*>(&layer_ckpt_fwd_kernel<TX, N, V>);
    return nullptr;
}

template <typename TX, int N, int V>
static const void* ck_static_fwd_fn() {
    if constexpr (layer_row_fits(N, V)) return reinterpret_cast<const void*>(&layer_ckpt_static_fwd_kernel<TX, N, V>);
    return nullptr;
}

template <typename TX, int N, int V, int MODE>
static const void* ck_bwd_fn(bool pf) {
    if constexpr (layer_row_fits(2 * N, V))
        return pf ? reinterpret_cast<const void*>(&layer_ckpt_bwd_kernel<TX, N, V, MODE, true>)
                  : reinterpret_cast<const void*>(&layer_ckpt_bwd_kernel<TX, N, V, MODE, false>);
    return nullptr;
}

static const void* pick_ck_fwd(int x_dtype, int n, int vpt) {
    const void* fn = nullptr;
    MHC_CL_N(n, MHC_CL_VPT(vpt, fn = x_dtype == kBF16 ? ck_fwd_fn<bf16_t, N_, V_>() : ck_fwd_fn<float, N_, V_>()));
    return fn;
}

// modes of bwd_token: bf16 rows take 0, 2 and, n = 2 and 4, 1; fp32 rows 0 and 1
template <int N, int V>
static const void* pick_ck_bwd_mode(int x_dtype, int mode, bool pf) {
    const bool bf = x_dtype == kBF16;
    if (mode == 0) return bf ? ck_bwd_fn<bf16_t, N, V, 0>(pf) : ck_bwd_fn<float, N, V, 0>(pf);
    if (mode == 2) return bf ? ck_bwd_fn<bf16_t, N, V, 2>(pf) : nullptr;
    if (!bf) return ck_bwd_fn<float, N, V, 1>(pf);
    if constexpr (N == 2 || N == 4) return ck_bwd_fn<bf16_t, N, V, 1>(pf);
    return nullptr;
}

static const void* pick_ck_bwd(int x_dtype, int n, int vpt, int mode, bool pf) {
    const void* fn = nullptr;
    MHC_CL_N(n, MHC_CL_VPT(vpt, fn = pick_ck_bwd_mode<N_, V_>(x_dtype, mode, pf)));
    return fn;
}

static bool ck_aligned(std::initializer_list<const void*> ps) {
    for (const void* p : ps)
        if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return false;
    return true;
}

bool layer_ckpt_fwd_rows(int n, int64_t B, int64_t C, std::initializer_list<const void*> ps) {
    return n >= 2 && n <= 8 && B > 0 && B <= 0x7fffffff && layer_fwd_tiling(C, n).vpt > 0 && ck_aligned(ps);
}

bool layer_ckpt_bwd_rows(int n, int64_t B, int64_t C, std::initializer_list<const void*> ps) {
    return n >= 2 && n <= 8 && B > 0 && layer_bwd_tiling(C, n, B).vpt > 0 && ck_aligned(ps);
}

hipError_t launch_layer_ckpt_fwd(int x_dtype, int fmt, int n, const void* x, const float* w, const float* coef,
                                 int64_t coef_stride, float* out, void* values, void* scales, int64_t B, int64_t C,
                                 float eps, hipStream_t s) {
    const RowTiling t = layer_fwd_tiling(C, n);
    const void* fn = pick_ck_fwd(x_dtype, n, t.vpt);
    if (!fn) return hipErrorInvalidValue;
    int Ci = (int)C;
    void* args[] = {(void*)&fmt, (void*)&x,   (void*)&w,      (void*)&coef,   (void*)&coef_stride, (void*)&out,
                    (void*)&values, (void*)&scales, (void*)&Ci, (void*)&eps};
    const int tok = timing_begin("layer_ckpt_fwd", s);
    hipError_t e = mhc_launch_kernel(fn, dim3((unsigned)B), dim3(t.threads), args, 0, s);
    timing_end(tok, s);
    return e != hipSuccess ? e : hipGetLastError();
}

hipError_t launch_layer_ckpt_coef(int n, const float* h_pre, const float* h_post, const float* h_res,
                                  const void* weight, int w_dtype, int64_t C, float* saved, int iters, float sk_eps,
                                  hipStream_t s) {
    const dim3 grid((unsigned)(1 + (C + 1023) / 1024));
    MHC_CL_N(n, MHC_LAUNCH_GGL((layer_ckpt_coef_kernel<N_>), grid, dim3(256), 0, s, weight, w_dtype == kBF16, h_pre,
                               h_post, h_res, saved, saved_w_offset(n), iters, sk_eps, (int)C));
    return hipGetLastError();
}

hipError_t launch_layer_ckpt_static_fwd(int x_dtype, int fmt, int n, const void* x, const void* weight, int w_dtype,
                                        const float* h_pre, const float* h_post, const float* h_res, float* saved,
                                        int iters, float sk_eps, float* out, void* values, void* scales, int64_t B,
                                        int64_t C, float eps, hipStream_t s) {
    const RowTiling t = layer_fwd_tiling(C, n);
    const void* fn = nullptr;
    MHC_CL_N(n, MHC_CL_VPT(t.vpt, fn = x_dtype == kBF16 ? ck_static_fwd_fn<bf16_t, N_, V_>()
                                                        : ck_static_fwd_fn<float, N_, V_>()));
    if (!fn) return hipErrorInvalidValue;
    int Ci = (int)C, w_bf16 = w_dtype == kBF16, w_off = saved_w_offset(n);
    void* args[] = {(void*)&fmt,   (void*)&x,     (void*)&weight, (void*)&w_bf16, (void*)&h_pre,
                    (void*)&h_post, (void*)&h_res, (void*)&saved,  (void*)&w_off,  (void*)&iters,
                    (void*)&sk_eps, (void*)&out,   (void*)&values, (void*)&scales, (void*)&Ci,
                    (void*)&eps};
    const int tok = timing_begin("layer_ckpt_fwd", s);
    hipError_t e = mhc_launch_kernel(fn, dim3((unsigned)B), dim3(t.threads), args, 0, s);
    timing_end(tok, s);
    return e != hipSuccess ? e : hipGetLastError();
}

// Workgroups of at most 256 lanes prefetch (layer.hip), and of 512 where two
// tokens' raw rows and the current one's values fit 256 registers and the CUs
// walk several tokens (n = 4, 320 x 1280 fp32: 8.9 us with, 7.0 without).
static bool ck_prefetch(const RowTiling& t, int n, int64_t B) {
    return t.threads <= 256 || (n * t.vpt <= 8 && B >= 4 * (int64_t)device_cu_count());
}
// One chunk a lane from n = 5 on too, where bwd_tiling takes two: half the raw
// words leave room for the prefetch (4096 tokens: n = 8, 1280 fp32 102 -> 93 us, n
// = 7, 1184 fp32 82 -> 76; n = 5, 1600 bf16 56 -> 61).
// Modes 1 and 2 on half the chunks and twice the lanes where a lane would hold
// 16 chunks: two waves a SIMD, one's sums under the other's loads (n = 4, 8192
// x 4096, bf16 dx: 174 us for 198).  Mode 0 keeps one more sum a lane and spills
// there (fp32: 310 us for 206).
static RowTiling ck_bwd_tiling(int64_t C, int n, int64_t B, int mode) {
    RowTiling t = with_min_threads(choose_row_tiling(C, kLayerWC, 2 * n, 256), 2 + n * n + 3 * n);
    if (mode != 0 && t.threads == 256 && t.vpt >= 2 && n * t.vpt == 16) {
        t.vpt /= 2;
        t.threads = 512;
    }
    return t;
}

int layer_ckpt_bwd_part_groups(int n, int64_t B, int64_t C) { return ck_bwd_tiling(C, n, B, 1).threads / 32; }

int layer_ckpt_bwd_grid(int x_dtype, int n, int mode, int64_t B, int64_t C) {
    const RowTiling t = ck_bwd_tiling(C, n, B, mode);
    const bool pf = ck_prefetch(t, n, B);
    int64_t per_cu = occupancy_per_cu(pick_ck_bwd(x_dtype, n, t.vpt, mode, pf), t.threads, 0);
    // A workgroup that prefetches wants eight tokens: it starts on none and ends
    // with a row of dw (n = 6, 2047 x 1040: one a CU 35.4 us, two 37.7); narrow
    // ones fill 512 lanes a CU all the same (n = 6, 3238 x 256 fp32, the dynamic
    // step: 110 us, 124 with one wave a CU).
    int64_t most = B / (8 * (int64_t)device_cu_count());
    if (most < 512 / t.threads) most = 512 / t.threads;
    if (pf && per_cu > most) per_cu = most;
    const int64_t g = (int64_t)device_cu_count() * per_cu;
    return (int)(g < B ? g : (B < 1 ? 1 : B));
}

hipError_t launch_layer_ckpt_bwd(int x_dtype, int fmt, int n, int mode, const float* g, const void* values,
                                 const void* scales, const float* w, const float* coef, int64_t coef_stride, void* dx,
                                 float* dw_part, float* scal_out, int grid, int64_t B, int64_t C, float eps,
                                 hipStream_t s, int32_t* dx_scale) {
    const RowTiling t = ck_bwd_tiling(C, n, B, mode);
    const void* fn = pick_ck_bwd(x_dtype, n, t.vpt, mode, ck_prefetch(t, n, B));
    if (!fn) return hipErrorInvalidValue;
    int Ci = (int)C;
    void* args[] = {(void*)&fmt, (void*)&g,       (void*)&values,   (void*)&scales,   (void*)&w, (void*)&coef, (void*)&coef_stride, (void*)&dx,
                    (void*)&dw_part, (void*)&scal_out, (void*)&dx_scale, (void*)&B, (void*)&Ci,   (void*)&eps};
    const int tok = timing_begin("layer_ckpt_bwd", s);
    hipError_t e = mhc_launch_kernel(fn, dim3(grid), dim3(t.threads), args, 0, s);
    timing_end(tok, s);
    return e != hipSuccess ? e : hipGetLastError();
}

}  // namespace mhc
