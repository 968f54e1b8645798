// RMSNorm of every head of queries and keys and the rotation of their
// positions, one pass each way.  For one head row x of D channels, weight w:
//   y = x / r * w,  r = sqrt(mean x^2 + eps)
//   (a, b) -> (a c - b s, b c + a s)  for the pairs of the first R channels,
//   pair p = (p, p + R/2), or (2p, 2p + 1) interleaved; c, s = table row of the
//   token's position, column p.  Channels past R stay.
// Backward, for cotangent z of the output: u = the rotation by the negative
// angle of z, dx = w u / r - x (sum u w x) / (D r^3), dw = sum over rows of
// u x / r.  With a checkpoint (mhc_ckpt.h) the forward writes x^ and the
// backward reads it in place of x, r from it as well.
//
// A position outside the table makes its rows NaN: the table is read inside
// its bounds only.
#include <type_traits>

#include "mhc_ckpt.h"
#include "mhc_device.h"
#include "mhc_internal.h"

namespace mhc {

__device__ __forceinline__ float qk_weight(const QkArgs& a, int s, int d) {
    return a.w_dtype == kBF16 ? bf16_to_f32(static_cast<const bf16_t*>(a.w[s])[d])
                              : static_cast<const float*>(a.w[s])[d];
}

// The table row of token t, or -1 where there is none.
__device__ __forceinline__ int64_t qk_position(const QkArgs& a, int64_t t) {
    const uint32_t i = (uint32_t)t % (uint32_t)a.period;
    int64_t p = i;
    if (a.pos_bytes == 8) p = static_cast<const int64_t*>(a.pos)[i];
    if (a.pos_bytes == 4) p = static_cast<const int32_t*>(a.pos)[i];
    return p >= 0 && p < a.table_rows ? p : -1;
}

// Where channel d stands in its pair: the table column, the other channel and
// the sign of the sine in d's output.  False past the rotated channels.
__device__ __forceinline__ bool qk_pair(const QkArgs& a, int d, int& col, int& other, float& sign) {
    if (d >= a.R) return false;
    bool hi;
    if (a.interleaved) {
        col = d >> 1;
        other = d ^ 1;
        hi = d & 1;
    } else {
        const int half = a.R >> 1;
        hi = d >= half;
        col = hi ? d - half : d;
        other = hi ? d - half : d + half;
    }
    sign = hi ? 1.f : -1.f;
    return true;
}

// ---------------------------------------------------------------------------
// Any head size, stride and alignment: one wave a head row, one channel a
// lane at a time.  A block of 32 channels is half a wave.
// ---------------------------------------------------------------------------
template <typename T, int FMT>
__global__ __launch_bounds__(256) void qk_fwd_any_kernel(QkArgs a) {
    const int lane = threadIdx.x & 63;
    const int hh = blockIdx.y * 4 + (threadIdx.x >> 6);
    if (hh >= a.heads[0] + a.heads[1]) return;  // whole waves, no barrier below
    const int64_t t = blockIdx.x;
    const int s = hh < a.heads[0] ? 0 : 1;
    const int h = s ? hh - a.heads[0] : hh;
    const T* x = static_cast<const T*>(a.x[s]) + t * a.x_token[s] + h * a.x_head[s];
    const int64_t row = t * a.heads[s] + h;
    T* y = static_cast<T*>(a.y[s]) + row * a.D;
    const int64_t pos = qk_position(a, t);
    float ss = 0.f;
    const int dmax = (a.D + 63) & ~63;
    for (int d = lane; d < dmax; d += 64) {
        const float v = d < a.D ? VecIO<T>::scalar(x + d) : 0.f;
        ss += v * v;
        if constexpr (FMT >= 0) {
            uint32_t m = ck_group_max<16>(ck_abs_bits(v));
            const auto p = __builtin_amdgcn_permlane16_swap(m, m, false, false);
            m = p[0] > p[1] ? p[0] : p[1];
            const uint32_t sc = Ck<FMT>::scale(m);
            const uint32_t w = Ck<FMT>::pack4(v, 0.f, 0.f, 0.f, Ck<FMT>::up(sc), sc == 255u ? 0u : 255u);
            if (d < (int)ck_stride(a.D)) a.q[s][row * ck_stride(a.D) + d] = (uint8_t)w;
            if ((lane & 31) == 0 && d < a.D) a.sc[s][row * ck_blocks(a.D) + (d >> 5)] = (uint8_t)sc;
        }
    }
    ss = group_sum<64>(ss);
    const float inv = pos < 0 ? __uint_as_float(0x7fc00000u) : 1.f / sqrtf(ss / (float)a.D + a.eps);
    const int64_t tab = (pos < 0 ? 0 : pos) * (int64_t)(a.R >> 1);
    for (int d = lane; d < a.D; d += 64) {
        float o = VecIO<T>::scalar(x + d) * inv * qk_weight(a, s, d);
        int col, other;
        float sign;
        if (qk_pair(a, d, col, other, sign)) {
            const float v = VecIO<T>::scalar(x + other) * inv * qk_weight(a, s, other);
            o = o * a.cos[tab + col] + sign * v * a.sin[tab + col];
        }
        VecIO<T>::put(y + d, o);
    }
}

// x[] is the row itself (FMT < 0) or its checkpoint in q / sc; y[] the
// gradient rows; g the cotangents.  Persistent workgroups over tokens, dw in
// LDS (every channel belongs to one lane of a wave), one partial row a
// workgroup: dw_part[grid][2 D], queries then keys.
template <typename T, int FMT>
__global__ __launch_bounds__(256) void qk_bwd_any_kernel(QkArgs a, float* __restrict__ dw_part) {
    extern __shared__ float dw[];  // [4 waves][2][D]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int i = threadIdx.x; i < 8 * a.D; i += 256) dw[i] = 0.f;
    __syncthreads();
    for (int64_t t = blockIdx.x; t < a.T; t += gridDim.x) {
        const int64_t pos = qk_position(a, t);
        const int64_t tab = (pos < 0 ? 0 : pos) * (int64_t)(a.R >> 1);
        for (int hh = wave; hh < a.heads[0] + a.heads[1]; hh += 4) {
            const int s = hh < a.heads[0] ? 0 : 1;
            const int h = s ? hh - a.heads[0] : hh;
            const int64_t row = t * a.heads[s] + h;
            const T* g = static_cast<const T*>(a.g[s]) + t * a.g_token[s] + h * a.g_head[s];
            T* dx = static_cast<T*>(a.y[s]) + row * a.D;
            auto x_at = [&](int d) {
                if constexpr (FMT >= 0) {
                    float v[4];
                    Ck<FMT>::unpack4(a.q[s][row * ck_stride(a.D) + d],
                                     Ck<FMT>::down(a.sc[s][row * ck_blocks(a.D) + (d >> 5)]), v);
                    return v[0];
                } else {
                    return VecIO<T>::scalar(static_cast<const T*>(a.x[s]) + t * a.x_token[s] + h * a.x_head[s] + d);
                }
            };
            auto u_at = [&](int d) {
                const float v = VecIO<T>::scalar(g + d);
                int col, other;
                float sign;
                if (!qk_pair(a, d, col, other, sign)) return v;
                return v * a.cos[tab + col] - sign * VecIO<T>::scalar(g + other) * a.sin[tab + col];
            };
            float ss = 0.f, dot = 0.f;
            for (int d = lane; d < a.D; d += 64) {
                const float v = x_at(d);
                ss += v * v;
                dot += u_at(d) * qk_weight(a, s, d) * v;
            }
            ss = group_sum<64>(ss);
            dot = group_sum<64>(dot);
            const float inv = pos < 0 ? __uint_as_float(0x7fc00000u) : 1.f / sqrtf(ss / (float)a.D + a.eps);
            const float k2 = dot * inv * inv * inv / (float)a.D;
            float* dws = dw + (wave * 2 + s) * a.D;
            for (int d = lane; d < a.D; d += 64) {
                const float v = x_at(d), u = u_at(d);
                VecIO<T>::put(dx + d, qk_weight(a, s, d) * u * inv - v * k2);
                dws[d] += u * v * inv;
            }
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * a.D; i += 256) {
        float v = 0.f;
        for (int w = 0; w < 4; ++w) v += dw[w * 2 * a.D + i];
        dw_part[(int64_t)blockIdx.x * 2 * a.D + i] = v;
    }
}

// ---------------------------------------------------------------------------
// Host launchers
// ---------------------------------------------------------------------------
#define MHC_QK_TYPED(dt, fmt, ...)                                            \
    do {                                                                      \
        auto pick = [&](auto f_) {                                            \
            constexpr int F_ = decltype(f_)::value;                           \
            if ((dt) == kBF16) { using T_ = bf16_t; __VA_ARGS__; }            \
            else { using T_ = float; __VA_ARGS__; }                           \
        };                                                                    \
        if ((fmt) < 0) pick(std::integral_constant<int, -1>{});               \
        else if ((fmt) == kCkInt8) pick(std::integral_constant<int, kCkInt8>{}); \
        else pick(std::integral_constant<int, kCkE4M3>{});                    \
    } while (0)

hipError_t launch_qk_norm_rope_fwd(int dt, int fmt, const QkArgs& a, hipStream_t s) {
    const int H = a.heads[0] + a.heads[1];
    if (a.T == 0 || H == 0) return hipSuccess;
    const int tok = timing_begin("qk_norm_rope_fwd", s);
    MHC_QK_TYPED(dt, fmt,
                 MHC_LAUNCH_GGL((qk_fwd_any_kernel<T_, F_>), dim3((unsigned)a.T, (unsigned)((H + 3) / 4)), dim3(256),
                                0, s, a));
    timing_end(tok, s);
    return hipGetLastError();
}

int qk_norm_rope_bwd_grid(int64_t T) {
    const int64_t g = 2 * (int64_t)device_cu_count();
    return (int)(T < g ? (T < 1 ? 1 : T) : g);
}

hipError_t launch_qk_norm_rope_bwd(int dt, int fmt, const QkArgs& a, float* dw_part, int grid, hipStream_t s) {
    const int tok = timing_begin("qk_norm_rope_bwd", s);
    MHC_QK_TYPED(dt, fmt,
                 MHC_LAUNCH_GGL((qk_bwd_any_kernel<T_, F_>), dim3((unsigned)grid), dim3(256),
                                (size_t)a.D * 8 * sizeof(float), s, a, dw_part));
    timing_end(tok, s);
    return hipGetLastError();
}

}  // namespace mhc
