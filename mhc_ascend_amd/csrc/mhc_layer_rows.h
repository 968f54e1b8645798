// The per-token arithmetic of the fused layer's register-row kernels (layer.hip,
// and layer_ckpt.hip, whose rows come from or go to an 8-bit checkpoint): one
// workgroup holds a token's row, as the formulas at the head of layer.hip.
#pragma once

#include <type_traits>

#include "mhc_device.h"
#include "mhc_internal.h"
#include "mhc_rows.h"

namespace mhc {

template <int N> constexpr int coef_size() { return 2 * N + N * N; }

// The shared N x N matrix (N = 3..8) on lanes 0 .. S^2 - 1 of one wave, one
// element per lane: `at` = the lane's element r N + c when `on`.  The wave's
// other lanes compute on zeros.
template <int N>
struct SkShared {
    static constexpr int S = sk_el_size(N);
    int at;
    bool on;
    float er, ec;
    __device__ __forceinline__ SkShared(int lane, float eps) {
        const int r = (lane / S) % S, c = lane % S;
        at = r * N + c;
        on = lane < S * S && r < N && c < N;
        er = SkEl<S>::pad_eps(r, N, eps);
        ec = SkEl<S>::pad_eps(c, N, eps);
    }
    __device__ __forceinline__ void forward(float& a, int iters) const { SkEl<S>::forward(a, iters, er, ec); }
    __device__ __forceinline__ void backward(float& g, float x0, int iters) const {
        SkEl<S>::backward(g, x0, iters, er, ec, on);
    }
};

// The shared coefficients of static H, by the first wave; each value goes to cf (LDS) and, when `save` is
// not null, to the saved state.
template <int N>
__device__ __forceinline__ void static_coefs_wave(const float* __restrict__ h_pre, const float* __restrict__ h_post,
                                                  const float* __restrict__ h_res, int iters, float eps,
                                                  float* __restrict__ cf, float* __restrict__ save) {
    const int r = threadIdx.x;
    auto put = [&](int i, float v) {
        cf[i] = v;
        if (save) save[i] = v;
    };
    if (r < N) {
        put(r, sigmoidf(h_pre[r]));
        put(N + r, 2.f * sigmoidf(h_post[r]));
    }
    if constexpr (N >= 3) {
        const SkShared<N> k(r, eps);
        float a = k.on ? expf(h_res[k.at]) : 0.f;
        k.forward(a, iters);
        if (k.on) put(2 * N + k.at, a);
    } else {
        float a[N];
#pragma unroll
        for (int c = 0; c < N; ++c) a[c] = (r < N) ? expf(h_res[r * N + c]) : 0.f;
        sk_forward<N>(a, iters, eps, r < N);
        if (r < N) {
#pragma unroll
            for (int c = 0; c < N; ++c) put(2 * N + r * N + c, a[c]);
        }
    }
}

template <typename TX, typename TO, int N, int VPT>
__device__ __forceinline__ void fwd_token(int64_t b, const float* __restrict__ coef, int64_t coef_stride,
                                          const float (&wv)[VPT][kLayerWC],
                                          const float (&xv)[N][VPT][kLayerWC], TO* __restrict__ out,
                                          float* __restrict__ rms_out, int C, float eps, float* red) {
    constexpr int WC = kLayerWC;
    constexpr int NC = coef_size<N>();
    const float* cf = coef + b * coef_stride;
    float cfv[NC];
#pragma unroll
    for (int k = 0; k < NC; ++k) cfv[k] = cf[k];
    float xa[VPT][WC];
    float ss = 0.f;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
#pragma unroll
        for (int e = 0; e < WC; ++e) {
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < N; ++i) s += cfv[i] * xv[i][k][e];
            xa[k][e] = s;
            ss += s * s;
        }
    }
    float v[1] = {ss};
    block_sum<1>(v, red);
    const float r = sqrtf(v[0] / (float)C + eps);
    const float inv = 1.f / r;
    // stores through a resource over the token's output rows, out-of-range
    // offsets past the row end (no store behind a branch)
    const buf_rsrc_t ors = make_buf_rsrc(out + b * (int64_t)N * C, (uint32_t)((int64_t)N * C * (int64_t)sizeof(TO)));
    static_assert(WC == 4, "4-channel chunks: one 16-byte (fp32) or 8-byte (bf16) store");
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        const int c0 = (k * blockDim.x + threadIdx.x) * WC;
        const uint32_t o0 = c0 < C ? (uint32_t)c0 * (uint32_t)sizeof(TO) : kBufOff;
        float y[WC];
#pragma unroll
        for (int e = 0; e < WC; ++e) y[e] = xa[k][e] * inv * wv[k][e];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float o[WC];
#pragma unroll
            for (int e = 0; e < WC; ++e) {
                float s = kTermLast<N> ? 0.f : cfv[N + i] * y[e];
#pragma unroll
                for (int j = 0; j < N; ++j) s += cfv[2 * N + i * N + j] * xv[j][k][e];
                o[e] = kTermLast<N> ? s + cfv[N + i] * y[e] : s;
            }
            const uint32_t off = o0 + (uint32_t)(i * C * (int)sizeof(TO));
            if constexpr (sizeof(TO) == 4) {
                buf_st16<true>(ors, off, 0u, make_uint4(__float_as_uint(o[0]), __float_as_uint(o[1]),
                                                        __float_as_uint(o[2]), __float_as_uint(o[3])));
            } else {
                buf_st8<true>(ors, off, 0u, make_uint2(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])));
            }
        }
    }
    if (rms_out) {
        const buf_rsrc_t rrs = make_buf_rsrc(rms_out + b, 4u);
        buf_st4(rrs, threadIdx.x == 0 ? 0u : kBufOff, 0u, r);
    }
}

// Wave totals of NV values with each total in one lane: a step folds the
// values of two lanes in pairs, so one lane goes on with the first half of the
// values and its partner with the second.  About 2.3 instructions a value in
// place of wave_sum_last's 6 (n = 4: 70 of 180), which the backward's row sums
// are a sixth of.  Returns the number of values a lane is left with; lane l's
// slot i holds the total of value fold_index(l, i) where that is below NV.
template <int NV>
constexpr int fold_left() { return (NV + 63) / 64; }

template <int NV>
__device__ __forceinline__ int fold_index(int lane, int slot) {
    constexpr int H1 = (NV + 1) / 2, H2 = (H1 + 1) / 2, H3 = (H2 + 1) / 2, H4 = (H3 + 1) / 2, H5 = (H4 + 1) / 2,
                  H6 = (H5 + 1) / 2;
    // from the last step to the first: the value among those the step began
    // with, NV where its second half had none left
    int i = slot;
    bool ok = true;
    const auto up = [&](int bit, int h, int cnt) {
        i += (lane & bit) ? h : 0;
        ok = ok && i < cnt;
    };
    up(1, H6, H5);
    up(2, H5, H4);
    up(4, H4, H3);
    up(8, H3, H2);
    up(16, H2, H1);
    up(32, H1, NV);
    return ok ? i : NV;
}

// One step on CNT values: slot i becomes the pair's sum of value i in the lower
// lanes and of value i + H in the upper (of nothing where there is none).
template <int CNT, typename F>
__device__ __forceinline__ void fold_step(float* v, F pair) {
    constexpr int H = (CNT + 1) / 2;
#pragma unroll
    for (int i = 0; i < H; ++i) v[i] = pair(v[i], i + H < CNT ? v[i + H] : 0.f);
}

template <int NV>
__device__ __forceinline__ void wave_fold(float (&v)[NV]) {
    constexpr int H1 = (NV + 1) / 2, H2 = (H1 + 1) / 2, H3 = (H2 + 1) / 2, H4 = (H3 + 1) / 2, H5 = (H4 + 1) / 2;
    const int lane = threadIdx.x & (kWave - 1);
    fold_step<NV>(v, [](float a, float b) {
        const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
        return __uint_as_float(p[0]) + __uint_as_float(p[1]);
    });
    fold_step<H1>(v, [](float a, float b) {
        const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
        return __uint_as_float(p[0]) + __uint_as_float(p[1]);
    });
    fold_step<H2>(v, [&](float a, float b) {
        return ((lane & 8) ? b : a) + dpp::mov<dpp::kRowRor8>((lane & 8) ? a : b);
    });
    fold_step<H3>(v, [&](float a, float b) {
        return ((lane & 4) ? b : a) + dpp::mov<dpp::kRowHalfMirror>((lane & 4) ? a : b);
    });
    fold_step<H4>(v, [&](float a, float b) {
        return ((lane & 2) ? b : a) + dpp::mov<dpp::kQuadXor2>((lane & 2) ? a : b);
    });
    fold_step<H5>(v, [&](float a, float b) {
        return ((lane & 1) ? b : a) + dpp::mov<dpp::kQuadXor1>((lane & 1) ? a : b);
    });
}

// dx of a mode: the storage type, or fp32 with MODE 2
template <typename TX, int MODE>
using BwdDx = std::conditional_t<MODE == 2, float, TX>;

// FOLD: the wave's row sums by wave_fold (in another order).
template <typename TX, int N, int VPT, int MODE, bool FOLD = false>
__device__ __forceinline__ void bwd_token(int64_t b, const float* __restrict__ coef, int64_t coef_stride,
                                          const float (&wv)[VPT][kLayerWC],
                                          const float (&xv)[N][VPT][kLayerWC],
                                          const float (&gv)[N][VPT][kLayerWC],
                                          float (&dwacc)[VPT][kLayerWC], float& sacc,
                                          BwdDx<TX, MODE>* __restrict__ dx, float* __restrict__ scal_out, int32_t* __restrict__ dx_scale, int C,
                                          float eps, float* red) {
    constexpr int WC = kLayerWC;
    constexpr int NC = coef_size<N>();
    constexpr int NS = N * N + 2 * N;
    constexpr int NR = 2 + N * N + 3 * N;  // ss, dot, dM, t_i, u_j, v_j
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = threadIdx.x / kWave;
    const int nwaves = blockDim.x / kWave;
    float* tot = red + 8 * NR;
    const float* cf = coef + b * coef_stride;
    float cfv[NC];
#pragma unroll
    for (int k = 0; k < NC; ++k) cfv[k] = cf[k];
    if constexpr (FOLD && N >= 5) {
        // in groups of at most 32: the sums are what the kernel keeps most of (n =
        // 6: 124 registers for 183 without the prefetch, three workgroups of 320
        // lanes a CU for one, 300 tokens x 1040 12.4 -> 9.3 us; n = 7, 8: no spills)
        float xa[VPT][WC], wgy[VPT][WC];
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
#pragma unroll
            for (int e = 0; e < WC; ++e) {
                float a = 0.f, gy = 0.f;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    a += cfv[i] * xv[i][k][e];
                    gy += cfv[N + i] * gv[i][k][e];
                }
                xa[k][e] = a;
                wgy[k][e] = wv[k][e] * gy;
            }
        }
        constexpr int NG = (NR + 31) / 32, PER = (NR + NG - 1) / NG;
        const auto group = [&](auto g_) {
            constexpr int F = decltype(g_)::value * PER, L = NR - F < PER ? NR - F : PER;
            float rv[L];
#pragma unroll
            for (int q = 0; q < L; ++q) {
                rv[q] = 0.f;
                const int id = F + q, m = id - 2 - N * N, i = m >= 0 ? m % N : (id >= 2 ? (id - 2) / N : 0),
                          j = id >= 2 && m < 0 ? (id - 2) % N : 0;
#pragma unroll
                for (int k = 0; k < VPT; ++k) {
#pragma unroll
                    for (int e = 0; e < WC; ++e) {
                        if (id == 0) rv[q] += xa[k][e] * xa[k][e];
                        else if (id == 1) rv[q] += wgy[k][e] * xa[k][e];
                        else if (m < 0) rv[q] += gv[i][k][e] * xv[j][k][e];
                        else if (m < N) rv[q] += gv[i][k][e] * (wv[k][e] * xa[k][e]);
                        else if (m < 2 * N) rv[q] += wgy[k][e] * xv[i][k][e];
                        else rv[q] += xa[k][e] * xv[i][k][e];
                    }
                }
            }
            wave_fold<L>(rv);
            static_assert(fold_left<L>() == 1, "a group is a wave's at most");
            const int i = fold_index<L>(lane, 0);
            if (i < L) red[wave * NR + F + i] = rv[0];
            __builtin_amdgcn_sched_barrier(0);
        };
        group(std::integral_constant<int, 0>{});
        if constexpr (NG > 1) group(std::integral_constant<int, 1>{});
        if constexpr (NG > 2) group(std::integral_constant<int, 2>{});
        static_assert(NG <= 3, "n up to 8");
    } else {
        float rv[NR];
#pragma unroll
        for (int k = 0; k < NR; ++k) rv[k] = 0.f;
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
#pragma unroll
            for (int e = 0; e < WC; ++e) {
                float xa = 0.f, gy = 0.f;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    xa += cfv[i] * xv[i][k][e];
                    gy += cfv[N + i] * gv[i][k][e];
                }
                const float wgy = wv[k][e] * gy;
                const float wxa = wv[k][e] * xa;
                rv[0] += xa * xa;
                rv[1] += wgy * xa;
#pragma unroll
                for (int i = 0; i < N; ++i) {
#pragma unroll
                    for (int j = 0; j < N; ++j) rv[2 + i * N + j] += gv[i][k][e] * xv[j][k][e];
                    rv[2 + N * N + i] += gv[i][k][e] * wxa;
                    rv[2 + N * N + N + i] += wgy * xv[i][k][e];
                    rv[2 + N * N + 2 * N + i] += xa * xv[i][k][e];
                }
            }
        }
        if constexpr (FOLD) {
            wave_fold<NR>(rv);
#pragma unroll
            for (int k = 0; k < fold_left<NR>(); ++k) {
                const int i = fold_index<NR>(lane, k);
                if (i < NR) red[wave * NR + i] = rv[k];
            }
        } else {
            wave_sum_last<NR>(rv);
            if (lane == kWave - 1) {
#pragma unroll
                for (int k = 0; k < NR; ++k) red[wave * NR + k] = rv[k];
            }
        }
    }
    __syncthreads();
    if (threadIdx.x < NR) {
        float s = 0.f;
        for (int q = 0; q < nwaves; ++q) s += red[q * NR + threadIdx.x];
        tot[threadIdx.x] = s;
    }
    __syncthreads();
    const float r = sqrtf(tot[0] / (float)C + eps);
    const float inv = 1.f / r;
    const float k2 = tot[1] * inv * inv * inv / (float)C;

    // Global stores of this routine go through resources with out-of-range
    // offsets for lanes that store nothing: no store sits behind a branch
    // (the caller's prefetch of the next token keeps exact wait counts).
    float v = 0.f;
    if (threadIdx.x < NS + 2) {
        const int t = threadIdx.x;
        if (t < N * N) {
            v = tot[2 + t];
        } else if (t < N * N + N) {
            v = tot[2 + t] * inv;  // dh_post_act = (sum G_i xa w) / r
        } else if (t < NS) {
            const int j = t - N * N - N;
            v = inv * tot[2 + N * N + N + j] - k2 * tot[2 + N * N + 2 * N + j];  // dh_pre_act
        } else {
            v = (t == NS) ? inv : k2;
        }
        if (MODE == 0) sacc += v;
    }
    if constexpr (MODE != 0) {
        const buf_rsrc_t srs = make_buf_rsrc(scal_out + b * (NS + 2), (uint32_t)((NS + 2) * 4));
        buf_st4(srs, threadIdx.x < NS + 2 ? (uint32_t)threadIdx.x * 4u : kBufOff, 0u, v);
    }

    if constexpr (MODE == 1 && sizeof(TX) == 2) {
        // The dynamic backward's stream part with bf16 x: the projection
        // kernel adds its terms and rounds the sum once, so this part travels
        // as fp16 against a power-of-two scale (part_pack4), one scale
        // exponent per half wave of this token: dx_scale[b][threadIdx.x / 32].
        float a[N][VPT][WC];
        float m = 0.f;  // largest |value|: fmaxf drops NaN, keeps +Inf
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
#pragma unroll
            for (int e = 0; e < WC; ++e) {
                float xa = 0.f, gy = 0.f;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    xa += cfv[i] * xv[i][k][e];
                    gy += cfv[N + i] * gv[i][k][e];
                }
                const float gxa = wv[k][e] * gy * inv - xa * k2;
                dwacc[k][e] += gy * xa * inv;
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    float s = kTermLast<N> ? 0.f : cfv[j] * gxa;
#pragma unroll
                    for (int i = 0; i < N; ++i) s += cfv[2 * N + i * N + j] * gv[i][k][e];
                    if (kTermLast<N>) s += cfv[j] * gxa;
                    a[j][k][e] = s;
                    m = fmaxf(m, fabsf(s));
                }
            }
        }
        m = half_wave_max_nonneg(m);
        if (__ballot(!(m < INFINITY))) {
            // an infinite value in this wave: the scale comes from the finite
            // values only (the whole wave takes this branch)
            m = 0.f;
#pragma unroll
            for (int k = 0; k < VPT; ++k)
#pragma unroll
                for (int e = 0; e < WC; ++e)
#pragma unroll
                    for (int j = 0; j < N; ++j) {
                        const float v = fabsf(a[j][k][e]);
                        m = v < INFINITY ? fmaxf(m, v) : m;
                    }
            m = half_wave_max_nonneg(m);
        }
        const int ks = part_scale_exp(m);
        const buf_rsrc_t drs = make_buf_rsrc(dx + b * (int64_t)N * C, (uint32_t)((int64_t)N * C * 2));
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            const int c0 = (k * blockDim.x + threadIdx.x) * WC;
            const uint32_t o0 = c0 < C ? (uint32_t)c0 * 2u : kBufOff;
#pragma unroll
            for (int j = 0; j < N; ++j) buf_st8<true>(drs, o0 + (uint32_t)(j * C * 2), 0u, part_pack4(a[j][k], ks));
        }
        const int ng = blockDim.x / 32;
        const buf_rsrc_t qrs = make_buf_rsrc(dx_scale + b * ng, (uint32_t)(ng * 4));
        buf_st4(qrs, (threadIdx.x & 31) == 0 ? (uint32_t)(threadIdx.x / 32) * 4u : kBufOff, 0u, __int_as_float(ks));
    } else {
        using TD = BwdDx<TX, MODE>;
        const buf_rsrc_t drs = make_buf_rsrc(dx + b * (int64_t)N * C, (uint32_t)((int64_t)N * C * (int64_t)sizeof(TD)));
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            const int c0 = (k * blockDim.x + threadIdx.x) * WC;
            float gxa[WC];
#pragma unroll
            for (int e = 0; e < WC; ++e) {
                float xa = 0.f, gy = 0.f;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    xa += cfv[i] * xv[i][k][e];
                    gy += cfv[N + i] * gv[i][k][e];
                }
                gxa[e] = wv[k][e] * gy * inv - xa * k2;
                dwacc[k][e] += gy * xa * inv;
            }
            const uint32_t o0 = c0 < C ? (uint32_t)c0 * (uint32_t)sizeof(TD) : kBufOff;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                float d[WC];
#pragma unroll
                for (int e = 0; e < WC; ++e) {
                    float s = kTermLast<N> ? 0.f : cfv[j] * gxa[e];
#pragma unroll
                    for (int i = 0; i < N; ++i) s += cfv[2 * N + i * N + j] * gv[i][k][e];
                    d[e] = kTermLast<N> ? s + cfv[j] * gxa[e] : s;
                }
                const uint32_t o = o0 + (uint32_t)(j * C * (int)sizeof(TD));
                static_assert(WC == 4, "4-channel chunks: one 16-byte (fp32) or 8-byte (bf16) store");
                if constexpr (sizeof(TD) == 4) {
                    buf_st16<true>(drs, o, 0u, make_uint4(__float_as_uint(d[0]), __float_as_uint(d[1]),
                                                          __float_as_uint(d[2]), __float_as_uint(d[3])));
                } else {
                    buf_st8<true>(drs, o, 0u, make_uint2(pack_bf16x2(d[0], d[1]), pack_bf16x2(d[2], d[3])));
                }
            }
        }
    }
}

}  // namespace mhc
