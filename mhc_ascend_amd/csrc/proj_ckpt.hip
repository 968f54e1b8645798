// Projection backward of the dynamic layer with the streams in an 8-bit
// checkpoint (mhc_ckpt.h), over the flattened rows x^[b][k], k = i C + c:
//   dx[b][k] = dx_in[b][k] + s[b] x^[b][k] + sum_o dP[b][o] Phi[o][k]
//   dPhi_part[tile][o][k] = sum_{b in tile} dP[b][o] x^[b][k]
// on the bf16 matrix cores: stages of 32 tokens as proj_bwd_mfma_kernel and
// proj_bwd_tiles_kernel (dynamic.hip), up to 96 output rows at once; more (n >
// 8) take a launch for each 96, the sum carried in fp32 and the s term on the
// first.
//
// x^ is exact in bf16, so dP alone is split: three bf16 planes for dPhi (to
// 2^-24 of a term; the kernels that read x use two, 2^-16).  For dx both dP and
// Phi are: three planes and the six products of 2^-16 and more for fp32 rows
// (2-4e-7 of dx in the 2-norm where all of it is dP Phi; two planes, 4.3e-6, and
// 4096 x 8 x 1280 in 104 us for 114, up to n = 6 1 us less), two planes and three
// products for bf16 rows, whose dx is rounded to 2^-9.  Bound by its bytes: 33/32 of a byte of x^, dx_in and dx a
// value (8192 x 4 x 4096 bf16: 674 MB in 131-148 us, 4.6-5.1 TB/s; the one that
// reads x, 806 MB, 143).
#include "mhc_ckpt.h"
#include "mhc_device.h"
#include "mhc_internal.h"
#include "mhc_mfma.h"

namespace mhc {

// v as the sum of PL bf16 planes, each the rest of the ones before it.
template <int PL>
__device__ __forceinline__ void split_planes8(const float (&v)[8], u32x4_t (&p)[PL]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float a = v[2 * e], b = v[2 * e + 1];
#pragma unroll
        for (int k = 0; k < PL; ++k) {
            const uint32_t h = pack_bf16(a, b);
            p[k][e] = h;
            a -= __uint_as_float(h << 16);
            b -= __uint_as_float(h & 0xffff0000u);
        }
    }
}

// Element (row, c) of a plane of dP in LDS: rows of 32 bf16 without padding (two
// workgroups of three tiles fit a CU), their 16-byte pieces turned by the row's
// bits 2 and 3, so that 16 rows' reads of one piece meet 64 banks.
__device__ __forceinline__ int dps_at(int row, int c) { return row * 32 + ((((c >> 3) ^ (row >> 2)) & 3) << 3) + (c & 7); }

// TD: dx's type.  PL: planes of dP and Phi for dx.  QIN: dx_in is the row pass's fp16 stream part against
// power-of-two scales (part_pack4) in dx itself; otherwise fp32 (dx itself for
// TD = float).  OT: tiles of 32 output rows.  NW waves of 32 columns each.
template <typename TD, int PL, bool QIN, int OT, int NW>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(QIN ? 4 : 2))) void proj_ckpt_bwd_kernel(
    int fmt, const uint8_t* __restrict__ q, const uint8_t* __restrict__ sc, const float* __restrict__ dP,
    int dp_stride, const float* __restrict__ s_tok, const float* __restrict__ phi_pre,
    const float* __restrict__ phi_post, const float* __restrict__ phi_res, int n, int o0, int np, const void* dx_in, TD* dx,
    const int32_t* __restrict__ dx_scale, int groups, int C, float* __restrict__ dphi_part, int64_t B, int64_t K,
    int64_t tile) {
    constexpr int NT = 64 * NW;
    constexpr int TB = 32;          // tokens per stage
    constexpr int CB = 32 * NW;     // columns per workgroup
    constexpr int VPR = CB / 8;     // pieces of 8 values per row
    constexpr int RPP = NT / VPR;   // rows per pass of pieces
    constexpr int PASSES = TB / RPP;
    constexpr int DW = QIN ? 2 : 4;              // bytes of dx_in
    constexpr int DVPR = CB * DW / 16;           // its 16-byte pieces per row
    constexpr int DRPP = NT / DVPR;
    constexpr int DPASSES = TB / DRPP;
    constexpr int XPITCH = CB * 2 + 8;
    constexpr int DPITCH = QIN ? CB * 2 + 8 : CB * 4 + 16;
    constexpr int NG = QIN ? CB / kPartGroup : 1;  // stream-part scale groups
    static_assert(PASSES * RPP == TB && DPASSES * DRPP == TB && NG * TB <= NT && NT >= 256, "stage shape");
    __shared__ __align__(16) char x_lds[TB * XPITCH];
    __shared__ __align__(16) char dx_lds[2][TB * DPITCH];
    // dP's planes by rows (tokens), PL of them, then by columns, three
    __shared__ __align__(16) bf16_t dps_lds[OT][PL + 3][32 * 32];
    __shared__ float s_lds[TB];
    __shared__ int q_lds[NG][TB];

    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = tid >> 6;
    const int lr = lane & 15;
    const int lg = lane >> 4;
    const int64_t kb0 = (int64_t)blockIdx.x * CB;
    const int wc0 = wave * 32;
    const bool wave_on = kb0 + wc0 < K;  // K % 32 == 0: whole waves are in or out
    const int lrow = tid / VPR, lvec = tid % VPR;
    const int64_t lcol = kb0 + (int64_t)lvec * 8;
    const int drow = tid / DVPR, dvec = tid % DVPR;
    const int64_t dcol = kb0 + (int64_t)dvec * (16 / DW);
    const bool dp_on = tid < 256;
    const int dtk = (tid & 255) >> 3;  // dP loaders: token (tid & 255) / 8,
    const int dpo = (tid & 7) * 4;     // outputs 32 ot + 4 (tid % 8) .. + 3

    // Phi^T: Phi[32 ot + 8 lg + e][column 16 ct + lr]
    u32x4_t ph[OT][2][PL];
#pragma unroll
    for (int ot = 0; ot < OT; ++ot) {
#pragma unroll
        for (int ct = 0; ct < 2; ++ct) {
            const int64_t k = kb0 + wc0 + 16 * ct + lr;
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int o = 32 * ot + 8 * lg + e;
                v[e] = (wave_on && o < np) ? phi_row(phi_pre, phi_post, phi_res, n, o0 + o, K)[k] : 0.f;
            }
            split_planes8<PL>(v, ph[ot][ct]);
        }
    }
    f32x4_t accP[2 * OT][2];
#pragma unroll
    for (int ot = 0; ot < 2 * OT; ++ot) {
#pragma unroll
        for (int ct = 0; ct < 2; ++ct) accP[ot][ct] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }

    const int64_t t_begin = (int64_t)blockIdx.y * tile;
    const int64_t t_end = (t_begin + tile < B) ? t_begin + tile : B;
    const int64_t nrows = t_end > t_begin ? t_end - t_begin : 0;
    const int64_t tb0 = nrows > 0 ? t_begin : 0;
    // (buffer resources as in proj_bwd_mfma_kernel: no access behind a branch)
    const int stride = (int)ck_stride(C), nb = (int)ck_blocks(C);
    const uint32_t qrow = (uint32_t)(n * stride), srow = (uint32_t)(n * nb);
    const uint32_t orow = (uint32_t)(K * (int64_t)sizeof(TD)), irow = (uint32_t)(K * DW);
    const buf_rsrc_t rs_x = make_buf_rsrc(q + tb0 * qrow, (uint32_t)nrows * qrow);
    const buf_rsrc_t rs_c = make_buf_rsrc(sc + tb0 * srow, (uint32_t)nrows * srow);
    const buf_rsrc_t rs_d = make_buf_rsrc(static_cast<const char*>(dx_in) + tb0 * (int64_t)irow, (uint32_t)nrows * irow);
    const buf_rsrc_t rs_o = make_buf_rsrc(dx + tb0 * K, (uint32_t)nrows * orow);
    const buf_rsrc_t rs_p = make_buf_rsrc(dP + tb0 * dp_stride, (uint32_t)(nrows * dp_stride * 4));
    const buf_rsrc_t rs_s = make_buf_rsrc(s_tok ? s_tok + tb0 : nullptr, s_tok ? (uint32_t)(nrows * 4) : 0u);
    const buf_rsrc_t rs_q = make_buf_rsrc(QIN ? dx_scale + tb0 * groups : nullptr, QIN ? (uint32_t)(nrows * groups * 4) : 0u);
    // a piece lies in one stream (C % 8 == 0): its place in the checkpoint's row
    const int64_t si = lcol < K ? lcol / C : 0;
    const int cc = (int)(lcol < K ? lcol - si * C : 0);
    const uint32_t xo = lcol < K ? (uint32_t)lrow * qrow + (uint32_t)(si * stride + cc) : kBufOff;
    const uint32_t co = lcol < K ? (uint32_t)lrow * srow + (uint32_t)(si * nb + (cc >> 5)) : kBufOff;
    const uint32_t dof = dcol < K ? (uint32_t)drow * irow + (uint32_t)(dcol * DW) : kBufOff;
    const uint32_t po = dp_on ? (uint32_t)(dtk * dp_stride + dpo) * 4u : kBufOff;
    const uint32_t so = tid < TB ? (uint32_t)tid * 4u : kBufOff;
    const int qg = tid / TB;
    const int grp = QIN ? (int)(((kb0 + (int64_t)qg * kPartGroup) % C) / kPartGroup) % groups : 0;
    const uint32_t qo = QIN && tid < NG * TB ? (uint32_t)((tid % TB) * groups + grp) * 4u : kBufOff;

    struct Fetched {
        uint2 x[PASSES];
        uint32_t c[PASSES];
        uint4 d[DPASSES];
    };
    struct Small {
        uint4 dp[OT];
        uint32_t s, q;
    };
    Fetched f0, f1;
    Small sm;
    auto fetch = [&](Fetched& f, uint32_t rel) __attribute__((always_inline)) {
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
            f.x[p] = buf_ld8<true>(rs_x, xo + (rel + p * RPP) * qrow, 0u);
            f.c[p] = (uint32_t)(uint8_t)__builtin_amdgcn_raw_buffer_load_b8(rs_c, (int)(co + (rel + p * RPP) * srow), 0, 0);
        }
#pragma unroll
        for (int p = 0; p < DPASSES; ++p) f.d[p] = buf_ld16<true>(rs_d, dof + (rel + p * DRPP) * irow, 0u);
    };
    auto fetch_small = [&](uint32_t rel) __attribute__((always_inline)) {
#pragma unroll
        for (int ot = 0; ot < OT; ++ot)
            sm.dp[ot] = buf_ld16<false>(rs_p, po + rel * (uint32_t)dp_stride * 4u + 128u * ot, 0u);
        sm.s = buf_ld4(rs_s, so + rel * 4u, 0u);
        sm.q = QIN ? buf_ld4(rs_q, qo + rel * (uint32_t)groups * 4u, 0u) : 0u;
    };
    auto commit = [&](const Fetched& f, int buf) __attribute__((always_inline)) {
        // an unconditional use of the small records (see proj_bwd_mfma_kernel)
        asm volatile("" ::"v"(sm.s), "v"(sm.q));
#pragma unroll
        for (int ot = 0; ot < OT; ++ot)
            asm volatile("" ::"v"(sm.dp[ot].x), "v"(sm.dp[ot].y), "v"(sm.dp[ot].z), "v"(sm.dp[ot].w));
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
            float v[8];
            if (fmt == kCkInt8) ck_unpack8<kCkInt8>(f.x[p], f.c[p], v);
            else ck_unpack8<kCkE4M3>(f.x[p], f.c[p], v);
            uint2* px = reinterpret_cast<uint2*>(&x_lds[(lrow + p * RPP) * XPITCH + lvec * 16]);
            px[0] = make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));  // exact
            px[1] = make_uint2(pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
        }
#pragma unroll
        for (int p = 0; p < DPASSES; ++p) {
            uint2* pd = reinterpret_cast<uint2*>(&dx_lds[buf][(drow + p * DRPP) * DPITCH + dvec * 16]);
            pd[0] = make_uint2(f.d[p].x, f.d[p].y);
            pd[1] = make_uint2(f.d[p].z, f.d[p].w);
        }
        if (dp_on) {
#pragma unroll
            for (int ot = 0; ot < OT; ++ot) {
                const uint32_t w4[4] = {sm.dp[ot].x, sm.dp[ot].y, sm.dp[ot].z, sm.dp[ot].w};
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = 32 * ot + dpo + e < np ? __uint_as_float(w4[e]) : 0.f;
#pragma unroll
                for (int k = 0; k < 3; ++k) {
                    const uint32_t p0 = pack_bf16(v[0], v[1]), p1 = pack_bf16(v[2], v[3]);
                    if (k < PL)
                        *reinterpret_cast<uint2*>(&dps_lds[ot][k][dps_at(dtk, dpo)]) = make_uint2(p0, p1);
                    bf16_t* col = dps_lds[ot][PL + k];
                    col[dps_at(dpo + 0, dtk)] = (bf16_t)(p0 & 0xffffu);
                    col[dps_at(dpo + 1, dtk)] = (bf16_t)(p0 >> 16);
                    col[dps_at(dpo + 2, dtk)] = (bf16_t)(p1 & 0xffffu);
                    col[dps_at(dpo + 3, dtk)] = (bf16_t)(p1 >> 16);
                    v[0] -= __uint_as_float(p0 << 16);
                    v[1] -= __uint_as_float(p0 & 0xffff0000u);
                    v[2] -= __uint_as_float(p1 << 16);
                    v[3] -= __uint_as_float(p1 & 0xffff0000u);
                }
            }
        }
        if (tid < TB) s_lds[tid] = __uint_as_float(sm.s);
        if constexpr (QIN) {
            if (tid < NG * TB) q_lds[qg][tid % TB] = (int)sm.q;
        }
    };
    auto read16 = [&](const bf16_t* p) __attribute__((always_inline)) -> u32x4_t {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        return u32x4_t{v.x, v.y, v.z, v.w};
    };
    auto compute = [&](int cur) __attribute__((always_inline)) {
        if (!wave_on) return;
        char* dt = dx_lds[cur];
        // dPhi: A = dP^T (row 16 ot + lr, tokens 8 lg .. + 7), B = x^ (same tokens, column 16 ct + lr)
        u32x4_t xh[2];
#pragma unroll
        for (int ct = 0; ct < 2; ++ct) {
            const int c = wc0 + 16 * ct + lr;
            const char* xp = x_lds + 8 * lg * XPITCH + c * 2;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t lo = *reinterpret_cast<const bf16_t*>(xp + 2 * e * XPITCH);
                const uint32_t hi = *reinterpret_cast<const bf16_t*>(xp + (2 * e + 1) * XPITCH);
                xh[ct][e] = lo | (hi << 16);
            }
        }
#pragma unroll
        for (int ot = 0; ot < 2 * OT; ++ot) {
#pragma unroll
            for (int k = 0; k < 3; ++k) {
                const u32x4_t a = read16(&dps_lds[ot / 2][PL + k][dps_at(16 * (ot & 1) + lr, 8 * lg)]);
#pragma unroll
                for (int ct = 0; ct < 2; ++ct) accP[ot][ct] = mfma16x16x32(a, xh[ct], accP[ot][ct]);
            }
        }
        // dx^T: D[column 16 ct + 4 lg + i][token 16 tt + lr]
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) {
            const int t = 16 * tt + lr;
            f32x4_t d[2] = {f32x4_t{0.f, 0.f, 0.f, 0.f}, f32x4_t{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
            for (int ot = 0; ot < OT; ++ot) {
                u32x4_t b[PL];
#pragma unroll
                for (int k = 0; k < PL; ++k) b[k] = read16(&dps_lds[ot][k][dps_at(t, 8 * lg)]);
#pragma unroll
                for (int ct = 0; ct < 2; ++ct) {
#pragma unroll
                    for (int o = 0; o < PL; ++o) {  // products of 2^(-8 o)
#pragma unroll
                        for (int i = o; i >= 0; --i) d[ct] = mfma16x16x32(ph[ot][ct][i], b[o - i], d[ct]);
                    }
                }
            }
            const float st = s_lds[t];
#pragma unroll
            for (int ct = 0; ct < 2; ++ct) {
                const int c0 = wc0 + 16 * ct + 4 * lg;
                const uint2 xw = *reinterpret_cast<const uint2*>(x_lds + t * XPITCH + c0 * 2);
                const float xv[4] = {__uint_as_float(xw.x << 16), __uint_as_float(xw.x & 0xffff0000u),
                                     __uint_as_float(xw.y << 16), __uint_as_float(xw.y & 0xffff0000u)};
                if constexpr (QIN) {
                    uint2* p = reinterpret_cast<uint2*>(dt + t * DPITCH + c0 * 2);
                    float dv[4];
                    part_unpack4(*p, q_lds[c0 / kPartGroup][t], dv);
#pragma unroll
                    for (int i = 0; i < 4; ++i) dv[i] = d[ct][i] + dv[i] + st * xv[i];
                    *p = make_uint2(pack_bf16(dv[0], dv[1]), pack_bf16(dv[2], dv[3]));
                } else {
                    float4* p = reinterpret_cast<float4*>(dt + t * DPITCH + c0 * 4);
                    const float4 a = *p;
                    *p = make_float4(fmaf(st, xv[0], d[ct][0] + a.x), fmaf(st, xv[1], d[ct][1] + a.y),
                                     fmaf(st, xv[2], d[ct][2] + a.z), fmaf(st, xv[3], d[ct][3] + a.w));
                }
            }
        }
    };
    // dx tile -> memory: pieces of 8 bf16 or 4 fp32
    const uint32_t oof = sizeof(TD) == 2 ? (lcol < K ? (uint32_t)lrow * orow + (uint32_t)(lcol * 2) : kBufOff) : dof;
    auto store = [&](uint32_t rel, int cur) __attribute__((always_inline)) {
        if constexpr (sizeof(TD) == 2) {
#pragma unroll
            for (int p = 0; p < PASSES; ++p) {
                const char* t = &dx_lds[cur][(lrow + p * RPP) * DPITCH];
                uint4 o;
                if constexpr (QIN) {
                    const uint2* u = reinterpret_cast<const uint2*>(t + lvec * 16);
                    o = make_uint4(u[0].x, u[0].y, u[1].x, u[1].y);
                } else {
                    const float4 a = *reinterpret_cast<const float4*>(t + lvec * 32);
                    const float4 b = *reinterpret_cast<const float4*>(t + lvec * 32 + 16);
                    o = make_uint4(pack_bf16(a.x, a.y), pack_bf16(a.z, a.w), pack_bf16(b.x, b.y), pack_bf16(b.z, b.w));
                }
                buf_st16<true>(rs_o, oof + (rel + p * RPP) * orow, 0u, o);
            }
        } else {
#pragma unroll
            for (int p = 0; p < DPASSES; ++p)
                buf_st16<true>(rs_o, oof + (rel + p * DRPP) * orow, 0u,
                               *reinterpret_cast<const uint4*>(&dx_lds[cur][(drow + p * DRPP) * DPITCH + dvec * 16]));
        }
    };
    // whole pairs of stages, as proj_bwd_mfma_kernel
    const uint32_t nr = (uint32_t)nrows;
    fetch_small(0u);
    fetch(f0, 0u);
    commit(f0, 0);
    fetch(f1, TB);
    __syncthreads();
    for (uint32_t r0 = 0; r0 < nr; r0 += 2 * TB) {
        fetch_small(r0 + TB);
        fetch(f0, r0 + 2 * TB);
        compute(0);
        __syncthreads();
        store(r0, 0);
        commit(f1, 1);
        __syncthreads();
        fetch_small(r0 + 2 * TB);
        fetch(f1, r0 + 3 * TB);
        compute(1);
        __syncthreads();
        store(r0 + TB, 1);
        commit(f0, 0);
        __syncthreads();
    }
    if (!wave_on) return;
    float* out = dphi_part + (int64_t)blockIdx.y * np * K;
#pragma unroll
    for (int ot = 0; ot < 2 * OT; ++ot) {
#pragma unroll
        for (int ct = 0; ct < 2; ++ct) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int o = 16 * ot + 4 * lg + i;
                if (o < np) out[(int64_t)o * K + kb0 + wc0 + 16 * ct + lr] = accP[ot][ct][i];
            }
        }
    }
}

// ---------------------------------------------------------------------------
// Host launchers
// ---------------------------------------------------------------------------
// x_dtype: the rows'.  Of several launches all but the last leave dx in fp32.
static const void* pick_proj_ckpt(int dx_dtype, int x_dtype, bool qin, int np) {
    if (qin) return reinterpret_cast<const void*>(&proj_ckpt_bwd_kernel<bf16_t, 2, true, 1, 8>);
    const int ot = proj_tiles(np);
#define MHC_PC(OT_)                                                                                       \
    (dx_dtype == kBF16  ? reinterpret_cast<const void*>(&proj_ckpt_bwd_kernel<bf16_t, 2, false, OT_, 4>)  \
     : x_dtype == kBF16 ? reinterpret_cast<const void*>(&proj_ckpt_bwd_kernel<float, 2, false, OT_, 4>)   \
                        : reinterpret_cast<const void*>(&proj_ckpt_bwd_kernel<float, 3, false, OT_, 4>))
    return ot == 1 ? MHC_PC(1) : (ot == 2 ? MHC_PC(2) : MHC_PC(3));
#undef MHC_PC
}

static int proj_ckpt_waves(bool qin) { return qin ? 8 : 4; }

// A token tile's rows in fp32, plus the stages the pipeline reads past its
// end, under 2 GiB (buffer resources and offsets).
static int64_t proj_ckpt_max_tile(int64_t K) { return ((int64_t(1) << 31) - 1) / (K * 4) - 4 * 32; }

bool proj_ckpt_supported(int np, int64_t K, int64_t C) {
    return np >= 1 && np <= kProjCkptMaxRows && K % 32 == 0 && C % 8 == 0 && proj_ckpt_max_tile(K) >= 64;
}

// Column blocks x token tiles fill one round of resident workgroups: the
// partials of dPhi are half of two rounds' (n = 6, 2047 x 1040 bf16: 34.6 us and
// 9.5 for their sums, against 40.7 and 12).
int proj_ckpt_bwd_tiles(int x_dtype, bool qin, int np, int64_t B, int64_t K) {
    const int nw = proj_ckpt_waves(qin);
    const int64_t gx = (K + 32 * nw - 1) / (32 * nw);
    const int per_cu = occupancy_per_cu(pick_proj_ckpt(x_dtype, x_dtype, qin, np), 64 * nw, 0);
    int64_t tiles = (int64_t)device_cu_count() * per_cu / gx;
    const int64_t blocks = (B + 63) / 64;
    if (tiles > blocks) tiles = blocks;
    if (tiles < 1) tiles = 1;
    const int64_t mt = proj_ckpt_max_tile(K) / 64 * 64;
    if ((B + tiles - 1) / tiles > mt) tiles = (B + mt - 1) / mt;
    return (int)tiles;
}

hipError_t launch_proj_ckpt_bwd(int dx_dtype, int x_dtype, bool qin, int fmt, const void* values, const void* scales,
                                const float* dP, int dp_stride, const float* s_tok, const float* phi_pre,
                                const float* phi_post, const float* phi_res, int n, int o0, int np,
                                const void* dx_in, void* dx, const int32_t* dx_scale, int groups, float* dphi_part, int tiles, int64_t B,
                                int64_t K, hipStream_t s) {
    int C = (int)(K / n);
    if (B == 0) return hipSuccess;
    if (!proj_ckpt_supported(np, K, C) || np > kProjCkptRows || tiles < 1) return hipErrorInvalidValue;
    dP += o0;
    if (qin && (dx_dtype != kBF16 || !dx_scale || groups < 1 || C % kPartGroup != 0 || np > kProjTile || dx_in != dx))
        return hipErrorInvalidValue;
    int64_t tile = (B + tiles - 1) / tiles;
    tile = ((tile + 63) / 64) * 64;
    if (tile > proj_ckpt_max_tile(K)) return hipErrorInvalidValue;
    const int nw = proj_ckpt_waves(qin);
    const dim3 grid((unsigned)((K + 32 * nw - 1) / (32 * nw)), (unsigned)tiles);
    void* args[] = {(void*)&fmt,      (void*)&values,  (void*)&scales, (void*)&dP,     (void*)&dp_stride, (void*)&s_tok,
                    (void*)&phi_pre,  (void*)&phi_post, (void*)&phi_res, (void*)&n,    (void*)&o0, (void*)&np,        (void*)&dx_in,
                    (void*)&dx,       (void*)&dx_scale, (void*)&groups, (void*)&C,     (void*)&dphi_part, (void*)&B,
                    (void*)&K,        (void*)&tile};
    const int tok = timing_begin("proj_ckpt_bwd", s);
    hipError_t e = mhc_launch_kernel(pick_proj_ckpt(dx_dtype, x_dtype, qin, np), grid, dim3(64 * nw), args, 0, s);
    timing_end(tok, s);
    return e != hipSuccess ? e : hipGetLastError();
}

}  // namespace mhc
