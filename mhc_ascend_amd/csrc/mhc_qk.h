// Kernels of the RMSNorm of every head of queries and keys and the rotation of
// their positions, one pass each way.  For one head row x of D channels, weight w:
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
//
// AX: a token has positions on 2 to 4 axes, and every pair turns by its own
// axis's, table entry (position on the axis, column p): sections of consecutive
// pairs, or pairs dealt to the axes in turn.  The kernels are instantiated
// without in qk_norm_rope.hip and with in qk_axes.hip.
#pragma once

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

// The axis of a pair; the sizes in one word and the division by a product keep
// the argument's memory and a long division out of the kernels' first loads.
__device__ __forceinline__ int qk_axis(const QkArgs& a, int col) {
    if (a.dealt) {
        const uint32_t turn = ((uint32_t)col * a.deal_mul) >> 16, axis = (uint32_t)col - turn * (uint32_t)a.axes;
        // what is not dealt belongs to axis 0
        return turn < ((uint32_t)(a.deal_sizes >> (16 * axis)) & 0xffffu) ? (int)axis : 0;
    }
    return (col >= a.part[0] ? 1 : 0) + (col >= a.part[1] ? 1 : 0) + (col >= a.part[2] ? 1 : 0);
}

// The axes of N consecutive pairs from `col` on (pairs past the last: any), two
// bits each.  The loop stands twice so that `dealt` is looked at once and not pair
// by pair (2% of the kernels' instructions).
template <int N>
__device__ __forceinline__ uint32_t qk_axes_of(const QkArgs& a, int col) {
    uint32_t m = 0;
    if (a.dealt) {
#pragma unroll
        for (int e = 0; e < N; ++e) m |= (uint32_t)qk_axis(a, col + e) << (2 * e);
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) m |= (uint32_t)qk_axis(a, col + e) << (2 * e);
    }
    return m;
}
// Opaque to the compiler, which otherwise works out selects ahead of the loop over
// tokens (qk_bwd_kernel of fp32: 3% more instructions, the registers the same to 4).
__device__ __forceinline__ uint32_t qk_opaque(uint32_t m) {
    asm volatile("" : "+v"(m));
    return m;
}

// A token's positions on its way from memory: loaded (before the rows, which the
// table's loads would wait for otherwise), then checked.  Two words each, without
// a branch on the element size.
template <bool AX> struct QkRaw {
    __device__ __forceinline__ QkRaw(const QkArgs&, int64_t) {}
};
template <> struct QkRaw<true> {
    uint32_t lo[4], hi[4];
    __device__ __forceinline__ QkRaw(const QkArgs& a, int64_t t) {
        const uint32_t i = (uint32_t)t % (uint32_t)a.period;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const char* p = static_cast<const char*>(a.pos) + ((s < a.axes ? s : 0) * a.period + i) * a.pos_bytes;
            lo[s] = *reinterpret_cast<const uint32_t*>(p);
            hi[s] = *reinterpret_cast<const uint32_t*>(p + a.pos_bytes - 4);
        }
    }
};

// Where a token's table rows begin: one, or one an axis.
template <bool AX> struct QkAt;
template <> struct QkAt<false> {
    int64_t pos, at;
    __device__ __forceinline__ QkAt(const QkArgs& a, int64_t t, const QkRaw<false>&) {
        pos = qk_position(a, t);
        at = (pos < 0 ? 0 : pos) * (int64_t)(a.R >> 1);
    }
    __device__ __forceinline__ bool ok() const { return pos >= 0; }
    __device__ __forceinline__ int64_t on(uint32_t) const { return at; }
    __device__ __forceinline__ int64_t of(const QkArgs&, int) const { return at; }
};
template <> struct QkAt<true> {
    int64_t at[4];
    bool good;
    __device__ __forceinline__ QkAt(const QkArgs& a, int64_t, const QkRaw<true>& raw) {
        good = true;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const uint32_t hi = a.pos_bytes == 8 ? raw.hi[s] : (uint32_t)((int32_t)raw.lo[s] >> 31);
            const int64_t p = (int64_t)((uint64_t)hi << 32 | raw.lo[s]);
            const bool in = p >= 0 && p < a.table_rows;
            good = good && in;
            at[s] = (in ? p : 0) * (int64_t)(a.R >> 1);
        }
    }
    __device__ __forceinline__ bool ok() const { return good; }
    // the low two bits of `axis`
    __device__ __forceinline__ int64_t on(uint32_t axis) const {
        const int64_t lo = axis & 1 ? at[1] : at[0], hi = axis & 1 ? at[3] : at[2];
        return axis & 2 ? hi : lo;
    }
    __device__ __forceinline__ int64_t of(const QkArgs& a, int col) const { return on(qk_axis(a, col)); }
};

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
// lane at a time.  A block of 32 channels is half a wave.  Bound by its
// instructions (8192 tokens x 40 heads of 128 bf16, forward and backward: 996 us,
// the kernels below 84), so for what qk_tiling finds no pieces for: heads that are
// no multiple of 4 or too wide, and halves of a rotated width that is no multiple
// of 8, whose pairs no piece of 4 meets whole (9147 x 40 heads of 72 bf16: 635 us
// with R = 36, 119 with R = 72; on three axes 688 and 121).
// ---------------------------------------------------------------------------
template <typename T, int FMT, bool AX>
__global__ __launch_bounds__(256) void qk_fwd_any_kernel(QkArgs a) {
    const int lane = threadIdx.x & 63;
    const int hh = blockIdx.y * 4 + (threadIdx.x >> 6);
    if (hh >= a.heads[0] + a.heads[1]) return;  // whole waves, no barrier below
    const int64_t t = a.t0 + blockIdx.x;
    const int s = hh < a.heads[0] ? 0 : 1;
    const int h = s ? hh - a.heads[0] : hh;
    const T* x = static_cast<const T*>(a.x[s]) + t * a.x_token[s] + h * a.x_head[s];
    const int64_t row = t * a.heads[s] + h;
    T* y = static_cast<T*>(a.y[s]) + row * a.D;
    const QkAt<AX> at(a, t, QkRaw<AX>(a, t));
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
    const float inv = !at.ok() ? __uint_as_float(0x7fc00000u) : 1.f / sqrtf(ss / (float)a.D + a.eps);
    for (int d = lane; d < a.D; d += 64) {
        float o = VecIO<T>::scalar(x + d) * inv * qk_weight(a, s, d);
        int col, other;
        float sign;
        if (qk_pair(a, d, col, other, sign)) {
            const float v = VecIO<T>::scalar(x + other) * inv * qk_weight(a, s, other);
            const int64_t tab = at.of(a, col);
            o = o * a.cos[tab + col] + sign * v * a.sin[tab + col];
        }
        VecIO<T>::put(y + d, o);
    }
}

// x[] is the row itself (FMT < 0) or its checkpoint in q / sc; y[] the
// gradient rows; g the cotangents.  Persistent workgroups over tokens, dw in
// LDS (every channel belongs to one lane of a wave), one partial row a
// workgroup: dw_part[grid][2 D], queries then keys.
template <typename T, int FMT, bool AX>
__global__ __launch_bounds__(256) void qk_bwd_any_kernel(QkArgs a, float* __restrict__ dw_part) {
    extern __shared__ float dw[];  // [4 waves][2][D]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int i = threadIdx.x; i < 8 * a.D; i += 256) dw[i] = 0.f;
    __syncthreads();
    for (int64_t t = blockIdx.x; t < a.T; t += gridDim.x) {
        const QkAt<AX> at(a, t, QkRaw<AX>(a, t));
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
                const int64_t tab = at.of(a, col);
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
            const float inv = !at.ok() ? __uint_as_float(0x7fc00000u) : 1.f / sqrtf(ss / (float)a.D + a.eps);
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
// Heads of whole pieces: V channels a lane, a group of G lanes (a power of
// two, D / V or the next) a head row, so a wave takes 64 / G heads of one token
// at a time and keeps the token's table row in registers for all of them.  A
// lane of the rotated halves reads its partner's piece itself: the bytes are
// in the cache line of another lane's load, and no exchange between lanes
// waits on the sums.  Tasks of U such steps have all their loads in flight.
// Few tokens: their tasks are spread over Y workgroups each.  Few heads and many
// tokens (MT): the groups of a wave share 2^tw tokens, each with its own table
// row, so that a step's groups all have a head (forward and backward, against one
// token a wave: 16384 x 1 + 1 heads of 64 fp32 30 us for 67, 16384 x 4 + 4 of 64
// bf16 int8 36 for 72, 16384 x 8 + 1 of 128 bf16 55 for 73).  Bound by bytes:
// 8192 tokens x 40 heads of 128 bf16, forward 32 us (5.2 TB/s), backward 52 (4.8);
// 16384 x 64 heads with an int8 checkpoint, 135-143 (4.7-5.0) and 164-184
// (3.7-4.1).  16 tokens x 40 heads: 4.7 us, the latency of its loads.
// ---------------------------------------------------------------------------
typedef uint32_t qk_u2_t __attribute__((ext_vector_type(2)));
typedef qk_u2_t qk_u2_a2_t __attribute__((aligned(2)));
typedef qk_u2_t qk_u2_a4_t __attribute__((aligned(4)));

template <typename T, int V> struct QkPiece;  // V elements as raw words
template <> struct QkPiece<float, 8> {
    ck_u4_t w[2];
    __device__ __forceinline__ void load(const float* p) {
        w[0] = *reinterpret_cast<const ck_u4_a4_t*>(p);
        w[1] = *reinterpret_cast<const ck_u4_a4_t*>(p + 4);
    }
    __device__ __forceinline__ float get(int e) const { return __uint_as_float(w[e / 4][e % 4]); }
};
template <> struct QkPiece<float, 4> {
    ck_u4_t w;
    __device__ __forceinline__ void load(const float* p) { w = *reinterpret_cast<const ck_u4_a4_t*>(p); }
    __device__ __forceinline__ float get(int e) const { return __uint_as_float(w[e]); }
};
template <> struct QkPiece<float, 2> {
    qk_u2_t w;
    __device__ __forceinline__ void load(const float* p) { w = *reinterpret_cast<const qk_u2_a4_t*>(p); }
    __device__ __forceinline__ float get(int e) const { return __uint_as_float(w[e]); }
};
template <> struct QkPiece<bf16_t, 8> {
    ck_u4_t w;
    __device__ __forceinline__ void load(const bf16_t* p) { w = *reinterpret_cast<const ck_u4_a2_t*>(p); }
    __device__ __forceinline__ float get(int e) const {
        return __uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
    }
};
template <> struct QkPiece<bf16_t, 4> {
    qk_u2_t w;
    __device__ __forceinline__ void load(const bf16_t* p) { w = *reinterpret_cast<const qk_u2_a2_t*>(p); }
    __device__ __forceinline__ float get(int e) const {
        return __uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
    }
};

template <typename T, int V>
__device__ __forceinline__ void qk_store(T* p, const float (&v)[V]) {
    if constexpr (V == 8) {
        ck_store8(p, v);
    } else if constexpr (sizeof(T) == 4) {
        const ck_u4_t a = {__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
        __builtin_nontemporal_store(a, reinterpret_cast<ck_u4_a4_t*>(p));
    } else {
        const qk_u2_t a = {pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
        __builtin_nontemporal_store(a, reinterpret_cast<qk_u2_a2_t*>(p));
    }
}

// One lane's place in its head row.
template <int V, bool IL>
struct QkLane {
    static constexpr int kTab = IL ? V / 2 : V;
    int c0;       // its first channel
    bool in;      // within the head
    bool turned;  // some channel of the piece rotates
    int other;    // first channel of its partners' piece (its own where it has none)
    float sign;   // of the partner's sine product
    uint32_t ax;  // the axes of its table entries (with AX)

    template <bool AX>
    __device__ __forceinline__ QkLane(const QkArgs& a, int lane, int lg, std::bool_constant<AX>) {
        c0 = (lane & ((1 << lg) - 1)) * V;
        in = c0 < a.D;
        turned = c0 < a.R;
        other = c0;
        sign = 1.f;
        if (!IL && turned) {
            const int half = a.R >> 1;
            other = c0 < half ? c0 + half : c0 - half;
            sign = c0 < half ? -1.f : 1.f;
        }
        ax = AX ? qk_axes_of<kTab>(a, first_pair(a)) : 0u;
    }
    // The pair of its first table entry.
    __device__ __forceinline__ int first_pair(const QkArgs& a) const {
        if (IL) return c0 >> 1;
        const int half = a.R >> 1;
        return turned ? (c0 < half ? c0 : c0 - half) : 0;
    }

    // The lane's table entries of a token: per channel with halves (the sine
    // with its sign), per pair interleaved.  1 and 0 elsewhere.  With axes, a
    // piece whose pairs are of one axis (a.whole) is read whole, others pair by
    // pair: their loads are in flight together, and hit the caches.
    template <bool AX>
    __device__ __forceinline__ void table(const QkArgs& a, const QkAt<AX>& row, float (&c)[kTab],
                                          float (&s)[kTab]) const {
        const int half = a.R >> 1;
        const uint32_t m = AX ? qk_opaque(ax) : 0u;
        if constexpr (IL) {
#pragma unroll
            for (int p = 0; p < kTab; ++p) {
                const int col = (c0 >> 1) + p;
                const bool on = col < half;
                const int64_t at = row.on(m >> (2 * p));
                c[p] = on ? a.cos[at + col] : 1.f;
                s[p] = on ? a.sin[at + col] : 0.f;
            }
        } else {
            const int col = first_pair(a);
            float pc[V], ps[V];
            if (!AX || a.whole) {
                const int64_t at = row.on(m) + col;
                QkPiece<float, V> qc, qs;
                qc.load(a.cos + at);
                qs.load(a.sin + at);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    pc[e] = qc.get(e);
                    ps[e] = qs.get(e);
                }
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const int64_t at = row.on(m >> (2 * e)) + col + e;
                    pc[e] = a.cos[at];
                    ps[e] = a.sin[at];
                }
                __builtin_amdgcn_sched_barrier(0);  // all loads, then their uses
            }
#pragma unroll
            for (int e = 0; e < V; ++e) {
                c[e] = turned ? pc[e] : 1.f;
                s[e] = turned ? sign * ps[e] : 0.f;
            }
        }
    }

    // Channel e's rotation of v (this piece) and o (the partners' piece) by
    // `way` = 1 or -1 times the angle.
    __device__ __forceinline__ float turn(const float (&v)[V], const float (&o)[V], const float (&c)[kTab],
                                          const float (&s)[kTab], int e, float way, int R) const {
        if constexpr (IL) {
            const float x = (e & 1) ? v[e - 1] : -v[e + 1];
            return c0 + e < R ? v[e] * c[e / 2] + way * x * s[e / 2] : v[e];
        } else {
            return turned ? v[e] * c[e] + way * o[e] * s[e] : v[e];
        }
    }

    __device__ __forceinline__ void weights(const QkArgs& a, int s, int at, float (&w)[V]) const {
        if (a.w_dtype == kBF16) {
            QkPiece<bf16_t, V> p;
            p.load(static_cast<const bf16_t*>(a.w[s]) + (in ? at : 0));
#pragma unroll
            for (int e = 0; e < V; ++e) w[e] = in ? p.get(e) : 0.f;
        } else {
            QkPiece<float, V> p;
            p.load(static_cast<const float*>(a.w[s]) + (in ? at : 0));
#pragma unroll
            for (int e = 0; e < V; ++e) w[e] = in ? p.get(e) : 0.f;
        }
    }
};

constexpr int kQkU = 2;
// Tasks of a token: its queries' steps, then its keys', U at a time.  lt: log2
// of the lanes a head times the tokens of a wave.
struct QkTasks {
    int per;    // heads of a task
    int nq, n;  // tasks of the queries, of both
    __host__ __device__ QkTasks(int H, int K, int lt) : per(kQkU * (64 >> lt)) {
        nq = (H + per - 1) / per;
        n = nq + (K + per - 1) / per;
    }
};

// A task's loads.
template <typename T, int V, bool IL>
struct QkRows {
    QkPiece<T, V> own[kQkU], far[IL ? 1 : kQkU];
    __device__ __forceinline__ void load(const QkLane<V, IL>& ln, const T* base, int64_t head_stride, int h0, int step,
                                         int heads) {
#pragma unroll
        for (int u = 0; u < kQkU; ++u) {
            const int h = h0 + u * step;
            const T* row = base + (h < heads ? h : 0) * head_stride;
            own[u].load(row + (ln.in ? ln.c0 : 0));
            if constexpr (!IL) far[u].load(row + (ln.in ? ln.other : 0));
        }
    }
};

template <typename T, int FMT, int V, bool IL, bool MT, bool AX>
__global__ __launch_bounds__(256) void qk_fwd_kernel(QkArgs a, int lg, int tw) {
    const int lane = threadIdx.x & 63;
    if (!MT) tw = 0;
    int64_t t = a.t0 + (((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) << tw);
    if (t >= a.T) return;
    const QkLane<V, IL> ln(a, lane, lg, std::bool_constant<AX>{});
    const QkTasks tasks(a.heads[0], a.heads[1], lg + tw);
    const int step = 64 >> (lg + tw), sub = (lane >> lg) & (step - 1);
    bool here = true;
    if (MT) {
        t += lane >> (6 - tw);
        here = t < a.T;
        t = here ? t : a.T - 1;
    }
    const int stride = (int)ck_stride(a.D), nb = (int)ck_blocks(a.D);
    const auto side = [&](int j) { return j < tasks.nq ? 0 : 1; };
    const auto first = [&](int j, int s) { return (s ? j - tasks.nq : j) * tasks.per + sub; };
    const auto fetch = [&](int j, QkRows<T, V, IL>& r) {
        const int s = side(j);
        r.load(ln, static_cast<const T*>(a.x[s]) + t * a.x_token[s], a.x_head[s], first(j, s), step, a.heads[s]);
    };
    int j = blockIdx.y;
    const QkRaw<AX> raw(a, t);
    QkRows<T, V, IL> next;
    fetch(j, next);  // the grid's y is at most the number of tasks
    const QkAt<AX> at(a, t, raw);
    float c[QkLane<V, IL>::kTab], sn[QkLane<V, IL>::kTab];
    ln.table(a, at, c, sn);
    float w[V], wo[V];
    int whose = -1;  // weights w and wo are
    for (; j < tasks.n; j += gridDim.y) {
        const int s = side(j), h0 = first(j, s);
        const QkRows<T, V, IL> rows = next;
        if (j + (int)gridDim.y < tasks.n) fetch(j + gridDim.y, next);
        if (s != whose) {
            whose = s;
            ln.weights(a, s, ln.c0, w);
            if constexpr (!IL) ln.weights(a, s, ln.other, wo);
        }
#pragma unroll
        for (int u = 0; u < kQkU; ++u) {
            const int h = h0 + u * step;
            const bool on = here && h < a.heads[s];
            const int64_t row = t * a.heads[s] + h;
            float v[V], o[V], y[V];
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                v[e] = ln.in ? rows.own[u].get(e) : 0.f;
                ss += v[e] * v[e];
            }
            if constexpr (FMT >= 0) {
                uint32_t m = 0;
#pragma unroll
                for (int e = 0; e < V; ++e) m = m > ck_abs_bits(v[e]) ? m : ck_abs_bits(v[e]);
                const uint32_t sc = Ck<FMT>::scale(ck_group_max<32 / V>(m));
                const float up = Ck<FMT>::up(sc);
                const uint32_t keep = sc == 255u ? 0u : ~0u;
                uint32_t q[V / 4];
#pragma unroll
                for (int e = 0; e < V; e += 4)
                    q[e / 4] = Ck<FMT>::pack4(v[e], v[e + 1], v[e + 2], v[e + 3], up, keep);
                if (on && ln.c0 < stride) {
                    uint8_t* qp = a.q[s] + row * stride + ln.c0;
                    if constexpr (V == 8) st8_nt(qp, make_uint2(q[0], q[1]));
                    else __builtin_nontemporal_store(q[0], reinterpret_cast<uint32_t*>(qp));
                }
                if (on && ln.in && (ln.c0 & 31) == 0) a.sc[s][row * nb + (ln.c0 >> 5)] = (uint8_t)sc;
            }
            ss = lane_group_sum(ss, lg);
            const float inv = !at.ok() ? __uint_as_float(0x7fc00000u) : 1.f / sqrtf(ss / (float)a.D + a.eps);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                v[e] = v[e] * inv * w[e];
                o[e] = 0.f;
                if constexpr (!IL) o[e] = rows.far[u].get(e) * inv * wo[e];
            }
#pragma unroll
            for (int e = 0; e < V; ++e) y[e] = ln.turn(v, o, c, sn, e, 1.f, a.R);
            if (on && ln.in) qk_store<T, V>(static_cast<T*>(a.y[s]) + row * a.D + ln.c0, y);
        }
    }
}

// Persistent waves over tokens; both weights' gradients in registers, added
// over the wave's groups and the workgroup's waves at the end, in a fixed
// order: dw_part[workgroup][2 D].
template <typename T, int FMT, int V, bool IL, bool MT, bool AX>
__global__ __launch_bounds__(512) void qk_bwd_kernel(QkArgs a, int lg, int tw, float* __restrict__ dw_part) {
    extern __shared__ float red[];  // [8 waves][2][D]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (!MT) tw = 0;
    const QkLane<V, IL> ln(a, lane, lg, std::bool_constant<AX>{});
    const QkTasks tasks(a.heads[0], a.heads[1], lg + tw);
    const int step = 64 >> (lg + tw), sub = (lane >> lg) & (step - 1);
    const int stride = (int)ck_stride(a.D), nb = (int)ck_blocks(a.D);
    const bool ragged = a.D != V << lg;
    float dw[2][V];
#pragma unroll
    for (int e = 0; e < V; ++e) dw[0][e] = dw[1][e] = 0.f;
    for (int64_t tb = ((int64_t)blockIdx.x * 8 + wave) << tw; tb < a.T; tb += ((int64_t)gridDim.x * 8) << tw) {
        int64_t t = tb;
        bool here = true;
        if (MT) {
            t += lane >> (6 - tw);
            here = t < a.T;
            t = here ? t : a.T - 1;
        }
        const QkAt<AX> at(a, t, QkRaw<AX>(a, t));
        float c[QkLane<V, IL>::kTab], sn[QkLane<V, IL>::kTab];
        ln.table(a, at, c, sn);
        for (int j = blockIdx.y; j < tasks.n; j += gridDim.y) {
            const int s = j < tasks.nq ? 0 : 1;
            const int h0 = (s ? j - tasks.nq : j) * tasks.per + sub;
            const T* g = static_cast<const T*>(a.g[s]) + t * a.g_token[s];
            QkPiece<T, V> gown[kQkU], gfar[kQkU], xr[kQkU];
            uint32_t q[kQkU][V / 4], sc[kQkU];
#pragma unroll
            for (int u = 0; u < kQkU; ++u) {
                const int h = h0 + u * step < a.heads[s] ? h0 + u * step : 0;
                const T* grow = g + h * a.g_head[s];
                gown[u].load(grow + (ln.in ? ln.c0 : 0));
                if constexpr (!IL) gfar[u].load(grow + (ln.in ? ln.other : 0));
                if constexpr (FMT >= 0) {
                    const int64_t row = t * a.heads[s] + h;
                    const uint8_t* qp = a.q[s] + row * stride + (ln.in ? ln.c0 : 0);
                    if constexpr (V == 8) {
                        const uint2 p = ld8_nt(qp);
                        q[u][0] = p.x;
                        q[u][V / 4 - 1] = p.y;
                    } else {
                        q[u][0] = *reinterpret_cast<const uint32_t*>(qp);
                    }
                    sc[u] = a.sc[s][row * nb + (ln.in ? ln.c0 >> 5 : 0)];
                } else {
                    xr[u].load(static_cast<const T*>(a.x[s]) + t * a.x_token[s] + h * a.x_head[s] +
                               (ln.in ? ln.c0 : 0));
                }
            }
            float w[V];
            ln.weights(a, s, ln.c0, w);
#pragma unroll
            for (int u = 0; u < kQkU; ++u) {
                const int h = h0 + u * step;
                const bool on = here && h < a.heads[s] && ln.in;
                float v[V], z[V], o[V], d[V];
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    z[e] = gown[u].get(e);
                    o[e] = IL ? 0.f : gfar[u].get(e);
                }
                if constexpr (FMT >= 0) {
#pragma unroll
                    for (int e = 0; e < V; e += 4) {
                        float f[4];
                        Ck<FMT>::unpack4(q[u][e / 4], Ck<FMT>::down(sc[u]), f);
#pragma unroll
                        for (int k = 0; k < 4; ++k) v[e + k] = f[k];
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < V; ++e) v[e] = xr[u].get(e);
                }
                if (ragged) {  // lanes past the head add nothing to its sums
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        z[e] = ln.in ? z[e] : 0.f;
                        o[e] = ln.in ? o[e] : 0.f;
                        v[e] = ln.in ? v[e] : 0.f;
                    }
                }
                float ss = 0.f, dot = 0.f;
#pragma unroll
                for (int e = 0; e < V; ++e) d[e] = ln.turn(z, o, c, sn, e, -1.f, a.R);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    ss += v[e] * v[e];
                    dot += d[e] * w[e] * v[e];
                }
                ss = lane_group_sum(ss, lg);
                dot = lane_group_sum(dot, lg);
                const float inv = !at.ok() ? __uint_as_float(0x7fc00000u) : 1.f / sqrtf(ss / (float)a.D + a.eps);
                const float k2 = dot * inv * inv * inv / (float)a.D;
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float p = on ? d[e] * v[e] * inv : 0.f;  // a head past the last adds nothing (inv may be infinite)
                    if (s == 0) dw[0][e] += p;
                    else dw[1][e] += p;
                    d[e] = w[e] * d[e] * inv - v[e] * k2;
                }
                if (on) qk_store<T, V>(static_cast<T*>(a.y[s]) + (t * a.heads[s] + h) * a.D + ln.c0, d);
            }
        }
    }
    // the wave's groups, then its channels to LDS
#pragma unroll
    for (int e = 0; e < V; ++e) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            float v = dw[s][e];
            for (int k = 1 << lg; k < 64; k <<= 1) v += __shfl_xor(v, k);
            if ((lane >> lg) == 0 && ln.in) red[(wave * 2 + s) * a.D + ln.c0 + e] = v;
        }
    }
    __syncthreads();
    const int64_t row = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
    for (int i = threadIdx.x; i < 2 * a.D; i += 512) {
        float v = 0.f;
        for (int w = 0; w < 8; ++w) v += red[w * 2 * a.D + i];
        dw_part[row * 2 * a.D + i] = v;
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

// V channels a lane (0: the kernels of any size) and log2 of the lanes a head.
struct QkTiling {
    int v, lg;
};
static QkTiling qk_tiling(int D, int R, bool interleaved) {
    for (int v = 8; v >= 4; v -= 4) {
        if (D % v != 0 || (!interleaved && R % (2 * v) != 0)) continue;
        int lg = v == 8 ? 2 : 3;  // a block of 32 channels lies in one group
        while ((v << lg) < D) ++lg;
        if (lg <= 6) return QkTiling{v, lg};
    }
    return QkTiling{0, 0};
}

// log2 of the tokens a wave takes at once: the fewest rounds a token (its tasks,
// and half a task for its table row) that leave two waves a CU (eight: 4188 x 1 +
// 1 heads of 64 fp32 int8, forward and backward 36 us, two 23); one token where
// that saves less than a quarter.
static int qk_tokens(const QkArgs& a, const QkTiling& t) {
    if (t.v == 0) return 0;
    const auto cost = [&](int tw) { return 2 * QkTasks(a.heads[0], a.heads[1], t.lg + tw).n + 1; };
    int best = 0;
    for (int tw = 1; t.lg + tw <= 6 && (a.T >> tw) >= 2 * (int64_t)device_cu_count(); ++tw)
        if (cost(tw) << best < cost(best) << tw) best = tw;
    return cost(best) * 4 <= (cost(0) << best) * 3 ? best : 0;
}

// Workgroups that share a wave's tasks: enough waves for the device.
static int qk_splits(int64_t waves, const QkTasks& tasks) {
    const int64_t want = 16 * (int64_t)device_cu_count();
    int64_t y = (want + waves - 1) / waves;
    if (y > tasks.n) y = tasks.n;
    return (int)(y < 1 ? 1 : y);
}

#define MHC_QK_TILED(dt, fmt, t, il, tw, ...)                                        \
    MHC_QK_TYPED(dt, fmt, {                                                          \
        auto tiled = [&](auto v_, auto il_) {                                        \
            constexpr int V_ = decltype(v_)::value;                                  \
            constexpr bool I_ = decltype(il_)::value;                                \
            if ((tw) > 0) { constexpr bool M_ = true; __VA_ARGS__; }                 \
            else { constexpr bool M_ = false; __VA_ARGS__; }                         \
        };                                                                           \
        using V8 = std::integral_constant<int, 8>;                                   \
        using V4 = std::integral_constant<int, 4>;                                   \
        if (t.v == 8) { if (il) tiled(V8{}, std::true_type{}); else tiled(V8{}, std::false_type{}); } \
        else { if (il) tiled(V4{}, std::true_type{}); else tiled(V4{}, std::false_type{}); }          \
    })

template <bool AX>
hipError_t qk_fwd_launch(int dt, int fmt, const QkArgs& a, hipStream_t s) {
    const int H = a.heads[0] + a.heads[1];
    if (a.T == 0 || H == 0) return hipSuccess;
    const QkTiling t = qk_tiling(a.D, a.R, a.interleaved);
    const int tw = qk_tokens(a, t);
    const int y = t.v == 0 ? (H + 3) / 4 : qk_splits(a.T >> tw, QkTasks(a.heads[0], a.heads[1], t.lg + tw));
    const int each = t.v == 0 ? 1 : 4 << tw;  // tokens a workgroup
    const int64_t most = (int64_t)1 << 23;  // workgroups along tokens a launch: 2^31 lanes
    const int tok = timing_begin("qk_norm_rope_fwd", s);
    hipError_t e = hipSuccess;
    QkArgs b = a;
    for (b.t0 = 0; b.t0 < a.T && e == hipSuccess; b.t0 += most * each) {
        const int64_t x = (a.T - b.t0 + each - 1) / each;
        const dim3 grid((unsigned)(x < most ? x : most), (unsigned)y);
        if (t.v == 0) {
            MHC_QK_TYPED(dt, fmt, MHC_LAUNCH_GGL((qk_fwd_any_kernel<T_, F_, AX>), grid, dim3(256), 0, s, b));
        } else {
            MHC_QK_TILED(dt, fmt, t, a.interleaved, tw,
                         MHC_LAUNCH_GGL((qk_fwd_kernel<T_, F_, V_, I_, M_, AX>), grid, dim3(256), 0, s, b, t.lg, tw));
        }
        e = hipGetLastError();
    }
    timing_end(tok, s);
    return e;
}

static dim3 qk_bwd_dims(const QkArgs& a) {
    const QkTiling t = qk_tiling(a.D, a.R, a.interleaved);
    const int64_t two = 2 * (int64_t)device_cu_count();
    if (a.T == 0) return dim3(1, 1);
    if (t.v == 0) return dim3((unsigned)(a.T < two ? a.T : two), 1);
    // the split with the fewest rounds: sweeps over the tokens times a wave's
    // tasks a token and half a task for its table row
    const int tw = qk_tokens(a, t);
    const int n = QkTasks(a.heads[0], a.heads[1], t.lg + tw).n;
    const int64_t x = (a.T + (8 << tw) - 1) / (8 << tw);
    int64_t best = INT64_MAX, bx = 1;
    int by = 1;
    for (int y = 1; y <= n && y <= two; ++y) {
        const int64_t most = two / y, gx = x < most ? x : most;
        const int64_t cost = (x + gx - 1) / gx * (2 * ((n + y - 1) / y) + 1);
        if (cost <= best) {
            best = cost;
            bx = gx;
            by = y;
        }
    }
    return dim3((unsigned)bx, (unsigned)by);
}

template <bool AX>
hipError_t qk_bwd_launch(int dt, int fmt, const QkArgs& a, float* dw_part, hipStream_t s) {
    const QkTiling t = qk_tiling(a.D, a.R, a.interleaved);
    const dim3 grid = qk_bwd_dims(a);
    const int tok = timing_begin("qk_norm_rope_bwd", s);
    if (t.v == 0) {
        MHC_QK_TYPED(dt, fmt,
                     MHC_LAUNCH_GGL((qk_bwd_any_kernel<T_, F_, AX>), grid, dim3(256), (size_t)a.D * 8 * sizeof(float), s,
                                    a, dw_part));
    } else {
        const int tw = qk_tokens(a, t);
        MHC_QK_TILED(dt, fmt, t, a.interleaved, tw,
                     MHC_LAUNCH_GGL((qk_bwd_kernel<T_, F_, V_, I_, M_, AX>), grid, dim3(512),
                                    (size_t)a.D * 16 * sizeof(float), s, a, t.lg, tw, dw_part));
    }
    timing_end(tok, s);
    return hipGetLastError();
}

}  // namespace mhc
