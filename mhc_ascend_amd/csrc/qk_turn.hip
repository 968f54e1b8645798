// Rotation of queries' and keys' heads by their tokens' positions, on one axis or
// several, by the angle or (the backward) its negative:
//   (a, b) -> (a c - b s, b c + a s)  for the pairs of the first R channels;
// pairs, tables, axes and positions outside the table as in mhc_qk.h.  Channels
// past R stay.
#include "mhc_qk.h"

namespace mhc {

// ---------------------------------------------------------------------------
// Any head size, stride and alignment: one wave a head row, one channel a lane.
// For heads that qk_turn_tiling finds no pieces for.
// ---------------------------------------------------------------------------
template <typename T, bool AX>
__global__ __launch_bounds__(256) void qk_turn_any_kernel(QkArgs a) {
    const int lane = threadIdx.x & 63;
    const int hh = blockIdx.y * 4 + (threadIdx.x >> 6);
    if (hh >= a.heads[0] + a.heads[1]) return;  // whole waves, no barrier below
    const int64_t t = a.t0 + blockIdx.x;
    const int s = hh < a.heads[0] ? 0 : 1;
    const int h = s ? hh - a.heads[0] : hh;
    const T* x = static_cast<const T*>(a.x[s]) + t * a.x_token[s] + h * a.x_head[s];
    T* y = static_cast<T*>(a.y[s]) + (t * a.heads[s] + h) * a.D;
    const QkAt<AX> at(a, t, QkRaw<AX>(a, t));
    const float way = a.inverse ? -1.f : 1.f;
    for (int d = lane; d < a.D; d += 64) {
        float o = VecIO<T>::scalar(x + d);
        int col, other;
        float sign;
        if (qk_pair(a, d, col, other, sign)) {
            const int64_t tab = at.of(a, col);
            o = o * a.cos[tab + col] + way * sign * VecIO<T>::scalar(x + other) * a.sin[tab + col];
        }
        VecIO<T>::put(y + d, at.ok() ? o : __uint_as_float(0x7fc00000u));
    }
}

// ---------------------------------------------------------------------------
// Heads of whole pieces of V channels.  A lane takes a unit of two pieces: with
// halves a piece of the first half and its partner of the second, interleaved two
// neighbouring pieces, and past R two pieces that stay.  So every channel is read
// once, no value crosses lanes, and the V table entries of the unit stay in
// registers for all heads of the token.  A group of 2^lg lanes takes a head, a
// wave 64 >> lg heads of a token (or of 2^tw tokens where heads are few) at a
// time, U such steps in flight.
// ---------------------------------------------------------------------------
template <int V, bool IL>
struct QkUnit {
    int c[2];      // its pieces' first channels
    bool in[2];    // within the head
    bool turned;   // some channel of the unit rotates
    uint32_t ax;   // the axes of its pairs (with AX)

    template <bool AX>
    __device__ __forceinline__ QkUnit(const QkArgs& a, int lane, int lg, std::bool_constant<AX>) {
        const int u = lane & ((1 << lg) - 1);
        if constexpr (IL) {
            c[0] = 2 * u * V;
            c[1] = c[0] + V;
            turned = c[0] < a.R;
        } else {
            const int half = a.R >> 1, n = half / V;
            turned = u < n;
            c[0] = turned ? u * V : a.R + 2 * (u - n) * V;
            c[1] = turned ? c[0] + half : c[0] + V;
        }
        in[0] = c[0] < a.D;
        in[1] = c[1] < a.D;
        ax = AX ? qk_axes_of<V>(a, turned ? (IL ? c[0] >> 1 : c[0]) : 0) : 0u;
    }

    // The entries of the unit's V pairs: with halves pair c[0] + e, interleaved
    // pair c[0] / 2 + e.
    template <bool AX>
    __device__ __forceinline__ void table(const QkArgs& a, const QkAt<AX>& row, float way, float (&cs)[V],
                                          float (&sn)[V]) const {
        const int half = a.R >> 1, col = IL ? c[0] >> 1 : c[0];
        const uint32_t m = AX ? qk_opaque(ax) : 0u;
        if ((!IL || a.R % (2 * V) == 0) && (!AX || a.whole)) {
            const int first = turned ? col : 0;
            const int64_t at = row.on(m) + first;
            QkPiece<float, V> qc, qs;
            qc.load(a.cos + at);
            qs.load(a.sin + at);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                cs[e] = qc.get(e);
                sn[e] = way * qs.get(e);
            }
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const int p = turned && col + e < half ? col + e : 0;
                const int64_t at = row.on(m >> (2 * e)) + p;
                cs[e] = a.cos[at];
                sn[e] = a.sin[at];
            }
            __builtin_amdgcn_sched_barrier(0);  // all loads, then their uses
#pragma unroll
            for (int e = 0; e < V; ++e) sn[e] *= way;
        }
    }

    __device__ __forceinline__ void turn(const QkArgs& a, const float (&cs)[V], const float (&sn)[V], float (&v)[2][V],
                                         bool ok) const {
        if constexpr (IL) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                float& x = v[e / (V / 2)][2 * (e % (V / 2))];
                float& y = v[e / (V / 2)][2 * (e % (V / 2)) + 1];
                const float p = x * cs[e] - y * sn[e], q = y * cs[e] + x * sn[e];
                const bool on = c[0] + 2 * e < a.R;
                x = on ? p : x;
                y = on ? q : y;
            }
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float p = v[0][e] * cs[e] - v[1][e] * sn[e], q = v[1][e] * cs[e] + v[0][e] * sn[e];
                v[0][e] = turned ? p : v[0][e];
                v[1][e] = turned ? q : v[1][e];
            }
        }
        if (!ok) {
#pragma unroll
            for (int e = 0; e < V; ++e) v[0][e] = v[1][e] = __uint_as_float(0x7fc00000u);
        }
    }
};

template <typename T, int V, bool IL, bool AX>
__global__ __launch_bounds__(256) void qk_turn_kernel(QkArgs a, int lg, int tw) {
    const int lane = threadIdx.x & 63;
    int64_t t = a.t0 + (((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) << tw);
    if (t >= a.T) return;
    const QkUnit<V, IL> un(a, lane, lg, std::bool_constant<AX>{});
    const QkTasks tasks(a.heads[0], a.heads[1], lg + tw);
    const int step = 64 >> (lg + tw), sub = (lane >> lg) & (step - 1);
    t += lane >> (6 - tw);
    const bool here = t < a.T;
    t = here ? t : a.T - 1;
    using Piece = std::conditional_t<V == 8, CkPiece<T>, QkPiece<T, V>>;
    struct Rows {
        Piece p[kQkU][2];
    };
    const auto side = [&](int j) { return j < tasks.nq ? 0 : 1; };
    const auto first = [&](int j, int s) { return (s ? j - tasks.nq : j) * tasks.per + sub; };
    const auto fetch = [&](int j, Rows& r) {
        const int s = side(j), h0 = first(j, s);
        const T* base = static_cast<const T*>(a.x[s]) + t * a.x_token[s];
#pragma unroll
        for (int u = 0; u < kQkU; ++u) {
            const int h = h0 + u * step;
            const T* row = base + (h < a.heads[s] ? h : 0) * a.x_head[s];
#pragma unroll
            for (int k = 0; k < 2; ++k) r.p[u][k].load(row + (un.in[k] ? un.c[k] : 0));
        }
    };
    int j = blockIdx.y;
    const QkRaw<AX> raw(a, t);
    Rows next;
    fetch(j, next);  // the grid's y is at most the number of tasks
    const QkAt<AX> at(a, t, raw);
    float cs[V], sn[V];
    un.table(a, at, a.inverse ? -1.f : 1.f, cs, sn);
    for (; j < tasks.n; j += gridDim.y) {
        const int s = side(j), h0 = first(j, s);
        const Rows rows = next;
        if (j + (int)gridDim.y < tasks.n) fetch(j + gridDim.y, next);
#pragma unroll
        for (int u = 0; u < kQkU; ++u) {
            const int h = h0 + u * step;
            float v[2][V];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                if constexpr (V == 8) {
                    rows.p[u][k].get(v[k]);
                } else {
#pragma unroll
                    for (int e = 0; e < V; ++e) v[k][e] = rows.p[u][k].get(e);
                }
            }
            un.turn(a, cs, sn, v, at.ok());
            if (here && h < a.heads[s]) {
                T* y = static_cast<T*>(a.y[s]) + (t * a.heads[s] + h) * a.D;
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    if (un.in[k]) qk_store<T, V>(y + un.c[k], v[k]);
            }
        }
    }
}

// V channels a piece (0: the kernel of any size) and log2 of the lanes a head.
static QkTiling qk_turn_tiling(int D, int R, bool interleaved) {
    for (int v = 8; v >= 4; v -= 4) {
        if (D % v != 0 || (!interleaved && R % (2 * v) != 0)) continue;
        const int units = interleaved ? (D + 2 * v - 1) / (2 * v) : R / (2 * v) + ((D - R) / v + 1) / 2;
        int lg = 0;
        while ((1 << lg) < units) ++lg;
        if (lg <= 6) return QkTiling{v, lg};
    }
    return QkTiling{0, 0};
}

hipError_t launch_qk_rope(int dt, const QkArgs& a, hipStream_t s) {
    const int H = a.heads[0] + a.heads[1];
    if (a.T == 0 || H == 0) return hipSuccess;
    const QkTiling t = qk_turn_tiling(a.D, a.R, a.interleaved);
    const int tw = qk_tokens(a, t);
    const int y = t.v == 0 ? (H + 3) / 4 : qk_splits(a.T >> tw, QkTasks(a.heads[0], a.heads[1], t.lg + tw));
    const int each = t.v == 0 ? 1 : 4 << tw;  // tokens a workgroup
    const int64_t most = (int64_t)1 << 23;  // workgroups along tokens a launch: 2^31 lanes
    const int tok = timing_begin("qk_rope", s);
    hipError_t e = hipSuccess;
    QkArgs b = a;
    b.whole = t.v != 0 && !a.dealt;
    for (int i = 0; i + 1 < a.axes; ++i)
        if (t.v != 0 && a.part[i] % t.v != 0) b.whole = 0;
    for (b.t0 = 0; b.t0 < a.T && e == hipSuccess; b.t0 += most * each) {
        const int64_t x = (a.T - b.t0 + each - 1) / each;
        const dim3 grid((unsigned)(x < most ? x : most), (unsigned)y);
        const auto run = [&](auto z_, auto ax_) {
            using T_ = decltype(z_);
            constexpr bool A_ = decltype(ax_)::value;
            if (t.v == 0) {
                MHC_LAUNCH_GGL((qk_turn_any_kernel<T_, A_>), grid, dim3(256), 0, s, b);
            } else if (t.v == 8 && a.interleaved) {
                MHC_LAUNCH_GGL((qk_turn_kernel<T_, 8, true, A_>), grid, dim3(256), 0, s, b, t.lg, tw);
            } else if (t.v == 8) {
                MHC_LAUNCH_GGL((qk_turn_kernel<T_, 8, false, A_>), grid, dim3(256), 0, s, b, t.lg, tw);
            } else if (a.interleaved) {
                MHC_LAUNCH_GGL((qk_turn_kernel<T_, 4, true, A_>), grid, dim3(256), 0, s, b, t.lg, tw);
            } else {
                MHC_LAUNCH_GGL((qk_turn_kernel<T_, 4, false, A_>), grid, dim3(256), 0, s, b, t.lg, tw);
            }
        };
        const auto typed = [&](auto z_) {
            if (a.axes > 1) run(z_, std::true_type{});
            else run(z_, std::false_type{});
        };
        if (dt == kBF16) typed(bf16_t{});
        else typed(float{});
        e = hipGetLastError();
    }
    timing_end(tok, s);
    return e;
}

}  // namespace mhc
