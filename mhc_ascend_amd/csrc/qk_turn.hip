// Rotation of queries' and keys' heads by their tokens' positions, on one axis or
// several, by the angle or (the backward) its negative:
//   (a, b) -> (a c - b s, b c + a s)  for the pairs of the first R channels;
// pairs, tables, axes and positions outside the table as in mhc_qk.h.  Channels
// past R stay.
#include <algorithm>

#include "mhc_qk.h"

namespace mhc {

// ---------------------------------------------------------------------------
// Any head size, stride and alignment: one wave a head row, one channel a lane.
// For heads that qk_turn_plan finds no pieces for: sizes that are no multiple of 4 (or
// too wide), and halves of an R that is no multiple of 8.  Bound by its instructions:
// forward and backward of 9147 x 40 heads of 72 bf16, 36 turned in halves, 159 us, on
// three axes 235 (72 turned: 38).
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
// halves a piece of the first half and its partner of the second, interleaved one of
// the head's first units and one behind them, and past R two pieces that stay, taken
// likewise: neighbouring lanes' loads lie next to each other (forward and backward of
// 16384 x 64 heads of 128 bf16 by pairs 184 us, of units of two neighbouring pieces
// 222; 16384 x 40 of 256 bf16, 128 turned, 235 and 286).  So every channel is read
// once, no value crosses lanes, and the V table entries of the unit stay in
// registers for all heads of the token.  Nothing is summed over a head, so its
// lanes are as many as its units, and a wave holds 64 / units heads; the queries'
// and the keys' are one list.  A task is U steps of it, its loads in flight
// together with the next task's.  Few heads: a wave's are those of several tokens.
// Few tokens: their tasks are spread over the grid's y.
// Lanes and steps with nothing of their own repeat another's work, store included:
// with branches around the stores the loads are waited for one by one.  Bound by
// bytes: 16384 x 64 heads of 128 bf16 on three axes 91 us, 5.9 TB/s; 16384 x 40 of 112
// bf16 56 us, 5.2; 13794 x 48 of 112 bf16, 56 turned by pairs dealt to four axes, 58 us,
// 5.1.  The keys' tasks apart from the queries': 16384 x 40 of 112 69 us for 67, 15643
// x 2 of 112 bf16 11 for 9.  16 x 40 heads: 4.6 us, the latency of positions, table and
// rows.
// ---------------------------------------------------------------------------
// How a wave is shared: units a head, heads a token takes at once, tokens, tasks;
// mul = ceil(2^16 / n) divides a lane or slot (under 64) by n exactly.
struct QkTurnPlan {
    int v, u, units, heads, tokens, n;
    uint32_t units_mul, heads_mul;
};

template <int V, bool IL>
struct QkUnit {
    int c[2];      // its pieces' first channels (the first again where the second is past the head)
    bool turned;   // its channels rotate (with halves)
    uint32_t ax;   // the axes of its pairs (with AX)

    template <bool AX>
    __device__ __forceinline__ QkUnit(const QkArgs& a, int u, int units, std::bool_constant<AX>) {
        if constexpr (IL) {
            c[0] = u * V;
            c[1] = c[0] + units * V;
        } else {
            const int half = a.R >> 1, n = half / V;
            turned = u < n;
            c[0] = turned ? u * V : a.R + (u - n) * V;
            c[1] = c[0] + (turned ? half : (units - n) * V);
        }
        if (c[1] >= a.D) c[1] = c[0];
        if constexpr (!AX) ax = 0u;
        else if constexpr (IL) ax = qk_axes_of<V / 2>(a, c[0] >> 1) | qk_axes_of<V / 2>(a, c[1] >> 1) << V;
        else ax = qk_axes_of<V>(a, turned ? c[0] : 0);
    }

    // The entries of the unit's V pairs: with halves pair c[0] + e, interleaved
    // pairs c[0] / 2 + e, then c[1] / 2 + e.
    template <bool AX>
    __device__ __forceinline__ void table(const QkArgs& a, const QkAt<AX>& row, float way, float (&cs)[V],
                                          float (&sn)[V]) const {
        constexpr int N = IL ? V / 2 : V;  // pairs next to each other
        const int half = a.R >> 1;
        const uint32_t m = AX ? qk_opaque(ax) : 0u;
        const auto first = [&](int k) { return IL ? c[k] >> 1 : c[0]; };
        if ((!IL || a.R % V == 0) && (!AX || a.whole)) {
#pragma unroll
            for (int k = 0; k < V / N; ++k) {
                const int64_t at = row.on(m >> (2 * N * k)) + (first(k) < half ? first(k) : 0);
                QkPiece<float, N> qc, qs;
                qc.load(a.cos + at);
                qs.load(a.sin + at);
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    cs[k * N + e] = qc.get(e);
                    sn[k * N + e] = way * qs.get(e);
                }
            }
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const int p = first(e / N) + e % N;
                const int64_t at = row.on(m >> (2 * e)) + (p < half ? p : 0);
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
                const bool on = c[e / (V / 2)] + 2 * (e % (V / 2)) < a.R;
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

// Rows past the caches (NT), where every load and store takes whole lines: halves of
// the turned channels and of the others of a multiple of 128 bytes.  In others the unit's two pieces share lines, which
// have to stay (forward and backward, streamed and not: 16384 x 64 heads of 128
// bf16 186 and 195 us, by neighbouring pairs 184 and 203; 32768 x 40 of 96 bf16 330
// and 206).
template <typename T, int V, bool NT>
struct QkTurnPiece : QkPiece<T, V> {
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (!NT) QkPiece<T, V>::load(p);
        else if constexpr (sizeof(T) == 4) this->w = __builtin_nontemporal_load(reinterpret_cast<const ck_u4_a4_t*>(p));
        else if constexpr (V == 8) this->w = __builtin_nontemporal_load(reinterpret_cast<const ck_u4_a2_t*>(p));
        else this->w = __builtin_nontemporal_load(reinterpret_cast<const qk_u2_a2_t*>(p));
    }
};

template <typename T, int V, bool NT>
__device__ __forceinline__ void qk_turn_store(T* p, const float (&v)[V]) {
    if constexpr (NT) {
        qk_store<T, V>(p, v);
    } else if constexpr (V == 8) {
        ck_store8<false>(p, v);
    } else if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<ck_u4_a4_t*>(p) = ck_u4_t{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]),
                                                    __float_as_uint(v[3])};
    } else {
        *reinterpret_cast<qk_u2_a2_t*>(p) = qk_u2_t{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
    }
}

template <typename T, int V, int U, bool IL, bool AX, bool NT>
__global__ __launch_bounds__(256) void qk_turn_kernel(QkArgs a, QkTurnPlan pl) {
    const int lane = threadIdx.x & 63;
    int slot = (int)(((uint32_t)lane * pl.units_mul) >> 16);
    const int unit = lane - slot * pl.units;
    slot = slot < pl.heads * pl.tokens ? slot : 0;
    const int tok = (int)(((uint32_t)slot * pl.heads_mul) >> 16);
    const int sub = slot - tok * pl.heads;
    int64_t t = a.t0 + ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * pl.tokens;
    if (t >= a.T) return;
    t = t + tok < a.T ? t + tok : a.T - 1;
    const QkUnit<V, IL> un(a, unit, pl.units, std::bool_constant<AX>{});
    const QkRaw<AX> raw(a, t);
    struct Rows {
        QkTurnPiece<T, V, NT> p[U][2];
    };
    // row `h` of the token's list begins at base[s] + h * stride, its side s
    const int H = a.heads[0], last = H + a.heads[1] - 1;
    const auto head = [&](int j, int u) {
        const int h = (j * U + u) * pl.heads + sub;
        return h < last ? h : last;
    };
    const int64_t in0 = t * a.x_token[0], in1 = t * a.x_token[1] - H * a.x_head[1];
    const int64_t out0 = t * H * a.D, out1 = (t * a.heads[1] - H) * a.D;
    const auto fetch = [&](int j, Rows& r) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int h = head(j, u);
            const bool q = h < H;
            const T* row = static_cast<const T*>(q ? a.x[0] : a.x[1]) + (q ? in0 : in1) +
                           h * (q ? a.x_head[0] : a.x_head[1]);
#pragma unroll
            for (int k = 0; k < 2; ++k) r.p[u][k].load(row + un.c[k]);
        }
    };
    int j = blockIdx.y;
    Rows next;
    fetch(j, next);  // the grid's y is at most the number of tasks
    const QkAt<AX> at(a, t, raw);
    float cs[V], sn[V];
    un.table(a, at, a.inverse ? -1.f : 1.f, cs, sn);
    for (; j < pl.n; j += gridDim.y) {
        const Rows rows = next;
        if (j + (int)gridDim.y < pl.n) fetch(j + gridDim.y, next);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float v[2][V];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
#pragma unroll
                for (int e = 0; e < V; ++e) v[k][e] = rows.p[u][k].get(e);
            }
            un.turn(a, cs, sn, v, at.ok());
            const int h = head(j, u);
            T* y = static_cast<T*>(h < H ? a.y[0] : a.y[1]) + (h < H ? out0 : out1) + (int64_t)h * a.D;
#pragma unroll
            for (int k = 0; k < 2; ++k) qk_turn_store<T, V, NT>(y + un.c[k], v[k]);
        }
    }
}

static QkTurnPlan qk_turn_plan(const QkArgs& a, int dt) {
    QkTurnPlan p{};
    // pieces of 16 bytes, or of 4 channels
    for (int v = dt == kBF16 ? 8 : 4; v >= 4 && p.v == 0; v -= 4) {
        if (a.D % v != 0 || (!a.interleaved && a.R % (2 * v) != 0)) continue;
        const int pieces = a.interleaved ? a.D / v : (a.D - a.R) / v;
        p.units = (pieces + 1) / 2 + (a.interleaved ? 0 : a.R / (2 * v));
        if (p.units <= 64) p.v = v;
    }
    if (p.v == 0) return p;
    const int slots = 64 / p.units, H = a.heads[0] + a.heads[1];
    // several tokens a wave where that saves a quarter of its steps and leaves
    // twelve waves a CU
    int64_t best = INT64_MAX;
    int steps = 0;
    for (int n = 1; n <= slots && (n == 1 || a.T / n >= 12 * (int64_t)device_cu_count()); ++n) {
        const int need = (H + slots / n - 1) / (slots / n);
        const int64_t cost = (int64_t)need * 10080 / n;
        if (n > 1 && cost * 4 > best * 3) continue;
        best = cost;
        steps = need;
        p.heads = slots / n;
        p.tokens = n;
    }
    // the longest tasks that leave the fewest steps idle
    for (int u = 4; u >= 1; u /= 2) {
        const int n = (steps + u - 1) / u;
        if (p.u != 0 && n * u >= p.n * p.u) continue;
        p.u = u;
        p.n = n;
    }
    p.units_mul = (65536u + (uint32_t)p.units - 1u) / (uint32_t)p.units;
    p.heads_mul = (65536u + (uint32_t)p.heads - 1u) / (uint32_t)p.heads;
    return p;
}

hipError_t launch_qk_rope(int dt, const QkArgs& a, hipStream_t s) {
    const int H = a.heads[0] + a.heads[1];
    if (a.T == 0 || H == 0) return hipSuccess;
    const QkTurnPlan p = qk_turn_plan(a, dt);
    const int each = p.v == 0 ? 1 : 4 * p.tokens;  // tokens a workgroup
    int y = (H + 3) / 4;
    if (p.v != 0) {  // four waves a CU, each with tasks of its own: every one loads the tables
        const int64_t waves = (a.T + p.tokens - 1) / p.tokens, want = 4 * (int64_t)device_cu_count();
        y = (int)std::min<int64_t>(p.n, (want + waves - 1) / waves);
    }
    // whole lines, and from 96 MiB of rows on: the two cross between 80 and 120 MiB
    // (128 bf16, streamed and not, forward: 4096 x 40 heads 19 and 16 us, 8192 x 40 33
    // and 32; with its backward 12288 x 40 97 and 102, 16384 x 40 125 and 133)
    const int64_t bytes = dt == kBF16 ? 2 : 4;
    const bool lines = a.D * bytes % 256 == 0 && (a.interleaved || a.R * bytes % 256 == 0) &&
                       a.T * H * a.D * bytes >= (int64_t)96 << 20;
    const int64_t most = (int64_t)1 << 23;  // workgroups along tokens a launch: 2^31 lanes
    const int tok = timing_begin("qk_rope", s);
    hipError_t e = hipSuccess;
    QkArgs b = a;
    b.whole = p.v != 0 && !a.dealt;
    for (int i = 0; i + 1 < a.axes; ++i)
        if (p.v != 0 && a.part[i] % (a.interleaved ? p.v / 2 : p.v) != 0) b.whole = 0;
    for (b.t0 = 0; b.t0 < a.T && e == hipSuccess; b.t0 += most * each) {
        const int64_t x = (a.T - b.t0 + each - 1) / each;
        const dim3 grid((unsigned)(x < most ? x : most), (unsigned)y);
        const auto run = [&](auto z_, auto ax_) {
            using T_ = decltype(z_);
            constexpr bool A_ = decltype(ax_)::value;
            if (p.v == 0) {
                MHC_LAUNCH_GGL((qk_turn_any_kernel<T_, A_>), grid, dim3(256), 0, s, b);
                return;
            }
            const auto steps = [&](auto v_, auto il_) {
                constexpr int V_ = decltype(v_)::value;
                constexpr bool I_ = decltype(il_)::value;
                const auto go = [&](auto u_) {
                    constexpr int U_ = decltype(u_)::value;
                    if (lines) {
                        MHC_LAUNCH_GGL((qk_turn_kernel<T_, V_, U_, I_, A_, true>), grid, dim3(256), 0, s, b, p);
                    } else {
                        MHC_LAUNCH_GGL((qk_turn_kernel<T_, V_, U_, I_, A_, false>), grid, dim3(256), 0, s, b, p);
                    }
                };
                if (p.u == 4) go(std::integral_constant<int, 4>{});
                else if (p.u == 2) go(std::integral_constant<int, 2>{});
                else go(std::integral_constant<int, 1>{});
            };
            const auto pieces = [&](auto v_) {
                if (a.interleaved) steps(v_, std::true_type{});
                else steps(v_, std::false_type{});
            };
            if constexpr (sizeof(T_) == 2) {
                if (p.v == 8) {
                    pieces(std::integral_constant<int, 8>{});
                    return;
                }
            }
            pieces(std::integral_constant<int, 4>{});
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
