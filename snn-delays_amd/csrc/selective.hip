// Selective state-space recurrence over (T, B, N) sequences with S states a channel, its reverse pass
// and its one-step form.
//     d_t = softplus(dt_t + dt_bias), a_t = exp(d_t A), u_t = d_t x_t
//     h_t = a_t h_{t-1} + u_t B_t,  c_t = <C_t, h_t> + D x_t,  y_t = c_t silu(g_t)
// (A (N, S); B and C (T, B, S), shared by all channels; h (B, N, S) in 32 bits). Backwards, with the
// core's gradient w_t = dy_t silu(g_t) and the carry k_t = a_t l_t (k_T = dlast):
//     l_t = w_t C_t + k_{t+1},  q_t = k_t h_{t-1}
//     dx = d <l, B> + D w,  dd = <A, q> + x <l, B>,  ddt = dd sigmoid(dt + dt_bias),
//     dg = dy c silu'(g),  dA = sum d q,  dB = sum_n l u,  dC = sum_n w h,  dh0 = k_0.
//
// Q lanes hold a channel, K states each. What a channel needs once a step (softplus, the gate, loads
// and stores) its lanes take in turn, a step each; the steps' values then reach the other lanes as
// DPP operands of the multiplications that use them. B and C of a block of steps are staged in LDS
// in 32 bits. The sums over states that end a step (y; backwards also <l, B> and <A, q>) are taken for
// Q steps together, half of them handed over in each exchange, and land in the lane of their step.
//
// The forward keeps the state before every 16th step; the backward runs 16 steps from there, holds
// their decays and states in registers and walks back. The sums over channels (dB, dC) go through
// the wave's lanes, the workgroup's LDS and one set of sums for each workgroup of channels in memory,
// added up in a second launch in a fixed order, as dA, dD and the bias' over the rows.
#include <algorithm>
#include <utility>

#include "gated.h"
#include "kernels.h"

namespace delrec {

namespace {

constexpr int kStepsB = DELREC_SELECTIVE_BLOCK;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kWavesWg = 4;

template <int... I, class F>
__device__ __forceinline__ void each_of(std::integer_sequence<int, I...>, F&& f) { (f(std::integral_constant<int, I>()), ...); }
template <int N, class F>
__device__ __forceinline__ void each(F&& f) { each_of(std::make_integer_sequence<int, N>(), f); }
template <int N, class F>
__device__ __forceinline__ void each_back(F&& f) {
    each<N>([&](auto i) { f(std::integral_constant<int, N - 1 - decltype(i)::value>()); });
}

// log(1 + e^x), and its slope. With e = e^-|x| and s = e / (2 + e) <= 1/3 it is max(x, 0) + 2 atanh(s),
// the series in s^2 by a polynomial (1.6e-8 relative): small values keep their last digits, which
// log(1 + e) loses.
__device__ __forceinline__ float softplus(float x, float* slope) {
    const float e = __builtin_amdgcn_exp2f(-fabsf(x) * kLog2e);
    const float s = e * __builtin_amdgcn_rcpf(2.0f + e), z = s * s;
    const float p = fmaf(fmaf(fmaf(0.13425749f, z, 0.1411831f), z, 0.2000378f), z, 0.3333332f);
    const float r = __builtin_amdgcn_rcpf(1.0f + e);
    *slope = x >= 0.0f ? r : e * r;
    return fmaxf(x, 0.0f) + 2.0f * fmaf(s * z, p, s);
}
__device__ __forceinline__ float sigmoid(float x) { return gate_in(-x); }

// lane I's value in each group of Q lanes
template <int Q, int I>
__device__ __forceinline__ float from_lane(float v) {
    constexpr int ctrl = Q == 4 ? I * 0x55 : 0x150 + I;     // quad_perm, row_newbcast
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), ctrl, 0xF, 0xF, true));
}
template <int CTRL>
__device__ __forceinline__ float add_dpp(float v, float w) {
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(w), CTRL, 0xF, 0xF, true));
}

// v[i] summed over the group's Q lanes, in lane i. Each exchange pairs lanes that differ in one bit
// (and in lower ones, which the later exchanges cover) and halves the values a lane holds.
template <int H, int CTRL>
__device__ __forceinline__ void hand_over(float* v, bool upper) {
#pragma unroll
    for (int i = 0; i < H; ++i) {
        const float keep = upper ? v[i + H] : v[i], give = upper ? v[i] : v[i + H];
        v[i] = add_dpp<CTRL>(keep, give);
    }
}
template <int Q>
__device__ __forceinline__ float sums_by_lane(float* v, int j) {
    if constexpr (Q == 16) {
        hand_over<8, 0x140>(v, j & 8);       // row_mirror: lane ^ 15
        hand_over<4, 0x141>(v, j & 4);       // row_half_mirror: lane ^ 7
    }
    hand_over<2, 0x4E>(v, j & 2);
    hand_over<1, 0xB1>(v, j & 1);
    return v[0];
}
template <int Q>
__device__ __forceinline__ float lanes_total(float v) {
    return group_sum_t<Q>(v);
}

__device__ __forceinline__ void swap32(float& a, float& b) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    a = __uint_as_float(r[0]);
    b = __uint_as_float(r[1]);
}
__device__ __forceinline__ void swap16(float& a, float& b) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    a = __uint_as_float(r[0]);
    b = __uint_as_float(r[1]);
}

// K of a lane's states (the first at column s0 of S); columns past S read 0 and are not written
template <int K>
__device__ __forceinline__ void load_states(float* v, const float* row, int s0, int S, bool on) {
    if (on && s0 + K <= S) {
        const auto t = vload<float, K>(row + s0);
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = t.get(k);
    } else {
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = on && s0 + k < S ? row[s0 + k] : 0.0f;
    }
}
template <int K>
__device__ __forceinline__ void store_states(float* row, const float* v, int s0, int S, bool on) {
    if (on && s0 + K <= S) {
        vstore<float, K>(row + s0, v);
    } else {
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (on && s0 + k < S) row[s0 + k] = v[k];
    }
}

template <int Q>
struct Shape {
    static constexpr int channels = 64 / Q * kWavesWg;      // of a workgroup
    static constexpr int own = kStepsB / Q;                 // steps of a block that a lane takes
};

// a workgroup's row and channels, a lane's channel and states
template <int Q, int K>
struct Place {
    int b, tile, w, lane, j, n, s0;
    bool on;
    __device__ __forceinline__ Place(const Selective& p) {
        const long long id = (long long)p.first + blockIdx.x;
        b = (int)(id / p.tiles);
        tile = (int)(id - (long long)b * p.tiles);
        lane = threadIdx.x & 63;
        w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        j = lane % Q;
        const int c = tile * Shape<Q>::channels + w * (64 / Q) + lane / Q;
        on = c < p.N;
        n = on ? c : p.N - 1;
        s0 = j * K;
    }
};

__device__ __forceinline__ int row_steps(const Selective& p, int b) {
    if (!p.lengths) return p.T;
    const int64_t v = p.lengths[b];
    return v < 0 ? 0 : (v < p.T ? (int)v : p.T);
}

// bit i: a sequence starts at step t0 + i
__device__ __forceinline__ uint32_t start_bits(const Selective& p, int b, int t0, int tend, int lane) {
    if (!p.starts) return 0;
    const int t = t0 + lane;
    return (uint32_t)__ballot(lane < kStepsB && t < tend && p.starts[(size_t)min(t, p.T - 1) * p.B + b] != 0);
}

// B and C of a block of steps, from memory to LDS as fp32; zeros past the row's end and past S
template <class E, int SP>
struct Stage {
    static constexpr int count = kStepsB * 2 * SP, per = (count + 255) / 256;
    E v[per];
    __device__ __forceinline__ void load(const Selective& p, int b, int t0, int tend) {
#pragma unroll
        for (int r = 0; r < per; ++r) {
            const int e = threadIdx.x + 256 * r, t = t0 + e / (2 * SP), s = e % SP;
            const delrec_rows& m = e / SP % 2 ? p.C : p.Bm;
            v[r] = (E)0.0f;
            if (e < count && t < tend && s < p.S) v[r] = ((const E*)m.data)[t * m.s0 + b * m.s1 + s];
        }
    }
    __device__ __forceinline__ void put(float* lds) const {
#pragma unroll
        for (int r = 0; r < per; ++r) {
            const int e = threadIdx.x + 256 * r;
            if (e < count) lds[e] = (float)v[r];
        }
    }
};

// a lane's own steps of a block of one of the (T, B, N) inputs; zeros past the row's end
template <class E, int Q>
struct Own {
    E v[Shape<Q>::own];
    __device__ __forceinline__ void load(const delrec_rows& x, const char* at, int t0, int j, int tend, bool on) {
#pragma unroll
        for (int i = 0; i < Shape<Q>::own; ++i) {
            const int t = t0 + i * Q + j;
            v[i] = (E)0.0f;
            if (on && t < tend) v[i] = ((const E*)at)[t * x.s0];
        }
    }
};
template <class E>
__device__ __forceinline__ const char* column(const delrec_rows& x, int b, int n) {
    return (const char*)((const E*)x.data + b * x.s1 + n);
}

}  // namespace

template <class E, int Q, int K>
__global__ void __launch_bounds__(256) selective_fwd_kernel(Selective p) {
    constexpr int SP = Q * K;
    __shared__ __align__(16) float bc[2][kStepsB][2][SP];
    const Place<Q, K> at(p);
    const int b = at.b, n = at.n, j = at.j, N = p.N, S = p.S;
    const size_t row = ((size_t)b * N + n) * S, plane = (size_t)p.B * N * S;
    const int tend = row_steps(p, b);
    float A2[K], h[K];
    load_states<K>(A2, p.A + (size_t)n * S, at.s0, S, true);
    load_states<K>(h, p.h0 + row, at.s0, S, p.h0 && at.on);
#pragma unroll
    for (int k = 0; k < K; ++k) A2[k] *= kLog2e;
    const float bias = p.dt_bias ? p.dt_bias[n] : 0.0f, D = p.D ? p.D[n] : 0.0f;
    const char *xp = column<E>(p.x, b, n), *dp = column<E>(p.dt, b, n), *gp = column<E>(p.g, b, n);
    E* yp = (E*)column<E>(p.y, b, n);

    Stage<E, SP> bcv;
    Own<E, Q> xv, dv, gv;
    auto load = [&](int t0) {
        bcv.load(p, b, t0, tend);
        dv.load(p.dt, dp, t0, j, tend, at.on);
        xv.load(p.x, xp, t0, j, tend, at.on);
        if (p.g.data) gv.load(p.g, gp, t0, j, tend, at.on);
    };
    if (tend > 0) load(0);
    int buf = 0;
    for (int t0 = 0; t0 < tend; t0 += kStepsB, buf ^= 1) {
        bcv.put(&bc[buf][0][0][0]);
        const Own<E, Q> x = xv, d = dv, g = gv;
        const uint32_t starts = start_bits(p, b, t0, tend, at.lane);
        barrier_lds();
        if (t0 + kStepsB < tend) load(t0 + kStepsB);
        if (p.states) store_states<K>(p.states + (size_t)(t0 / kStepsB) * plane + row, h, at.s0, S, at.on);
        auto walk = [&](auto masked) {
            each<Shape<Q>::own>([&](auto sub) {
                constexpr int c = decltype(sub)::value;
                const int t = t0 + c * Q + j;
                const bool valid = at.on && t < tend;
                float slope, ys[Q];
                const float xs = (float)x.v[c], delta = valid ? softplus((float)d.v[c] + bias, &slope) : 0.0f, u = delta * xs;
                each<Q>([&](auto step) {
                    constexpr int i = decltype(step)::value;
                    if (decltype(masked)::value && starts >> (c * Q + i) & 1)
#pragma unroll
                        for (int k = 0; k < K; ++k) h[k] = 0.0f;
                    const auto Bv = *(const Vec<float, K>*)&bc[buf][c * Q + i][0][at.s0];
                    const auto Cv = *(const Vec<float, K>*)&bc[buf][c * Q + i][1][at.s0];
                    const float di = from_lane<Q, i>(delta), ui = from_lane<Q, i>(u);
                    ys[i] = 0.0f;
#pragma unroll
                    for (int k = 0; k < K; ++k) {
                        h[k] = fmaf(__builtin_amdgcn_exp2f(di * A2[k]), h[k], ui * Bv.get(k));
                        ys[i] = fmaf(h[k], Cv.get(k), ys[i]);
                    }
                });
                float y = fmaf(D, xs, sums_by_lane<Q>(ys, j));
                if (p.g.data) {
                    const float gs = (float)g.v[c];
                    y *= gs * sigmoid(gs);
                }
                if (valid) yp[t * p.y.s0] = (E)y;
            });
        };
        starts ? walk(std::true_type()) : walk(std::false_type());
    }
    for (int t = tend + j; t < p.T; t += Q)
        if (at.on) yp[t * p.y.s0] = (E)0.0f;
    store_states<K>(p.h_last + row, h, at.s0, S, at.on);
}

template <class E, int Q, int K>
__global__ void __launch_bounds__(256) selective_bwd_kernel(Selective p) {
    constexpr int SP = Q * K, OWN = Shape<Q>::own;
    __shared__ __align__(16) float bc[2][kStepsB][2][SP];
    __shared__ __align__(16) float sums[kWavesWg][kStepsB][2][SP];
    const Place<Q, K> at(p);
    const int b = at.b, n = at.n, j = at.j, N = p.N, S = p.S;
    const size_t row = ((size_t)b * N + n) * S, plane = (size_t)p.B * N * S;
    const int tend = row_steps(p, b);
    float A2[K], kc[K], dA[K], dD = 0.0f, dbias = 0.0f;
    load_states<K>(A2, p.A + (size_t)n * S, at.s0, S, true);
    load_states<K>(kc, p.dlast + row, at.s0, S, p.dlast && at.on);
#pragma unroll
    for (int k = 0; k < K; ++k) A2[k] *= kLog2e, dA[k] = 0.0f;
    const float bias = p.dt_bias ? p.dt_bias[n] : 0.0f, D = p.D ? p.D[n] : 0.0f;
    const char *xp = column<E>(p.x, b, n), *dp = column<E>(p.dt, b, n), *gp = column<E>(p.g, b, n), *yp = column<E>(p.dy, b, n);
    E *dxp = (E*)column<E>(p.dx, b, n), *ddp = (E*)column<E>(p.ddt, b, n), *dgp = (E*)column<E>(p.dg, b, n);

    Stage<E, SP> bcv;
    Own<E, Q> xv, dv, gv, yv;
    auto load = [&](int t0) {
        bcv.load(p, b, t0, tend);
        dv.load(p.dt, dp, t0, j, tend, at.on);
        xv.load(p.x, xp, t0, j, tend, at.on);
        if (p.g.data) gv.load(p.g, gp, t0, j, tend, at.on);
        yv.load(p.dy, yp, t0, j, tend, at.on);
    };
    const int last = (tend - 1) / kStepsB * kStepsB;
    if (tend > 0) load(last);
    int buf = 0;
    for (int t0 = last; tend > 0 && t0 >= 0; t0 -= kStepsB, buf ^= 1) {
        bcv.put(&bc[buf][0][0][0]);
        const Own<E, Q> x = xv, d = dv, g = gv, dy = yv;
        const uint32_t starts = start_bits(p, b, t0, tend, at.lane);
        float h0[K];
        load_states<K>(h0, p.states + (size_t)(t0 / kStepsB) * plane + row, at.s0, S, at.on);
        barrier_lds();
        if (t0 >= kStepsB) load(t0 - kStepsB);
        auto walk = [&](auto masked) {
            constexpr bool MASK = decltype(masked)::value;
            float a[kStepsB][K], h[kStepsB][K], delta[OWN], slope[OWN], u[OWN], w[OWN], gate[OWN], gslope[OWN];
            each<OWN>([&](auto sub) {
                constexpr int c = decltype(sub)::value;
                const bool valid = at.on && t0 + c * Q + j < tend;
                delta[c] = softplus((float)d.v[c] + bias, &slope[c]);
                delta[c] = valid ? delta[c] : 0.0f;
                u[c] = delta[c] * (float)x.v[c];
                gate[c] = 1.0f;
                if (p.g.data) {
                    const float gs = (float)g.v[c], sg = sigmoid(gs);
                    gate[c] = gs * sg;
                    gslope[c] = fmaf(gate[c], 1.0f - sg, sg);
                }
                w[c] = (float)dy.v[c] * gate[c];
                each<Q>([&](auto step) {
                    constexpr int i = decltype(step)::value, s = c * Q + i;
                    const auto Bv = *(const Vec<float, K>*)&bc[buf][s][0][at.s0];
                    const float di = from_lane<Q, i>(delta[c]), ui = from_lane<Q, i>(u[c]);
#pragma unroll
                    for (int k = 0; k < K; ++k) {
                        const float before = MASK && (starts >> s & 1) ? 0.0f : s ? h[s ? s - 1 : 0][k] : h0[k];
                        a[s][k] = __builtin_amdgcn_exp2f(di * A2[k]);
                        h[s][k] = fmaf(a[s][k], before, ui * Bv.get(k));
                    }
                });
            });
            each_back<OWN>([&](auto sub) {
                constexpr int c = decltype(sub)::value;
                float ys[Q], lb[Q], aq[Q], left[Q][K / 2];
                each_back<Q>([&](auto step) {
                    constexpr int i = decltype(step)::value, s = c * Q + i;
                    const auto Bv = *(const Vec<float, K>*)&bc[buf][s][0][at.s0];
                    const auto Cv = *(const Vec<float, K>*)&bc[buf][s][1][at.s0];
                    const float di = from_lane<Q, i>(delta[c]), ui = from_lane<Q, i>(u[c]), wi = from_lane<Q, i>(w[c]);
                    const bool fresh = MASK && (starts >> s & 1);
                    float db[K], dc[K];
                    ys[i] = lb[i] = aq[i] = 0.0f;
#pragma unroll
                    for (int k = 0; k < K; ++k) {
                        const float before = fresh ? 0.0f : s ? h[s ? s - 1 : 0][k] : h0[k];
                        const float l = fmaf(wi, Cv.get(k), kc[k]);
                        ys[i] = fmaf(h[s][k], Cv.get(k), ys[i]);
                        lb[i] = fmaf(l, Bv.get(k), lb[i]);
                        db[k] = l * ui;
                        dc[k] = wi * h[s][k];
                        kc[k] = fresh ? 0.0f : a[s][k] * l;
                        const float q = kc[k] * before;
                        aq[i] = fmaf(A2[k], q, aq[i]);
                        dA[k] = fmaf(di, q, dA[k]);
                    }
                    // over the wave's rows of lanes: lanes below 32 go on with dB, the others with
                    // dC; odd rows with the upper half of the states
#pragma unroll
                    for (int k = 0; k < K; ++k) swap32(db[k], dc[k]), db[k] += dc[k];
#pragma unroll
                    for (int k = 0; k < K / 2; ++k) swap16(db[k], db[k + K / 2]), left[i][k] = db[k] + db[k + K / 2];
                });
                const int kind = at.lane >> 5, part = at.s0 + (at.lane >> 4 & 1) * (K / 2);
                if constexpr (Q == 4) {
                    // over the row's four groups of lanes, each of which writes a step
                    float mine[K / 2];
#pragma unroll
                    for (int k = 0; k < K / 2; ++k) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            left[i][k] = add_dpp<0x124>(left[i][k], left[i][k]);   // row_ror:4
                            left[i][k] = add_dpp<0x128>(left[i][k], left[i][k]);   // row_ror:8
                        }
                        const float lo = at.lane & 4 ? left[1][k] : left[0][k], hi = at.lane & 4 ? left[3][k] : left[2][k];
                        mine[k] = at.lane & 8 ? hi : lo;
                    }
                    vstore<float, K / 2>(&sums[at.w][c * 4 + (at.lane >> 2 & 3)][kind][part], mine);
                } else {
                    each<Q>([&](auto step) {
                        constexpr int i = decltype(step)::value;
                        vstore<float, K / 2>(&sums[at.w][i][kind][part], left[i]);
                    });
                }
                const int t = t0 + c * Q + j;
                const float xs = (float)x.v[c], core = fmaf(D, xs, sums_by_lane<Q>(ys, j));
                const float slb = sums_by_lane<Q>(lb, j), saq = sums_by_lane<Q>(aq, j);
                const float ddt = fmaf(saq, kLn2, xs * slb) * slope[c];
                if (at.on && t < tend) {
                    dD = fmaf(w[c], xs, dD);
                    dbias += ddt;
                    dxp[t * p.dx.s0] = (E)fmaf(delta[c], slb, D * w[c]);
                    ddp[t * p.ddt.s0] = (E)ddt;
                    if (p.g.data) dgp[t * p.dg.s0] = (E)((float)dy.v[c] * core * gslope[c]);
                }
            });
        };
        starts ? walk(std::true_type()) : walk(std::false_type());
        barrier_lds();
        // the waves' sums added up, to the workgroup's place in memory
        for (int e = threadIdx.x; e < kStepsB * 2 * SP; e += 256) {
            const int t = t0 + e / (2 * SP);
            const float* v = &sums[0][0][0][0] + e;
            constexpr int pitch = kStepsB * 2 * SP;
            if (t < tend) p.bcsums[(((size_t)at.tile * p.T + t) * p.B + b) * (2 * SP) + e % (2 * SP)] = (v[0] + v[pitch]) + (v[2 * pitch] + v[3 * pitch]);
        }
    }
    for (int t = tend + j; t < p.T; t += Q)
        if (at.on) {
            dxp[t * p.dx.s0] = (E)0.0f;
            ddp[t * p.ddt.s0] = (E)0.0f;
            if (p.g.data) dgp[t * p.dg.s0] = (E)0.0f;
        }
    if (p.dh0) store_states<K>(p.dh0 + row, kc, at.s0, S, at.on);
    float* rows = p.rowsums + (size_t)b * N * (S + 2);
    store_states<K>(rows + (size_t)n * S, dA, at.s0, S, at.on);
    dD = lanes_total<Q>(dD);
    dbias = lanes_total<Q>(dbias);
    if (at.on && j == 0) {
        rows[(size_t)N * S + n] = dD;
        rows[(size_t)N * (S + 1) + n] = dbias;
    }
}

// what the workgroups left: dB and dC over the tiles of channels (workgroups [0, wide)), dA, dD and
// the bias' over the rows
template <class E>
__global__ void __launch_bounds__(256) selective_sums_kernel(Selective p, int SP, unsigned wide, int rows) {
    if (blockIdx.x < wide) {
        const size_t steps = (size_t)p.T * p.B, all = steps * 2 * p.S;
        for (size_t e = blockIdx.x * 256ULL + threadIdx.x; e < all; e += wide * 256ULL) {
            const size_t r = e / (2 * p.S);
            const int c = (int)(e - r * (2 * p.S)), kind = c >= p.S, s = c - kind * p.S;
            const int t = (int)(r / p.B), b = (int)(r - (size_t)t * p.B);
            float v = 0.0f;
            if (t < row_steps(p, b))
                for (int q = 0; q < p.tiles; ++q) v += p.bcsums[(q * steps + r) * (2 * SP) + kind * SP + s];
            ((E*)(kind ? p.dC : p.dB))[r * p.S + s] = (E)v;
        }
        return;
    }
    const size_t all = (size_t)p.N * (p.S + 2);
    for (size_t e = (blockIdx.x - wide) * 256ULL + threadIdx.x; e < all; e += (gridDim.x - wide) * 256ULL) {
        float v = 0.0f;
        for (int q = 0; q < rows; ++q) v += p.rowsums[q * all + e];
        const size_t A = (size_t)p.N * p.S;
        float* out = e < A ? p.dA : e < A + p.N ? p.dD : p.dbias;
        if (out) out[e < A ? e : e < A + p.N ? e - A : e - A - p.N] = v;
    }
}

// one time step
template <class E, int Q, int K>
__global__ void __launch_bounds__(256) selective_step_kernel(Selective p) {
    const Place<Q, K> at(p);
    const int b = at.b, n = at.n, S = p.S;
    const size_t row = ((size_t)b * p.N + n) * S;
    float A[K], h[K], slope, y = 0.0f;
    load_states<K>(A, p.A + (size_t)n * S, at.s0, S, true);
    load_states<K>(h, p.h0 + row, at.s0, S, at.on);
    const float x = (float)*(const E*)column<E>(p.x, b, n);
    const float delta = softplus((float)*(const E*)column<E>(p.dt, b, n) + (p.dt_bias ? p.dt_bias[n] : 0.0f), &slope);
    const E *Bv = (const E*)p.Bm.data + b * p.Bm.s1, *Cv = (const E*)p.C.data + b * p.C.s1;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const bool in = at.s0 + k < S;
        h[k] = fmaf(__builtin_amdgcn_exp2f(delta * (A[k] * kLog2e)), h[k], in ? delta * x * (float)Bv[at.s0 + k] : 0.0f);
        y += in ? h[k] * (float)Cv[at.s0 + k] : 0.0f;
    }
    store_states<K>(p.h_last + row, h, at.s0, S, at.on);
    y = lanes_total<Q>(y);
    if (!at.on || at.j) return;
    if (p.D) y = fmaf(p.D[n], x, y);
    if (p.g.data) {
        const float g = (float)*(const E*)column<E>(p.g, b, n);
        y *= g * sigmoid(g);
    }
    *(E*)column<E>(p.y, b, n) = (E)y;
}

namespace {

struct Plan {
    int Q, K, tiles;
};
Plan selective_plan(int N, int S) {
    Plan q;
    q.Q = S <= 16 ? 4 : 16;
    q.K = S <= 8 || (S > 16 && S <= 32) ? 2 : 4;
    const int channels = 64 / q.Q * kWavesWg;
    q.tiles = (N + channels - 1) / channels;
    return q;
}

enum { kFwd, kBwd, kStep };

template <class E, int Q, int K>
void run_selective(Selective p, int what, hipStream_t stream) {
    const long long groups = (long long)p.B * p.tiles;
    for (long long first = 0; first < groups; first += kMostBlocks) {
        p.first = first;
        const dim3 grid((unsigned)std::min<long long>(groups - first, kMostBlocks)), block(64 * kWavesWg);
        if (what == kFwd) hipLaunchKernelGGL((selective_fwd_kernel<E, Q, K>), grid, block, 0, stream, p);
        else if (what == kBwd) hipLaunchKernelGGL((selective_bwd_kernel<E, Q, K>), grid, block, 0, stream, p);
        else hipLaunchKernelGGL((selective_step_kernel<E, Q, K>), grid, block, 0, stream, p);
    }
    if (what == kBwd) {
        const long long a = ((long long)p.T * p.B * 2 * p.S + 255) / 256, c = ((long long)p.N * (p.S + 2) + 255) / 256;
        const unsigned wide = (unsigned)std::min<long long>(a, 4096), rest = (unsigned)std::min<long long>(c, 4096);
        hipLaunchKernelGGL((selective_sums_kernel<E>), dim3(wide + rest), dim3(256), 0, stream, p, Q * K, wide, p.B);
    }
}

template <class E>
void run_selective_q(const Selective& p, const Plan& q, int what, hipStream_t stream) {
    if (q.Q == 4) q.K == 2 ? run_selective<E, 4, 2>(p, what, stream) : run_selective<E, 4, 4>(p, what, stream);
    else q.K == 2 ? run_selective<E, 16, 2>(p, what, stream) : run_selective<E, 16, 4>(p, what, stream);
}

void launch_selective(Selective p, int what, hipStream_t stream) {
    const Plan q = selective_plan(p.N, p.S);
    p.tiles = q.tiles;
    if (what == kBwd) {
        p.bcsums = p.ws;
        p.rowsums = p.ws + (size_t)q.tiles * p.T * p.B * 2 * q.Q * q.K;
    }
    if (p.bf16) run_selective_q<__bf16>(p, q, what, stream);
    else run_selective_q<float>(p, q, what, stream);
}

}  // namespace

size_t selective_fwd_ws(int, int, int, int) { return 0; }
size_t selective_bwd_ws(int T, int B, int N, int S) {
    const Plan q = selective_plan(N, S);
    return (size_t)q.tiles * T * B * 2 * q.Q * q.K + (size_t)B * N * (S + 2);
}
void launch_selective_fwd(const Selective& p, hipStream_t stream) { launch_selective(p, kFwd, stream); }
void launch_selective_bwd(const Selective& p, hipStream_t stream) { launch_selective(p, kBwd, stream); }
void launch_selective_step(const Selective& p, hipStream_t stream) { launch_selective(p, kStep, stream); }

}  // namespace delrec
