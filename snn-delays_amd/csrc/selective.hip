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
// The forward keeps the state before every 8th step in 32 bits (S / 2 bytes a value and step); the
// backward runs eight steps from there, holds their decays and states in registers and walks back (16
// steps took a second wave's registers: 397 us instead of 277 at the sizes below). The sums over
// channels (dB, dC) go through the wave's lanes, the workgroup's LDS and one set of sums for each
// workgroup of channels in memory, added up in a second launch in a fixed order, as dA, dD and the
// bias' over the rows.
//
// Bound by vector issue: forward 8.8 and backward 25.6 instructions a state and step, the exponential at
// less than half the rate, with the vector units busy 83 % of the time. At T250 B128 N512 S16 bf16 (262
// million states and steps) forward 87 us, with the kept states 100; backward 248 us, the sums 8. (The
// bytes take 26 and 65 us.) Exchanging lanes for dB and dC costs a sixth of the backward; as fp32
// matrix products with a selector, which do not run beside the vector instructions, they took it to
// 357 us, and through LDS to 272 (252 then).
#include <algorithm>
#include <utility>

#include "gated.h"
#include "kernels.h"

namespace delrec {

namespace {

constexpr int kStepsB = 16;                       // steps of a block
constexpr int kKept = DELREC_SELECTIVE_BLOCK;     // steps from one kept state to the next
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

// log(1 + e^x), and its slope. With e = e^-|x| and s = e / (2 + e) <= 1/3 it is max(x, 0) + 2 atanh(s), the
// series in s^2 by a polynomial (1.6e-8 relative): small values come in proportion to e, where log(1 + e)
// rounds them away. e itself is off by the exponent's roundings, 7.3e-8 |x| relative, and the rest by 4
// last places: within 5e-7 + 7.3e-8 |x| of itself.
__device__ __forceinline__ float softplus(float x, float* slope) {
    const float e = __builtin_amdgcn_exp2f(-fabsf(x) * kLog2e);
    const float s = e * __builtin_amdgcn_rcpf(2.0f + e), z = s * s;
    const float p = fmaf(fmaf(fmaf(0.13425749f, z, 0.1411831f), z, 0.2000378f), z, 0.3333332f);
    const float r = __builtin_amdgcn_rcpf(1.0f + e);
    *slope = x >= 0.0f ? r : e * r;
    return fmaxf(x, 0.0f) + 2.0f * fmaf(s * z, p, s);
}
__device__ __forceinline__ float sigmoid(float x) { return gate_in(-x); }

// a decay rate for powers of 2; infinite ones as the largest numbers, so that a step size of 0 (padding)
// still leaves the state as it is
__device__ __forceinline__ float rate2(float A) {
    const float r = A * kLog2e;
    return fabsf(r) == __builtin_inff() ? copysignf(3.402823466e38f, r) : r;
}

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
// A step's partial sums of a group's lanes, taken in until the lanes' own steps are complete: then each
// lane has its step's total. Four steps at a time are reduced over quads of lanes (16 lanes: the quads'
// sums over the row's four quads at the end), so that few registers wait.
template <int Q>
struct Sums {
    float v[4], quad[Q == 16 ? 4 : 1];
    template <int I>
    __device__ __forceinline__ void add(float x, int j) {
        v[I % 4] = x;
        if constexpr (Q == 16 && I % 4 == 0) {      // (steps come last first)
            hand_over<2, 0x4E>(v, j & 2);
            hand_over<1, 0xB1>(v, j & 1);
            quad[I / 4] = v[0];
        }
    }
    __device__ __forceinline__ float total(int j) {
        if constexpr (Q == 4) return sums_by_lane<4>(v, j);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            quad[i % (Q / 4)] = add_dpp<0x124>(quad[i % (Q / 4)], quad[i % (Q / 4)]);   // row_ror:4
            quad[i % (Q / 4)] = add_dpp<0x128>(quad[i % (Q / 4)], quad[i % (Q / 4)]);   // row_ror:8
        }
        const float lo = j & 4 ? quad[1 % (Q / 4)] : quad[0], hi = j & 4 ? quad[3 % (Q / 4)] : quad[2 % (Q / 4)];
        return j & 8 ? hi : lo;
    }
};
template <int Q>
__device__ __forceinline__ float lanes_total(float v) {
    return group_sum_t<Q>(v);
}

// halves of the wave exchanged: a keeps its lower and takes b's lower, b its upper and takes a's upper
__device__ __forceinline__ void swap32(float& a, float& b) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    a = __uint_as_float(r[0]);
    b = __uint_as_float(r[1]);
}
// the same with the odd rows of 16 lanes of a and the even ones of b
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

// the same past the caches: a step's states are next read in another step, after the rest of a model
template <int K>
__device__ __forceinline__ void stream_states(float* row, const float* v, int s0, int S, bool on) {
    if (on && s0 + K <= S) {
        typename Vec<float, K>::unaligned t;
#pragma unroll
        for (int k = 0; k < K; ++k) t[k] = v[k];
        __builtin_nontemporal_store(t, (typename Vec<float, K>::unaligned*)(row + s0));
    } else {
        store_states<K>(row, v, s0, S, on);
    }
}

// What stands before is finished before what stands after begins, and LDS is read again: the compiler
// otherwise keeps what it read once, and mixes the steps, until registers run out.
__device__ __forceinline__ void fence() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
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

template <class E>
__device__ __forceinline__ E* row_of(const delrec_rows& x, int b) { return (E*)x.data + b * x.s1; }

// bit i: a sequence starts at step t0 + i
__device__ __forceinline__ uint32_t start_bits(const Selective& p, int b, int t0, int tend, int lane) {
    const int t = t0 + lane;
    return (uint32_t)__ballot(lane < kStepsB && t < tend && p.starts[(size_t)min(t, p.T - 1) * p.B + b] != 0);
}

// B and C of a block of steps, from memory to LDS as fp32; zeros past the row's end and past S. A thread
// takes the same column of B or C in every `every`-th step.
template <class E, int SP>
struct Stage {
    static constexpr int count = kStepsB * 2 * SP, per = (count + 255) / 256, every = 256 / (2 * SP);
    E v[per];
    const E* at;                                            // the thread's first element of block t0
    long long pitch;
    int t, lds;
    bool in;
    __device__ __forceinline__ Stage(const Selective& p, int b, int t0) {
        const int tid = threadIdx.x, s = tid % SP;
        const delrec_rows& m = tid / SP % 2 ? p.C : p.Bm;
        t = tid / (2 * SP);
        lds = tid;
        in = s < p.S && t < kStepsB;
        pitch = m.s0;
        at = (const E*)m.data + (t0 + t) * pitch + b * m.s1 + s;
    }
    // block t0; then on to the next one, `move` steps away
    __device__ __forceinline__ void load(int t0, int tend, int move) {
#pragma unroll
        for (int r = 0; r < per; ++r) {
            v[r] = (E)0.0f;
            if (in && t0 + t + r * every < tend) v[r] = at[r * every * pitch];
        }
        at += move * pitch;
    }
    __device__ __forceinline__ void put(float* to) const {
#pragma unroll
        for (int r = 0; r < per; ++r)
            if (256 * per <= count || lds < count) to[lds + 256 * r] = (float)v[r];
    }
};

// A lane's place in one of the (T, B, N) tensors, moved from own step to own step: one addition an access
// and none in scalar registers.
template <class E, int Q, int DIR>
struct Column {
    E* at;
    long long move;
    // of own step t0 + i Q + j
    __device__ __forceinline__ Column(const delrec_rows& x, int b, int n, int t)
        : at((E*)x.data + t * x.s0 + b * x.s1 + n), move(DIR * Q * x.s0) {}
    __device__ __forceinline__ E* next() {
        E* r = at;
        at += move;
        return r;
    }
};
// COUNT own steps from t0 + j on, the last one first where DIR < 0; zeros past the row's end and in lanes
// without a channel
template <class E, int Q, int DIR, int COUNT = Shape<Q>::own>
struct Own {
    E v[COUNT];
    template <bool FULL>
    __device__ __forceinline__ void load(Column<E, Q, DIR>& x, int t0, int j, int tend, bool on) {
#pragma unroll
        for (int k = 0; k < COUNT; ++k) {
            const int i = DIR > 0 ? k : COUNT - 1 - k;
            const E* from = x.next();
            if (FULL) {
                v[i] = *from;
            } else {
                v[i] = (E)0.0f;
                if (on && t0 + i * Q + j < tend) v[i] = *from;
            }
        }
    }
};

// The states that ranges of time start from. A range's map is h -> exp(A sum d) h + L (and of the carry,
// backwards, the same with its own L); a start in it cuts off what comes before: sum d is then -1. The factor
// comes in two halves, which leave fp32 only where the product does and of which none is 0, and a state of 0
// needs none: as step by step it stays 0 however far its rate would grow it, and an infinite one infinite.
template <int K>
__device__ __forceinline__ void enter_range(float* h, const Selective& p, const float* A2, size_t row, size_t chan, int s0, bool on,
                                            int from, int dir, int count) {
    const size_t plane = (size_t)p.B * p.N * p.S;
    for (int q = 0; q < count; ++q) {
        const size_t r = from + dir * q;
        float L[K];
        load_states<K>(L, p.maps + r * plane + row, s0, p.S, on);
        const float sd = on ? p.mapsums[r * p.B * p.N + chan] : 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const float e = __builtin_amdgcn_exp2f(fmaxf(A2[k] * (0.5f * sd), -126.0f));
            // (without a step, or with steps of size 0, the state is as it was, whatever the rate)
            h[k] = sd == 0.0f ? h[k] + L[k] : sd < 0.0f || h[k] == 0.0f ? L[k] : fmaf(h[k] * e, e, L[k]);
        }
    }
}

// what a step needs of its own lane
struct Gate {
    float value, slope;
    __device__ __forceinline__ Gate(float g, bool has) {
        const float s = sigmoid(g), v = g * s;
        value = has ? v : 1.0f;
        slope = fmaf(v, 1.0f - s, s);
    }
};

}  // namespace

// A launch without ranges takes all steps; with them blockIdx.y is the range.
template <class E, int Q, int K, bool STARTS>
__global__ void __launch_bounds__(256) selective_fwd_kernel(Selective p) {
    constexpr int SP = Q * K, OWN = Shape<Q>::own;
    __shared__ __align__(16) float bc[2][kStepsB][2][SP];
    const Place<Q, K> at(p);
    const int b = at.b, n = at.n, j = at.j, S = p.S;
    const size_t chan = (size_t)b * p.N + n, row = chan * S, plane = (size_t)p.B * p.N * S;
    const int len = row_steps(p, b), ts = blockIdx.y * p.range, te = min(ts + p.range, p.T), tend = min(te, len);
    const bool whole = (at.tile + 1) * Shape<Q>::channels <= p.N, gated = p.g.data != nullptr;
    float A2[K], h[K];
    load_states<K>(A2, p.A + (size_t)n * S, at.s0, S, true);
    load_states<K>(h, p.h0 + row, at.s0, S, p.h0 && at.on);
#pragma unroll
    for (int k = 0; k < K; ++k) A2[k] = rate2(A2[k]);
    if (blockIdx.y) enter_range<K>(h, p, A2, row, chan, at.s0, at.on, 0, 1, blockIdx.y);
    const float bias = p.dt_bias ? p.dt_bias[n] : 0.0f, D = p.D ? p.D[n] : 0.0f;
    Column<E, Q, 1> xc(p.x, b, n, ts + j), dc(p.dt, b, n, ts + j), gc(gated ? p.g : p.x, b, n, ts + j), yc(p.y, b, n, ts + j);

    Stage<E, SP> bcv(p, b, ts);
    Own<E, Q, 1> xv, dv, gv;
    auto load = [&](int t0) {
        bcv.load(t0, tend, kStepsB);
        auto three = [&](auto full) {
            constexpr bool F = decltype(full)::value;
            dv.template load<F>(dc, t0, j, tend, at.on);
            xv.template load<F>(xc, t0, j, tend, at.on);
            gv.template load<F>(gc, t0, j, tend, at.on);
        };
        whole && t0 + kStepsB <= tend ? three(std::true_type()) : three(std::false_type());
    };
    if (ts < tend) load(ts);
    int buf = 0;
    for (int t0 = ts; t0 < tend; t0 += kStepsB, buf ^= 1) {
        bcv.put(&bc[buf][0][0][0]);
        const Own<E, Q, 1> x = xv, d = dv, g = gv;
        const uint32_t starts = STARTS ? start_bits(p, b, t0, tend, at.lane) : 0;
        barrier_lds();
        if (t0 + kStepsB < tend) load(t0 + kStepsB);
        auto keep = [&](int step) {
            if (p.states && t0 + step < tend)
                store_states<K>(p.states + (size_t)((t0 + step) / kKept) * plane + row, h, at.s0, S, at.on);
        };
        const bool full = whole && t0 + kStepsB <= tend;
        each<OWN>([&](auto sub) {
            constexpr int c = decltype(sub)::value;
            const bool valid = at.on && t0 + c * Q + j < tend;
            float slope, ys[Q];
            const float xs = (float)x.v[c], soft = softplus((float)d.v[c] + bias, &slope), delta = valid ? soft : 0.0f, u = delta * xs;
            each<Q>([&](auto step) {
                constexpr int i = decltype(step)::value, s = c * Q + i;
                if constexpr (s % kKept == 0) keep(s);
                if (STARTS && starts >> s & 1)
#pragma unroll
                    for (int k = 0; k < K; ++k) h[k] = 0.0f;
                const auto Bv = *(const Vec<float, K>*)&bc[buf][s][0][at.s0];
                const auto Cv = *(const Vec<float, K>*)&bc[buf][s][1][at.s0];
                const float di = from_lane<Q, i>(delta), ui = from_lane<Q, i>(u);
                ys[i] = 0.0f;
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    h[k] = fmaf(__builtin_amdgcn_exp2f(di * A2[k]), h[k], ui * Bv.get(k));
                    ys[i] = fmaf(h[k], Cv.get(k), ys[i]);
                }
            });
            const float y = fmaf(D, xs, sums_by_lane<Q>(ys, j)) * Gate((float)g.v[c], gated).value;
            E* to = yc.next();
            if (full || valid) *to = (E)y;
        });
    }
    for (int t = max(ts, tend) + j; t < te; t += Q)
        if (at.on) row_of<E>(p.y, b)[t * p.y.s0 + n] = (E)0.0f;
    if (te == p.T) store_states<K>(p.h_last + row, h, at.s0, S, at.on);
}

// A range's map into p.maps and p.mapsums, forwards (of the states) or backwards (of the carry).
template <class E, int Q, int K, bool STARTS, bool BWD>
__global__ void __launch_bounds__(256) selective_range_kernel(Selective p) {
    constexpr int SP = Q * K, OWN = Shape<Q>::own;
    __shared__ __align__(16) float bc[2][kStepsB][2][SP];
    const Place<Q, K> at(p);
    const int b = at.b, n = at.n, j = at.j, S = p.S;
    const int y = blockIdx.y + (BWD ? 1 : 0);          // the last range forward, the first backward lead nowhere
    const size_t chan = (size_t)b * p.N + n, row = chan * S, plane = (size_t)p.B * p.N * S;
    const int ts = y * p.range, te = min(ts + p.range, p.T), tend = min(te, row_steps(p, b));
    const bool whole = (at.tile + 1) * Shape<Q>::channels <= p.N, gated = p.g.data != nullptr;
    float A2[K], h[K], total = 0.0f;
    load_states<K>(A2, p.A + (size_t)n * S, at.s0, S, true);
#pragma unroll
    for (int k = 0; k < K; ++k) A2[k] = rate2(A2[k]), h[k] = 0.0f;
    const float bias = p.dt_bias ? p.dt_bias[n] : 0.0f;
    const delrec_rows& xr = BWD ? p.dy : p.x;
    constexpr int DIR = BWD ? -1 : 1;
    const int blocks = tend > ts ? (tend - ts + kStepsB - 1) / kStepsB : 0;
    auto first = [&](int i) { return ts + (BWD ? blocks - 1 - i : i) * kStepsB; };
    const int t1 = first(0) + j + (BWD ? (OWN - 1) * Q : 0);
    Column<E, Q, DIR> xc(xr, b, n, t1), dc(p.dt, b, n, t1), gc(gated ? p.g : xr, b, n, t1);
    Stage<E, SP> bcv(p, b, first(0));
    Own<E, Q, DIR> xv, dv, gv;
    auto load = [&](int t0) {
        bcv.load(t0, tend, DIR * kStepsB);
        auto all = [&](auto full) {
            constexpr bool F = decltype(full)::value;
            dv.template load<F>(dc, t0, j, tend, at.on);
            xv.template load<F>(xc, t0, j, tend, at.on);
            if constexpr (BWD) gv.template load<F>(gc, t0, j, tend, at.on);
        };
        whole && t0 + kStepsB <= tend ? all(std::true_type()) : all(std::false_type());
    };
    bool cut = false;
    int buf = 0;
    if (blocks) load(first(0));
    for (int i = 0; i < blocks; ++i, buf ^= 1) {
        const int t0 = first(i);
        bcv.put(&bc[buf][0][0][0]);
        const Own<E, Q, DIR> x = xv, d = dv, g = gv;
        const uint32_t starts = STARTS ? start_bits(p, b, t0, tend, at.lane) : 0;
        cut |= starts != 0;
        barrier_lds();
        if (i + 1 < blocks) load(first(i + 1));
        each<OWN>([&](auto sub) {
            constexpr int c = BWD ? OWN - 1 - decltype(sub)::value : decltype(sub)::value;
            const bool valid = at.on && t0 + c * Q + j < tend;
            float slope, soft = softplus((float)d.v[c] + bias, &slope);
            const float delta = valid ? soft : 0.0f;
            const float u = BWD ? (float)x.v[c] * Gate((float)g.v[c], gated).value : delta * (float)x.v[c];
            total += delta;
            each<Q>([&](auto step) {
                constexpr int k0 = decltype(step)::value, q = BWD ? Q - 1 - k0 : k0, s = c * Q + q;
                const bool fresh = STARTS && (starts >> s & 1);
                const auto Mv = *(const Vec<float, K>*)&bc[buf][s][BWD ? 1 : 0][at.s0];
                const float di = from_lane<Q, q>(delta), ui = from_lane<Q, q>(u);
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    const float a = __builtin_amdgcn_exp2f(di * A2[k]);
                    if constexpr (BWD) h[k] = fresh ? 0.0f : a * fmaf(ui, Mv.get(k), h[k]);
                    else h[k] = fmaf(a, fresh ? 0.0f : h[k], ui * Mv.get(k));
                }
            });
        });
    }
    store_states<K>(p.maps + y * plane + row, h, at.s0, S, at.on);
    total = lanes_total<Q>(total);
    if (at.on && j == 0) p.mapsums[(size_t)y * p.B * p.N + chan] = cut ? -1.0f : total;
}

// Two waves a SIMD, and three where 168 registers nearly do (S 17 to 32, T250 B64 N512: 250 us, 285 with two;
// S 8: 13 registers would not fit, 202 us instead of 172).
template <class E, int Q, int K, bool STARTS>
__global__ void __launch_bounds__(256, Q == 16 && K == 2 ? 3 : 2) selective_bwd_kernel(Selective p) {
    constexpr int SP = Q * K, OWN = Shape<Q>::own;
    constexpr int HALF = OWN > 1 ? OWN / 2 : 1;       // own steps of a kept state's eight
    __shared__ __align__(16) float bc[2][kStepsB][2][SP];
    __shared__ __align__(16) float sums[kWavesWg][kStepsB][2][SP];
    const Place<Q, K> at(p);
    const int b = at.b, n = at.n, j = at.j, N = p.N, S = p.S;
    const size_t chan = (size_t)b * N + n, row = chan * S, plane = (size_t)p.B * N * S;
    const int ts = blockIdx.y * p.range, te = min(ts + p.range, p.T), tend = min(te, row_steps(p, b));
    const bool whole = (at.tile + 1) * Shape<Q>::channels <= N, gated = p.g.data != nullptr;
    float A2[K], kc[K], dA[K], dD = 0.0f, dbias = 0.0f;
    load_states<K>(A2, p.A + (size_t)n * S, at.s0, S, true);
    load_states<K>(kc, p.dlast + row, at.s0, S, p.dlast && at.on);
#pragma unroll
    for (int k = 0; k < K; ++k) A2[k] = rate2(A2[k]), dA[k] = 0.0f;
    enter_range<K>(kc, p, A2, row, chan, at.s0, at.on, gridDim.y - 1, -1, gridDim.y - 1 - blockIdx.y);
    const float bias = p.dt_bias ? p.dt_bias[n] : 0.0f, D = p.D ? p.D[n] : 0.0f;
    const int last = ts + (tend > ts ? (tend - ts - 1) / kStepsB * kStepsB : 0), t1 = last + (OWN - 1) * Q + j;
    Column<E, Q, -1> xc(p.x, b, n, t1), dc(p.dt, b, n, t1), gc(gated ? p.g : p.x, b, n, t1), yc(p.dy, b, n, t1);
    Column<E, Q, -1> dxc(p.dx, b, n, t1), ddc(p.ddt, b, n, t1), dgc(gated ? p.dg : p.dx, b, n, t1);
    Stage<E, SP> bcv(p, b, last);
    // the own steps of the half block (Q 16: block) from t on, a half (block) ahead of their use
    Own<E, Q, -1, HALF> xv, dv, gv, yv;
    auto load = [&](int t) {
        auto four = [&](auto full) {
            constexpr bool F = decltype(full)::value;
            dv.template load<F>(dc, t, j, tend, at.on);
            xv.template load<F>(xc, t, j, tend, at.on);
            gv.template load<F>(gc, t, j, tend, at.on);
            yv.template load<F>(yc, t, j, tend, at.on);
        };
        whole && t + HALF * Q <= tend ? four(std::true_type()) : four(std::false_type());
    };
    // the state kept before step t, a half ahead of its use (0 where the eight steps are padding: an
    // infinite state times their step size of 0)
    float hn[K];
    auto fetch_kept = [&](int t) {
        load_states<K>(hn, p.states + (size_t)(t / kKept) * plane + row, at.s0, S, at.on && t < tend);
    };
    if (tend > ts) {
        fetch_kept(last + kKept);
        bcv.load(last, tend, -kStepsB);
        load(last + kStepsB - HALF * Q);
    }
    int buf = 0;
    for (int t0 = last; tend > ts && t0 >= ts; t0 -= kStepsB, buf ^= 1) {
        bcv.put(&bc[buf][0][0][0]);
        const uint32_t starts = STARTS ? start_bits(p, b, t0, tend, at.lane) : 0;
        const bool full = whole && t0 + kStepsB <= tend;
        barrier_lds();
        if (t0 > ts) bcv.load(t0 - kStepsB, tend, -kStepsB);
        // the values of a lane's own steps of half a block (Q 4), or of its one (Q 16)
        float delta[HALF], slope[HALF], u[HALF], w[HALF], ga[HALF], xs[HALF];
        Sums<Q> ys, lb, aq;
        each_back<2>([&](auto half) {
            constexpr int hf = decltype(half)::value, s0 = hf * kKept;
            float hk[K], a[kKept][K], h[kKept][K];
#pragma unroll
            for (int k = 0; k < K; ++k) hk[k] = hn[k];
            if (t0 + s0 > ts) fetch_kept(t0 + s0 - kKept);
            if constexpr (OWN > 1 || hf == 1) {
                each<HALF>([&](auto own) {
                    constexpr int o = decltype(own)::value, c = (OWN > 1 ? hf * HALF : 0) + o;
                    const bool valid = at.on && t0 + c * Q + j < tend;
                    const float soft = softplus((float)dv.v[o] + bias, &slope[o]);
                    delta[o] = valid ? soft : 0.0f;
                    xs[o] = (float)xv.v[o];
                    u[o] = delta[o] * xs[o];
                    const Gate gate((float)gv.v[o], gated);
                    w[o] = (float)yv.v[o] * gate.value;
                    ga[o] = (float)yv.v[o] * gate.slope;
                });
                constexpr int before = (OWN > 1 ? hf * kKept : 0) - HALF * Q;
                if (t0 + before >= ts) load(t0 + before);
            }
            each<kKept>([&](auto step) {
                constexpr int e = decltype(step)::value, s = s0 + e, o = OWN > 1 ? e / Q : 0, i = s % Q;
                const auto Bv = *(const Vec<float, K>*)&bc[buf][s][0][at.s0];
                const float di = from_lane<Q, i>(delta[o]), ui = from_lane<Q, i>(u[o]);
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    const float before = STARTS && (starts >> s & 1) ? 0.0f : e ? h[e ? e - 1 : 0][k] : hk[k];
                    a[e][k] = __builtin_amdgcn_exp2f(di * A2[k]);
                    h[e][k] = fmaf(a[e][k], before, ui * Bv.get(k));
                }
            });
            fence();
            float left[Q == 4 ? 4 : 1][K / 2];
            // B and C of a step, read a step ahead
            Vec<float, K> Bn, Cn;
            auto read_maps = [&](int s) {
                Bn = *(const Vec<float, K>*)&bc[buf][s][0][at.s0];
                Cn = *(const Vec<float, K>*)&bc[buf][s][1][at.s0];
            };
            read_maps(s0 + kKept - 1);
            each_back<kKept>([&](auto step) {
                constexpr int e = decltype(step)::value, s = s0 + e, o = OWN > 1 ? e / Q : 0, i = s % Q;
                const Vec<float, K> Bv = Bn, Cv = Cn;
                if constexpr (e > 0) read_maps(s - 1);
                const float di = from_lane<Q, i>(delta[o]), ui = from_lane<Q, i>(u[o]), wi = from_lane<Q, i>(w[o]);
                const bool fresh = STARTS && (starts >> s & 1);
                float ls[K], sy = 0.0f, sl = 0.0f, sq = 0.0f;
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    const float before = fresh ? 0.0f : e ? h[e ? e - 1 : 0][k] : hk[k];
                    ls[k] = fmaf(wi, Cv.get(k), kc[k]);
                    sy = fmaf(h[e][k], Cv.get(k), sy);
                    sl = fmaf(ls[k], Bv.get(k), sl);
                    kc[k] = fresh ? 0.0f : a[e][k] * ls[k];
                    const float q = kc[k] * before;
                    sq = fmaf(A2[k], q, sq);
                    dA[k] = fmaf(di, q, dA[k]);
                }
                ys.template add<i>(sy, j), lb.template add<i>(sl, j), aq.template add<i>(sq, j);
                // over the wave's rows of lanes: lanes below 32 go on with dB, the others with dC (their
                // factors change places, not the products); odd rows with the upper half of the states
                float us = ui, ws = wi, db[K];
                swap32(us, ws);
#pragma unroll
                for (int k = 0; k < K; ++k) swap32(ls[k], h[e][k]), db[k] = fmaf(us, ls[k], ws * h[e][k]);
                const int kind = at.lane >> 5, part = at.s0 + (at.lane >> 4 & 1) * (K / 2);
                constexpr int r = Q == 4 ? i : 0;
#pragma unroll
                for (int k = 0; k < K / 2; ++k) swap16(db[k], db[k + K / 2]), left[r][k] = db[k] + db[k + K / 2];
                if constexpr (Q == 16) {
                    vstore<float, K / 2>(&sums[at.w][s][kind][part], left[0]);
                } else if constexpr (i == 0) {
                    // over the row's four groups of lanes, each of which writes a step
                    float mine[K / 2];
#pragma unroll
                    for (int k = 0; k < K / 2; ++k) {
#pragma unroll
                        for (int v = 0; v < 4; ++v) {
                            left[v][k] = add_dpp<0x124>(left[v][k], left[v][k]);   // row_ror:4
                            left[v][k] = add_dpp<0x128>(left[v][k], left[v][k]);   // row_ror:8
                        }
                        const float lo = at.lane & 4 ? left[1][k] : left[0][k], hi = at.lane & 4 ? left[3][k] : left[2][k];
                        mine[k] = at.lane & 8 ? hi : lo;
                    }
                    vstore<float, K / 2>(&sums[at.w][s + (at.lane >> 2 & 3)][kind][part], mine);
                }
                fence();
                if constexpr (i == 0) {
                    constexpr int c = s / Q;
                    const float core = fmaf(D, xs[o], ys.total(j)), slb = lb.total(j), ddt = fmaf(aq.total(j), kLn2, xs[o] * slb) * slope[o];
                    E *dgp = dgc.next(), *dxp = dxc.next(), *ddp = ddc.next();
                    if (full || (at.on && t0 + c * Q + j < tend)) {
                        dD = fmaf(w[o], xs[o], dD);
                        dbias += ddt;
                        if (gated) *dgp = (E)(ga[o] * core);
                        *dxp = (E)fmaf(delta[o], slb, D * w[o]);
                        *ddp = (E)ddt;
                    }
                }
            });
        });
        barrier_lds();
        // the waves' sums added up, to the workgroup's place in memory
        for (int e = threadIdx.x; e < kStepsB * 2 * SP; e += 256) {
            const int t = t0 + e / (2 * SP);
            const float* v = &sums[0][0][0][0] + e;
            constexpr int pitch = kStepsB * 2 * SP;
            if (t < tend) p.bcsums[(((size_t)at.tile * p.T + t) * p.B + b) * (2 * SP) + e % (2 * SP)] = (v[0] + v[pitch]) + (v[2 * pitch] + v[3 * pitch]);
        }
    }
    for (int t = max(ts, tend) + j; t < te; t += Q)
        if (at.on) {
            if (gated) row_of<E>(p.dg, b)[t * p.dg.s0 + n] = (E)0.0f;
            row_of<E>(p.dx, b)[t * p.dx.s0 + n] = (E)0.0f;
            row_of<E>(p.ddt, b)[t * p.ddt.s0 + n] = (E)0.0f;
        }
    if (p.dh0 && blockIdx.y == 0) store_states<K>(p.dh0 + row, kc, at.s0, S, at.on);
    float* rows = p.rowsums + ((size_t)blockIdx.y * p.B + b) * N * (S + 2);
    store_states<K>(rows + (size_t)n * S, dA, at.s0, S, at.on);
    dD = lanes_total<Q>(dD);
    dbias = lanes_total<Q>(dbias);
    if (at.on && j == 0) {
        rows[(size_t)N * S + n] = dD;
        rows[(size_t)N * (S + 1) + n] = dbias;
    }
}

// What the workgroups left, added up in a fixed order: dB and dC over the tiles of channels (workgroups
// [0, wide), four columns a thread), and dA, dD and the bias' over the rows and ranges (64 columns a
// workgroup, the rows over its waves).
template <class E, int SP>
__global__ void __launch_bounds__(1024) selective_sums_kernel(Selective p, unsigned wide, unsigned rows) {
    if (blockIdx.x < wide) {
        constexpr int PER = 2 * SP / 4;
        const size_t steps = (size_t)p.T * p.B, all = steps * PER;
        for (size_t e = blockIdx.x * 1024ULL + threadIdx.x; e < all; e += wide * 1024ULL) {
            const size_t r = e / PER;
            const int c = (int)(e % PER) * 4, kind = c / SP, s = c % SP;
            bool on = true;
            if (p.lengths) {
                const unsigned t = (unsigned)r / (unsigned)p.B, b = (unsigned)r - t * (unsigned)p.B;
                on = (int)t < row_steps(p, b);
            }
            float v[4] = {};
            if (on) {
                const float* at = p.bcsums + r * (2 * SP) + c;
#pragma unroll 4
                for (int q = 0; q < p.tiles; ++q, at += steps * (2 * SP)) {
                    const auto x = vload<float, 4>(at);
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] += x.get(i);
                }
            }
            E* out = (E*)(kind ? p.dC : p.dB) + r * p.S + s;
            if (s + 4 <= p.S) {
                vstore<E, 4>(out, v);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (s + i < p.S) out[i] = (E)v[i];
            }
        }
        return;
    }
    __shared__ float red[16][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const size_t all = (size_t)p.N * (p.S + 2), A = (size_t)p.N * p.S;
    for (size_t c0 = (blockIdx.x - wide) * 64ULL; c0 < all; c0 += (gridDim.x - wide) * 64ULL) {
        const size_t c = c0 + lane;
        const float* at = p.rowsums + min(c, all - 1);
        float s4[4] = {};
        // four rows' loads in flight at a time (past the end the last row again, left out)
        for (unsigned r = w; r < rows; r += 64) {
            float v[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) v[q] = at[(size_t)min(r + 16 * q, rows - 1) * all];
#pragma unroll
            for (int q = 0; q < 4; ++q) s4[q] += r + 16 * q < rows ? v[q] : 0.0f;
        }
        red[w][lane] = (s4[0] + s4[1]) + (s4[2] + s4[3]);
        __syncthreads();
        if (w == 0 && c < all) {
            float v = red[0][lane];
            for (int q = 1; q < 16; ++q) v += red[q][lane];
            float* out = c < A ? p.dA : c < A + p.N ? p.dD : p.dbias;
            if (out) out[c < A ? c : c < A + p.N ? c - A : c - A - p.N] = v;
        }
        __syncthreads();
    }
}

// K of a row's S values from column s0 on, as fp32; 0 past S
template <class E, int K>
__device__ __forceinline__ void load_low(float* v, const E* row, int s0, int S) {
    if (s0 + K <= S) {
        const auto t = vload<E, K>(row + s0);
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = t.get(k);
    } else {
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = s0 + k < S ? (float)row[s0 + k] : 0.0f;
    }
}

// One time step of R rows (p.B of them counts rows, p.tiles workgroups of channels). Bound by the states'
// memory: a lane's states of R rows are under way together, and A is read once for them. What a channel
// needs once a row its lanes take in turn, a row each, as the scan's lanes their steps. All states are
// read before the first is written: they may be written where they were read. 29.5 us at B512 N2048 S16
// bf16 (134 MB of states, 4.6 TB/s); one row a lane, each with its own A, took 40. States stored past the
// caches: to a second buffer 34.8 us with the convolution's step instead of 45.8, and in place 28.0
// instead of 28.8 (B512), 9.4 instead of 10.4 (B64 N1024 S64, four layers), 15.6 instead of 15.3 (B256).
template <class E, int Q, int K, int R>
__global__ void __launch_bounds__(256) selective_step_kernel(Selective p) {
    const Place<Q, K> at(p);                      // (b counts groups of R rows)
    const int n = at.n, j = at.j, S = p.S, b0 = at.b * R;
    const size_t plane = (size_t)p.N * S, chan = (size_t)n * S;
    float A2[K], h[R][K], ys[Q];
    auto row_at = [&](int i) { return min(b0 + i, p.B - 1); };
#pragma unroll
    for (int i = 0; i < R; ++i) load_states<K>(h[i], p.h0 + row_at(i) * plane + chan, at.s0, S, at.on);
    load_states<K>(A2, p.A + chan, at.s0, S, true);
#pragma unroll
    for (int k = 0; k < K; ++k) A2[k] = rate2(A2[k]);
    const int mine = row_at(j % R);
    const float x = (float)row_of<E>(p.x, mine)[n];
    const Gate gate(p.g.data ? (float)row_of<E>(p.g, mine)[n] : 0.0f, p.g.data);
    float slope;
    const float delta = softplus((float)row_of<E>(p.dt, mine)[n] + (p.dt_bias ? p.dt_bias[n] : 0.0f), &slope), u = delta * x;
    each<R>([&](auto row) {
        constexpr int i = decltype(row)::value;
        float Bv[K], Cv[K];
        load_low<E, K>(Bv, row_of<E>(p.Bm, row_at(i)), at.s0, S);
        load_low<E, K>(Cv, row_of<E>(p.C, row_at(i)), at.s0, S);
        const float di = from_lane<Q, i>(delta), ui = from_lane<Q, i>(u);
        ys[i] = 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            h[i][k] = fmaf(__builtin_amdgcn_exp2f(di * A2[k]), h[i][k], ui * Bv[k]);
            ys[i] = fmaf(h[i][k], Cv[k], ys[i]);
        }
    });
#pragma unroll
    for (int i = R; i < Q; ++i) ys[i] = 0.0f;
    const float y = fmaf(p.D ? p.D[n] : 0.0f, x, sums_by_lane<Q>(ys, j)) * gate.value;
#pragma unroll
    for (int i = 0; i < R; ++i) stream_states<K>(p.h_last + row_at(i) * plane + chan, h[i], at.s0, S, at.on && b0 + i < p.B);
    if (at.on && j < R && b0 + j < p.B) row_of<E>(p.y, b0 + j)[n] = (E)y;
}

namespace {

struct Plan {
    int Q, K, tiles, range, ranges;
};
// Four lanes a channel up to 16 states, 16 lanes beyond (their sums over lanes cost more, but 16 states a
// lane would leave the backward no registers).
//
// Time over the grid where rows and channels give too few workgroups. A first launch over all ranges but
// one then composes the ranges' maps, without outputs, half to two thirds of a pass' work. A SIMD runs a
// vector instruction every ten cycles for one wave and every four for four, so that one workgroup a CU
// pays for it in the backward only (bf16, N 2048, S 16, T 1024; whole and in ranges, us: B 4 forward 128 and
// 74, backward 313 and 160; B 8 126 and 124, 320 and 290; B 12 171 and 178, 470 and 425; B 16 182 and
// 220, 475 and 535). Padded ranges end early and leave room for others: with masks more of them, and up
// to more workgroups (T1000 B50 N333 S8: forward 127 us whole, 86 with 12, 93 with 32; backward 290, 215
// with 8, 256 with 24; T300 B100 N512 S16, 800 workgroups: backward 224 and 203 with 3, forward 78 and
// 103). At least two blocks a range, at most 32 ranges (T2048 B1: backward 101 us with 32, 134 with 64,
// each of which composes the maps of those before it).
Plan selective_plan(int T, int B, int N, int S, bool fwd, bool mask) {
    Plan q;
    q.Q = S <= 16 ? 4 : 16;
    q.K = S <= 8 || (S > 16 && S <= 32) ? 2 : 4;
    const int channels = 64 / q.Q * kWavesWg;
    q.tiles = (N + channels - 1) / channels;
    const long long groups = (long long)B * q.tiles;
    const int blocks = (T + kStepsB - 1) / kStepsB, few = (fwd ? 256 : 512) * (mask ? 2 : 1);
    const int wanted = fwd ? (mask ? 4096 : 1024) : (mask ? 2400 : 1536);
    const int want = groups >= few ? 1 : std::max(1, std::min({(int)(wanted / groups), 32, blocks / 2}));
    const int per = (blocks + want - 1) / want;
    q.range = per * kStepsB;
    q.ranges = (blocks + per - 1) / per;
    return q;
}

enum { kFwd, kBwd, kStep };
constexpr int kStepRows = 4;

template <class E, int Q, int K, bool STARTS>
void run_selective(Selective p, const Plan& q, int what, hipStream_t stream) {
    const long long groups = (long long)(what == kStep ? (p.B + kStepRows - 1) / kStepRows : p.B) * p.tiles;
    for (int pass = what != kStep && q.ranges > 1 ? 0 : 1; pass < 2; ++pass)
        for (long long first = 0; first < groups; first += kMostBlocks) {
            p.first = first;
            const unsigned wgs = (unsigned)std::min<long long>(groups - first, kMostBlocks);
            const dim3 grid(wgs, q.ranges), inner(wgs, q.ranges - 1), block(64 * kWavesWg);
            if (what == kStep) hipLaunchKernelGGL((selective_step_kernel<E, Q, K, kStepRows>), dim3(wgs), block, 0, stream, p);
            else if (pass == 0 && what == kFwd) hipLaunchKernelGGL((selective_range_kernel<E, Q, K, STARTS, false>), inner, block, 0, stream, p);
            else if (pass == 0) hipLaunchKernelGGL((selective_range_kernel<E, Q, K, STARTS, true>), inner, block, 0, stream, p);
            else if (what == kFwd) hipLaunchKernelGGL((selective_fwd_kernel<E, Q, K, STARTS>), grid, block, 0, stream, p);
            else hipLaunchKernelGGL((selective_bwd_kernel<E, Q, K, STARTS>), grid, block, 0, stream, p);
        }
    if (what == kBwd) {
        const long long a = ((long long)p.T * p.B * (Q * K / 2) + 1023) / 1024, c = ((long long)p.N * (p.S + 2) + 63) / 64;
        const unsigned wide = (unsigned)std::min<long long>(a, 2048), rest = (unsigned)std::min<long long>(c, 8192);
        hipLaunchKernelGGL((selective_sums_kernel<E, Q * K>), dim3(wide + rest), dim3(1024), 0, stream, p, wide, (unsigned)q.ranges * p.B);
    }
}

template <class E, int Q, int K>
void run_selective_s(const Selective& p, const Plan& q, int what, hipStream_t stream) {
    p.starts ? run_selective<E, Q, K, true>(p, q, what, stream) : run_selective<E, Q, K, false>(p, q, what, stream);
}
template <class E>
void run_selective_q(const Selective& p, const Plan& q, int what, hipStream_t stream) {
    if (q.Q == 4) q.K == 2 ? run_selective_s<E, 4, 2>(p, q, what, stream) : run_selective_s<E, 4, 4>(p, q, what, stream);
    else q.K == 2 ? run_selective_s<E, 16, 2>(p, q, what, stream) : run_selective_s<E, 16, 4>(p, q, what, stream);
}

size_t map_floats(const Plan& q, int B, int N, int S) { return q.ranges > 1 ? (size_t)q.ranges * B * N * (S + 1) : 0; }

void launch_selective(Selective p, int what, hipStream_t stream) {
    const Plan q = selective_plan(p.T, p.B, p.N, p.S, what != kBwd, p.starts || p.lengths);
    p.tiles = q.tiles;
    p.range = q.range;
    float* ws = p.ws;
    if (what != kStep && q.ranges > 1) {
        p.maps = ws;
        p.mapsums = ws + (size_t)q.ranges * p.B * p.N * p.S;
        ws += map_floats(q, p.B, p.N, p.S);
    }
    if (what == kBwd) {
        p.bcsums = ws;
        p.rowsums = ws + (size_t)q.tiles * p.T * p.B * 2 * q.Q * q.K;
    }
    if (p.bf16) run_selective_q<__bf16>(p, q, what, stream);
    else run_selective_q<float>(p, q, what, stream);
}

}  // namespace

// floats of workspace, with and without masks
size_t selective_fwd_ws(int T, int B, int N, int S) {
    return std::max(map_floats(selective_plan(T, B, N, S, true, false), B, N, S), map_floats(selective_plan(T, B, N, S, true, true), B, N, S));
}
size_t selective_bwd_ws(int T, int B, int N, int S) {
    size_t n = 0;
    for (const bool mask : {false, true}) {
        const Plan q = selective_plan(T, B, N, S, false, mask);
        n = std::max(n, map_floats(q, B, N, S) + (size_t)q.tiles * T * B * 2 * q.Q * q.K + (size_t)q.ranges * B * N * (S + 2));
    }
    return n;
}
void launch_selective_fwd(const Selective& p, hipStream_t stream) { launch_selective(p, kFwd, stream); }
void launch_selective_bwd(const Selective& p, hipStream_t stream) { launch_selective(p, kBwd, stream); }
void launch_selective_step(const Selective& p, hipStream_t stream) { launch_selective(p, kStep, stream); }

}  // namespace delrec
