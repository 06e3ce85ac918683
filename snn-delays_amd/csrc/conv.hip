// Short causal convolution of each channel over time, with its activation, over (T, B, N) sequences:
//     p_t = bias + sum_i w_i x_{t-W+1+i} (i < W), y_t = p_t sigmoid(p_t) (or p_t).
// Steps before the first are the rows of `state` (B, W-1, N); a start cuts off what lies before it,
// a row's steps from its length on are padding. Backwards, with r_t = dy_t times the activation's
// slope at p_t: dx_s = sum_i w_i r_{s+W-1-i}, dw_i = sum_t r_t x_{t-W+1+i}, dbias = sum r.
//
// Bound by memory. A lane takes V neighbouring channels and a run of steps, in blocks of U whose loads are
// under way together, and keeps the last W - 1 inputs in registers: x is read once, but for the W - 1
// steps before each run (from the cache). The backward computes p again from x and carries the last W - 1
// values of r along; the W - 1 steps after a run that its last dx need are computed twice. The sums of
// dw go over a lane's steps, then through LDS over the workgroup's runs of the same channels, then from
// memory over the workgroups, each in a fixed order. At T250 B128 N512 W4 bf16 forward 16 us (65 MB, 4.1
// TB/s) and backward 29 + 4 (98 MB, 3.4 TB/s; some 30 vector instructions a value come near the memory's
// time).
#include <algorithm>

#include "gated.h"
#include "kernels.h"

namespace delrec {

namespace {

constexpr int kVec = 4;          // channels of a lane
constexpr int kBlock = 4;        // steps of a block

__device__ __forceinline__ int conv_steps(const CausalConv& p, int b) {
    if (!p.lengths) return p.T;
    const int64_t v = p.lengths[b];
    return v < 0 ? 0 : (v < p.T ? (int)v : p.T);
}

// `have` of V channels (the last lane of a row may have fewer), the others 0
template <class E, int V>
__device__ __forceinline__ void load_part(float* v, const E* at, int have) {
    if (have == V) {
        const auto t = vload<E, V>(at);
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = t.get(j);
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = j < have ? (float)at[j] : 0.0f;
    }
}
template <class E, int V>
__device__ __forceinline__ void store_part(E* at, const float* v, int have) {
    if (have == V) {
        vstore<E, V>(at, v);
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (j < have) at[j] = (E)v[j];
    }
}

// the lane's channels n .. n + have - 1 of row b, and its run's steps t0 .. te - 1
struct Run {
    int b, n, have, t0, te, slot;
    bool on;
    long long tasks;                          // first run of the workgroup
    __device__ __forceinline__ Run(const CausalConv& p, int V) {
        const long long id = p.first + blockIdx.x;
        const long long tb = id / p.lane_blocks;
        const int lane = threadIdx.x & (p.lanes - 1);
        slot = threadIdx.x / p.lanes;
        tasks = tb * (256 / p.lanes);
        const long long task = tasks + slot;
        const int run = (int)(task / p.B);
        n = ((int)(id - tb * p.lane_blocks) * p.lanes + lane) * V;
        b = (int)(task - (long long)run * p.B);
        t0 = run * p.steps;
        te = min(t0 + p.steps, p.T);
        have = min(p.N - n, V);
        on = run < p.runs && have > 0;
    }
};

template <int V, int W>
__device__ __forceinline__ void load_weights(float (&w)[W][V], float* bias, const CausalConv& p, const Run& r) {
    if (r.have == V) {
        // V channels' weights lie together
        const float* at = p.w + (size_t)r.n * W;
#pragma unroll
        for (int q = 0; q < W; ++q) {
            const auto t = vload<float, V>(at + q * V);
#pragma unroll
            for (int e = 0; e < V; ++e) w[(q * V + e) % W][(q * V + e) / W] = t.get(e);
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
#pragma unroll
            for (int i = 0; i < W; ++i) w[i][j] = j < r.have ? p.w[(size_t)(r.n + j) * W + i] : 0.0f;
    }
    load_part<float, V>(bias, p.bias + r.n, p.bias ? r.have : 0);
}

// the state's row of step t < 0
template <class E, int W, int V>
__device__ __forceinline__ void state_row(float* v, const CausalConv& p, const Run& r, int t) {
    if (p.state) {
        load_part<E, V>(v, (const E*)p.state + ((size_t)r.b * (W - 1) + t + W - 1) * p.N + r.n, r.have);
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = 0.0f;
    }
}

// Steps of a (T, B, N) tensor as a lane reads them: rows t .. t + C - 1 below `end` (the others 0), fetched
// a block ahead of their use
template <class E, int V, int C>
struct Rows {
    Vec<E, V> v[C];
    __device__ __forceinline__ void fetch(const E* at, long long pitch, int t, int end, int have) {
        if (t >= end) {
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int j = 0; j < V; ++j) v[c].v[j] = (E)0.0f;
        } else if (t + C <= end && have == V) {
#pragma unroll
            for (int c = 0; c < C; ++c) v[c] = vload<E, V>(at + (t + c) * pitch);
        } else {
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int j = 0; j < V; ++j) v[c].v[j] = t + c < end && j < have ? at[(t + c) * pitch + j] : (E)0.0f;
        }
    }
    __device__ __forceinline__ void get(float (*x)[V]) const {
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int j = 0; j < V; ++j) x[c][j] = v[c].get(j);
    }
};

// rows t .. te - 1 of an output are padding
template <class E, int V>
__device__ __forceinline__ void clear_rows(E* at, long long pitch, int t, int te, int have) {
    const float none[V] = {};
    for (; t < te; ++t) store_part<E, V>(at + t * pitch, none, have);
}

// bit c: a sequence starts at step t + c, of those below `end`
template <int C>
__device__ __forceinline__ uint32_t start_bits(const CausalConv& p, int b, int t, int end) {
    uint32_t bits = 0;
#pragma unroll
    for (int c = 0; c < C; ++c)
        if (t + c >= 0 && t + c < end && p.starts[(size_t)(t + c) * p.B + b] != 0) bits |= 1u << c;
    return bits;
}
// whether step i of the bits' window and a step `ahead` of it are of one sequence: no start after i
__device__ __forceinline__ constexpr uint32_t between(int i, int ahead) { return ((1u << ahead) - 1u) << (i + 1); }

// the W - 1 steps before the run
template <class E, int V, int W>
__device__ __forceinline__ void load_before(float (*x)[V], const CausalConv& p, const Run& r, const E* xp, int len) {
#pragma unroll
    for (int i = 0; i < W - 1; ++i) {
        const int t = r.t0 - (W - 1) + i;
        if (t < 0) state_row<E, W, V>(x[i], p, r, t);
        else load_part<E, V>(x[i], xp + t * p.x.s0, t < len ? r.have : 0);
    }
}

}  // namespace

template <class E, int V, int W, bool STARTS>
__global__ void __launch_bounds__(256) conv_fwd_kernel(CausalConv p) {
    constexpr int U = kBlock;
    const Run r(p, V);
    if (!r.on) return;
    const int len = conv_steps(p, r.b), end = min(len, r.te);
    const E* xp = (const E*)p.x.data + r.b * p.x.s1 + r.n;
    E* yp = (E*)p.y.data + r.b * p.y.s1 + r.n;
    float w[W][V], bias[V], x[W - 1 + U][V];
    load_weights<V, W>(w, bias, p, r);
    load_before<E, V, W>(x, p, r, xp, len);
    uint32_t starts = STARTS ? start_bits<W - 1>(p, r.b, r.t0 - (W - 1), len) : 0;
    Rows<E, V, U> xn;
    xn.fetch(xp, p.x.s0, r.t0, end, r.have);
    int t = r.t0;
    for (; t < end; t += U) {
        xn.get(x + W - 1);
        xn.fetch(xp, p.x.s0, t + U, end, r.have);
        if (STARTS) starts |= start_bits<U>(p, r.b, t, end) << (W - 1);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float y[V];
#pragma unroll
            for (int j = 0; j < V; ++j) y[j] = bias[j];
#pragma unroll
            for (int i = 0; i < W; ++i) {
                const bool cut = STARTS && i < W - 1 && starts & between(u + i, W - 1 - i);
#pragma unroll
                for (int j = 0; j < V; ++j) y[j] = fmaf(w[i][j], cut ? 0.0f : x[u + i][j], y[j]);
            }
#pragma unroll
            for (int j = 0; j < V; ++j) {
                if (p.silu) y[j] *= gate_in(-y[j]);
                if (t + u >= end) y[j] = 0.0f;
            }
            if (t + u < r.te) store_part<E, V>(yp + (t + u) * p.y.s0, y, r.have);
        }
#pragma unroll
        for (int i = 0; i < W - 1; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) x[i][j] = x[U + i][j];
        starts >>= U;
    }
    clear_rows<E, V>(yp, p.y.s0, t, r.te, r.have);
    // The rows that the next call starts from, by the first run's lanes. All are read before the first is
    // written: with one step they may lie where the state does.
    if (!p.state_out || r.t0) return;
    const uint32_t ends = STARTS ? start_bits<W - 1>(p, r.b, len - (W - 1), len) : 0;
#pragma unroll
    for (int i = 0; i < W - 1; ++i) {
        const int t = len - (W - 1) + i;
        if (t < 0) state_row<E, W, V>(x[i], p, r, t);
        else load_part<E, V>(x[i], xp + t * p.x.s0, r.have);
        if (STARTS && i < W - 2 && ends & between(i, W - 2 - i))
#pragma unroll
            for (int j = 0; j < V; ++j) x[i][j] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < W - 1; ++i) store_part<E, V>((E*)p.state_out + ((size_t)r.b * (W - 1) + i) * p.N + r.n, x[i], r.have);
}

// (with the tests for starts there are no registers left to fetch a block ahead: 64 us instead of 44 for
// T1000 B50 N333 W3 fp32)
template <class E, int V, int W, bool STARTS>
__global__ void __launch_bounds__(256) conv_bwd_kernel(CausalConv p) {
    constexpr int U = kBlock;
    constexpr bool AHEAD = !STARTS;
    __shared__ float red[256][V * (W + 1) + 1];
    const Run r(p, V);
    const int len = r.on ? conv_steps(p, r.b) : 0;
    float dw[W][V], db[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        db[j] = 0.0f;
#pragma unroll
        for (int i = 0; i < W; ++i) dw[i][j] = 0.0f;
    }
    if (r.on) {
        const E* xp = (const E*)p.x.data + r.b * p.x.s1 + r.n;
        const E* dyp = (const E*)p.dy.data + r.b * p.dy.s1 + r.n;
        E* dxp = (E*)p.dx.data + r.b * p.dx.s1 + r.n;
        float w[W][V], bias[V], x[W - 1 + U][V], d[W - 1 + U][V];
        load_weights<V, W>(w, bias, p, r);
        load_before<E, V, W>(x, p, r, xp, len);
#pragma unroll
        for (int i = 0; i < W - 1; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) d[i][j] = 0.0f;
        uint32_t starts = STARTS ? start_bits<W - 1>(p, r.b, r.t0 - (W - 1), len) : 0;
        const int end = min(len, r.te + W - 1);
        // the run's own steps, and W - 1 more that finish their gradients; row i of the windows is step
        // t - (W - 1) + i
        Rows<E, V, U> xn, dn;
        auto fetch = [&](int t) {
            xn.fetch(xp, p.x.s0, t, end, r.have);
            dn.fetch(dyp, p.dy.s0, t, end, r.have);
        };
        if (AHEAD) fetch(r.t0);
        // (past the last step that is no padding, W - 1 more finish what it began)
        const int stop = r.te + W - 1, live = min(stop, max(end, r.t0) + W - 1);
        int t = r.t0;
        for (; t < live; t += U) {
            if (!AHEAD) fetch(t);
            xn.get(x + W - 1);
            dn.get(d + W - 1);
            if (AHEAD) fetch(t + U);
            if (STARTS) starts |= start_bits<U>(p, r.b, t, end) << (W - 1);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float pre[V], own[V];
#pragma unroll
                for (int j = 0; j < V; ++j) pre[j] = bias[j];
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    const bool cut = STARTS && i < W - 1 && starts & between(u + i, W - 1 - i);
#pragma unroll
                    for (int j = 0; j < V; ++j) pre[j] = fmaf(w[i][j], cut ? 0.0f : x[u + i][j], pre[j]);
                }
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    float g = d[W - 1 + u][j];
                    if (p.silu) {
                        const float s = gate_in(-pre[j]);
                        g *= fmaf(pre[j] * s, 1.0f - s, s);
                    }
                    // (nothing comes of a padded step, whatever the weights)
                    g = t + u < end ? g : 0.0f;
                    d[W - 1 + u][j] = g;
                    own[j] = t + u < r.te ? g : 0.0f;
                    db[j] += own[j];
                }
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    const bool cut = STARTS && i < W - 1 && starts & between(u + i, W - 1 - i);
#pragma unroll
                    for (int j = 0; j < V; ++j) dw[i][j] = fmaf(own[j], cut ? 0.0f : x[u + i][j], dw[i][j]);
                }
            }
            // steps t - (W - 1) .. t + U - W are finished
#pragma unroll
            for (int q = 0; q < U; ++q) {
                const int s = t - (W - 1) + q, k = s - (len - (W - 1));
                if (s < r.te && (s >= r.t0 || r.t0 == 0)) {
                    float g[V];
#pragma unroll
                    for (int j = 0; j < V; ++j) g[j] = w[W - 1][j] * d[q][j];
#pragma unroll
                    for (int m = 1; m < W; ++m) {
                        const bool cut = STARTS && starts & between(q, m);
#pragma unroll
                        for (int j = 0; j < V; ++j) g[j] = fmaf(w[W - 1 - m][j], cut ? 0.0f : d[q + m][j], g[j]);
                    }
                    if (p.dstate_out && k >= 0 && s < len && !(STARTS && starts & between(q, W - 1))) {
                        float more[V];
                        load_part<E, V>(more, (const E*)p.dstate_out + ((size_t)r.b * (W - 1) + k) * p.N + r.n, r.have);
#pragma unroll
                        for (int j = 0; j < V; ++j) g[j] += more[j];
                    }
#pragma unroll
                    for (int j = 0; j < V; ++j) g[j] = s < len ? g[j] : 0.0f;      // (infinite weights times 0)
                    if (s >= 0) store_part<E, V>(dxp + s * p.dx.s0, g, r.have);
                    else if (p.dstate) store_part<E, V>((E*)p.dstate + ((size_t)r.b * (W - 1) + s + W - 1) * p.N + r.n, g, r.have);
                }
            }
#pragma unroll
            for (int i = 0; i < W - 1; ++i)
#pragma unroll
                for (int j = 0; j < V; ++j) x[i][j] = x[U + i][j], d[i][j] = d[U + i][j];
            starts >>= U;
        }
        clear_rows<E, V>(dxp, p.dx.s0, max(t - (W - 1), 0), r.te, r.have);
    }
    // over the workgroup's runs: of channel c the values c (W + 1) .. are those of its dw, then its db
#pragma unroll
    for (int j = 0; j < V; ++j) {
#pragma unroll
        for (int i = 0; i < W; ++i) red[threadIdx.x][j * (W + 1) + i] = dw[i][j];
        red[threadIdx.x][j * (W + 1) + W] = db[j];
    }
    __syncthreads();
    const int values = p.lanes * V * (W + 1), runs = 256 / p.lanes;
    const long long block = p.first + blockIdx.x, tb = block / p.lane_blocks;
    const int n0 = (int)(block - tb * p.lane_blocks) * p.lanes * V;
    float* part = p.part + (size_t)tb * p.N * (W + 1);
    for (int v = threadIdx.x; v < values; v += 256) {
        const int lane = v / (V * (W + 1)), e = v % (V * (W + 1)), n = n0 + lane * V + e / (W + 1), i = e % (W + 1);
        float s = 0.0f;
        for (int q = 0; q < runs; ++q) s += red[q * p.lanes + lane][e];
        if (n < p.N) part[i < W ? (size_t)n * W + i : (size_t)p.N * W + n] = s;
    }
}

// one time step without masks; the state's rows are read before the first is written
template <class E, int V, int W>
__global__ void __launch_bounds__(256) conv_step_kernel(CausalConv p) {
    const Run r(p, V);
    if (!r.on) return;
    float w[W][V], bias[V], x[W][V], y[V];
#pragma unroll
    for (int i = 0; i < W - 1; ++i) state_row<E, W, V>(x[i], p, r, i - (W - 1));
    load_part<E, V>(x[W - 1], (const E*)p.x.data + r.b * p.x.s1 + r.n, r.have);
    load_weights<V, W>(w, bias, p, r);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        y[j] = bias[j];
#pragma unroll
        for (int i = 0; i < W; ++i) y[j] = fmaf(w[i][j], x[i][j], y[j]);
        if (p.silu) y[j] *= gate_in(-y[j]);
    }
    store_part<E, V>((E*)p.y.data + r.b * p.y.s1 + r.n, y, r.have);
    if (!p.state_out) return;
#pragma unroll
    for (int i = 0; i < W - 1; ++i) store_part<E, V>((E*)p.state_out + ((size_t)r.b * (W - 1) + i) * p.N + r.n, x[i + 1], r.have);
}

// dw and dbias from the workgroups' sums: columns by 64, the workgroups over 16 waves
__global__ void __launch_bounds__(1024) conv_sums_kernel(const float* part, unsigned rows, long long cols, long long first, float* dw,
                                                         long long nw, float* db) {
    __shared__ float red[16][64];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const long long c = (first + blockIdx.x) * 64 + lane;
    const float* at = part + min(c, cols - 1);
    float s4[4] = {};
    // four rows' loads in flight at a time (past the end the last row again, left out)
    for (unsigned r = wv; r < rows; r += 64) {
        float v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = at[(size_t)min(r + 16 * q, rows - 1) * cols];
#pragma unroll
        for (int q = 0; q < 4; ++q) s4[q] += r + 16 * q < rows ? v[q] : 0.0f;
    }
    float s = (s4[0] + s4[1]) + (s4[2] + s4[3]);
    red[wv][lane] = s;
    __syncthreads();
    if (wv || c >= cols) return;
    for (int q = 1; q < 16; ++q) s += red[q][lane];
    if (c < nw) dw[c] = s;
    else if (db) db[c - nw] = s;
}

namespace {

struct Plan {
    int lanes, lane_blocks, steps, runs;
    long long task_blocks;
};
// 32 lanes of neighbouring channels, fewer where a row has fewer. Forward runs of 16 steps (T250 B128 N512
// bf16 W4 16.0 us, 17.8 with 32, 24.5 with 64; T1000 B50 N333 with masks 26, 33 and 53). Backward runs
// take whole blocks with the W - 1 steps past their end, as many as make the least work for the CU that
// has the most workgroups (32 steps and this many, us: the first case 32.4 and 29.0, T8192 B1 N2048 32.4
// and 31.0, T1000 B16 N1024 W8 55 and 41, fp32 W4 49 and 45). With masks some runs end early, and up to
// 32 steps are better (T1000 B50 N333 W3 50 us with 40 steps, 45 with 32).
Plan conv_plan(int T, int B, int N, int W, bool fwd, bool mask) {
    Plan best{};
    const int groups = (N + kVec - 1) / kVec;
    best.lanes = 1;
    while (best.lanes < 32 && best.lanes < groups) best.lanes *= 2;
    best.lane_blocks = (groups + best.lanes - 1) / best.lanes;
    const int per = 256 / best.lanes;
    double least = 0.0;
    for (int m = 4; m <= (mask ? 8 : 16); ++m) {
        Plan q = best;
        q.steps = std::min(T, m * kBlock - (fwd ? 0 : W - 1));
        q.runs = (T + q.steps - 1) / q.steps;
        q.task_blocks = ((long long)q.runs * B + per - 1) / per;
        const double work = (double)((q.task_blocks * q.lane_blocks + 255) / 256) * (m * kBlock);
        if (m == 4 || work < least) best = q, least = work;
        if (fwd || q.steps == T) break;
    }
    return best;
}

template <class E, int W, bool STARTS>
void run_conv(CausalConv p, bool fwd, hipStream_t stream) {
    const Plan q = conv_plan(p.T, p.B, p.N, W, fwd, p.starts || p.lengths);
    p.lanes = q.lanes;
    p.lane_blocks = q.lane_blocks;
    p.steps = q.steps;
    p.runs = q.runs;
    const long long blocks = q.task_blocks * q.lane_blocks;
    for (p.first = 0; p.first < blocks; p.first += kMostBlocks) {
        const dim3 grid((unsigned)std::min<long long>(blocks - p.first, kMostBlocks));
        if (fwd && p.T == 1 && !p.starts && !p.lengths) hipLaunchKernelGGL((conv_step_kernel<E, kVec, W>), grid, dim3(256), 0, stream, p);
        else if (fwd) hipLaunchKernelGGL((conv_fwd_kernel<E, kVec, W, STARTS>), grid, dim3(256), 0, stream, p);
        else hipLaunchKernelGGL((conv_bwd_kernel<E, kVec, W, STARTS>), grid, dim3(256), 0, stream, p);
    }
    if (fwd) return;
    const long long cols = (long long)p.N * (W + 1), cblocks = (cols + 63) / 64;
    for (long long first = 0; first < cblocks; first += kMostBlocks)
        hipLaunchKernelGGL(conv_sums_kernel, dim3((unsigned)std::min<long long>(cblocks - first, kMostBlocks)), dim3(1024), 0, stream, p.part,
                           (unsigned)q.task_blocks, cols, first, p.dw, (long long)p.N * W, p.db);
}

template <class E, int W>
void run_conv_s(const CausalConv& p, bool fwd, hipStream_t stream) {
    p.starts ? run_conv<E, W, true>(p, fwd, stream) : run_conv<E, W, false>(p, fwd, stream);
}

template <class E>
void run_conv_w(const CausalConv& p, bool fwd, hipStream_t stream) {
    switch (p.W) {
        case 2: return run_conv_s<E, 2>(p, fwd, stream);
        case 3: return run_conv_s<E, 3>(p, fwd, stream);
        case 4: return run_conv_s<E, 4>(p, fwd, stream);
        case 5: return run_conv_s<E, 5>(p, fwd, stream);
        case 6: return run_conv_s<E, 6>(p, fwd, stream);
        case 7: return run_conv_s<E, 7>(p, fwd, stream);
        default: return run_conv_s<E, 8>(p, fwd, stream);
    }
}

}  // namespace

size_t conv_bwd_ws(int T, int B, int N, int W) {
    return (size_t)std::max(conv_plan(T, B, N, W, false, false).task_blocks, conv_plan(T, B, N, W, false, true).task_blocks) * N * (W + 1);
}

void launch_conv(const CausalConv& p, bool fwd, hipStream_t stream) {
    if (p.bf16) run_conv_w<__bf16>(p, fwd, stream);
    else run_conv_w<float>(p, fwd, stream);
}

}  // namespace delrec
