// Short causal convolution of each channel over time, with its activation, over (T, B, N) sequences:
//     p_t = bias + sum_i w_i x_{t-W+1+i} (i < W), y_t = p_t sigmoid(p_t) (or p_t).
// Steps before the first are the rows of `state` (B, W-1, N); a start cuts off what lies before it,
// a row's steps from its length on are padding. Backwards, with r_t = dy_t times the activation's
// slope at p_t: dx_s = sum_i w_i r_{s+W-1-i}, dw_i = sum_t r_t x_{t-W+1+i}, dbias = sum r.
//
// Bound by memory. A lane takes V neighbouring channels and a run of steps, and keeps the window of
// the last W inputs in registers: x is read once, but for the W - 1 steps before each run (from the
// cache). The backward computes p again from x and carries W unfinished dx along.
#include <algorithm>

#include "gated.h"
#include "kernels.h"

namespace delrec {

namespace {

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

// the lane's channels n .. n + have - 1 of row b, and its run's first step
struct Run {
    int b, n, have, t0, run;
    bool on;
    __device__ __forceinline__ Run(const CausalConv& p, int V) {
        const long long id = (p.first + blockIdx.x) * 256LL + threadIdx.x;
        const long long r = id / p.groups;
        n = (int)(id - r * p.groups) * V;
        run = (int)(r / p.B);
        b = (int)(r - (long long)run * p.B);
        t0 = run * p.steps;
        have = min(p.N - n, V);
        on = run < p.runs;
    }
};

// input row of step t (before the first step: of the state)
template <class E, int W, int V>
__device__ __forceinline__ void input_row(float* v, const CausalConv& p, const Run& r, int t) {
    if (t >= 0) {
        load_part<E, V>(v, (const E*)p.x.data + t * p.x.s0 + r.b * p.x.s1 + r.n, r.have);
    } else if (p.state) {
        load_part<E, V>(v, (const E*)p.state + ((size_t)r.b * (W - 1) + t + W - 1) * p.N + r.n, r.have);
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = 0.0f;
    }
}

__device__ __forceinline__ bool starts_at(const CausalConv& p, int b, int t) {
    return p.starts && t >= 0 && p.starts[(size_t)t * p.B + b] != 0;
}

template <int V, int W>
__device__ __forceinline__ void load_weights(float (&w)[W][V], float* bias, const CausalConv& p, const Run& r) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
        bias[j] = p.bias && j < r.have ? p.bias[r.n + j] : 0.0f;
#pragma unroll
        for (int i = 0; i < W; ++i) w[i][j] = j < r.have ? p.w[(size_t)(r.n + j) * W + i] : 0.0f;
    }
}

}  // namespace

template <class E, int V, int W>
__global__ void __launch_bounds__(256) conv_fwd_kernel(CausalConv p) {
    const Run r(p, V);
    if (!r.on) return;
    const int len = conv_steps(p, r.b), te = min(r.t0 + p.steps, p.T);
    float w[W][V], bias[V], x[W][V];
    load_weights<V, W>(w, bias, p, r);
    // x[i]: the row of step t - W + 1 + i, zero where a start cuts it off
#pragma unroll
    for (int i = 0; i < W - 1; ++i) {
        const int t = r.t0 - (W - 1) + i;
        if (starts_at(p, r.b, t) && t < len)
#pragma unroll
            for (int q = 0; q < i; ++q)
#pragma unroll
                for (int j = 0; j < V; ++j) x[q][j] = 0.0f;
        if (t < len) input_row<E, W, V>(x[i], p, r, t);
    }
    E* yp = (E*)p.y.data + r.b * p.y.s1 + r.n;
    for (int t = r.t0; t < te; ++t) {
        float y[V];
        if (t < len) {
            if (starts_at(p, r.b, t))
#pragma unroll
                for (int i = 0; i < W - 1; ++i)
#pragma unroll
                    for (int j = 0; j < V; ++j) x[i][j] = 0.0f;
            input_row<E, W, V>(x[W - 1], p, r, t);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                y[j] = bias[j];
#pragma unroll
                for (int i = 0; i < W; ++i) y[j] = fmaf(w[i][j], x[i][j], y[j]);
                if (p.silu) y[j] *= gate_in(-y[j]);
            }
#pragma unroll
            for (int i = 0; i < W - 1; ++i)
#pragma unroll
                for (int j = 0; j < V; ++j) x[i][j] = x[i + 1][j];
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) y[j] = 0.0f;
        }
        store_part<E, V>(yp + t * p.y.s0, y, r.have);
    }
    // the rows that the next call starts from: the window after the row's last step, by the lane
    // whose run holds it (the first run's for a row without steps)
    if (!p.state_out || (len > r.t0 ? len > te : !(r.t0 == 0))) return;
#pragma unroll
    for (int i = 0; i < W - 1; ++i) store_part<E, V>((E*)p.state_out + ((size_t)r.b * (W - 1) + i) * p.N + r.n, x[i], r.have);
}

template <class E, int V, int W>
__global__ void __launch_bounds__(256) conv_bwd_kernel(CausalConv p) {
    const Run r(p, V);
    if (!r.on) return;
    const int len = conv_steps(p, r.b), te = min(r.t0 + p.steps, p.T);
    float w[W][V], bias[V], x[W][V], dx[W][V], dw[W][V], db[V];
    load_weights<V, W>(w, bias, p, r);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        db[j] = 0.0f;
#pragma unroll
        for (int i = 0; i < W; ++i) x[i][j] = dx[i][j] = dw[i][j] = 0.0f;
    }
    // bit i: the row of step t - W + 1 + i is not cut off
    uint32_t joined = 0;
#pragma unroll
    for (int i = 0; i < W - 1; ++i) {
        const int t = r.t0 - (W - 1) + i;
        if (t < len) {
            if (starts_at(p, r.b, t)) {
                joined = 0;
#pragma unroll
                for (int q = 0; q < i; ++q)
#pragma unroll
                    for (int j = 0; j < V; ++j) x[q][j] = 0.0f;
            }
            input_row<E, W, V>(x[i], p, r, t);
            joined |= 1u << i;
        }
    }
    const E* dyp = (const E*)p.dy.data + r.b * p.dy.s1 + r.n;
    E* dxp = (E*)p.dx.data + r.b * p.dx.s1 + r.n;
    // the run's own steps, and W - 1 more that finish their gradients
    for (int t = r.t0; t < te + W - 1; ++t) {
        if (t < len) {
            if (starts_at(p, r.b, t)) {
                joined = 0;
#pragma unroll
                for (int i = 0; i < W - 1; ++i)
#pragma unroll
                    for (int j = 0; j < V; ++j) x[i][j] = 0.0f;
            }
            joined |= 1u << (W - 1);
            float dy[V];
            input_row<E, W, V>(x[W - 1], p, r, t);
            load_part<E, V>(dy, dyp + t * p.dy.s0, r.have);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                float pre = bias[j], d = dy[j];
#pragma unroll
                for (int i = 0; i < W; ++i) pre = fmaf(w[i][j], x[i][j], pre);
                if (p.silu) {
                    const float s = gate_in(-pre);
                    d *= fmaf(pre * s, 1.0f - s, s);
                }
                const float own = t < te ? d : 0.0f;
                db[j] += own;
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    dw[i][j] = fmaf(own, x[i][j], dw[i][j]);
                    dx[i][j] = fmaf(joined >> i & 1 ? w[i][j] : 0.0f, d, dx[i][j]);
                }
            }
        }
        // step s is finished
        const int s = t - (W - 1), k = s - (len - (W - 1));
        if (s >= r.t0 || r.t0 == 0) {
            if (p.dstate_out && k >= 0 && s < len && joined & 1) {
                float d[V];
                load_part<E, V>(d, (const E*)p.dstate_out + ((size_t)r.b * (W - 1) + k) * p.N + r.n, r.have);
#pragma unroll
                for (int j = 0; j < V; ++j) dx[0][j] += d[j];
            }
            if (s >= 0) store_part<E, V>(dxp + s * p.dx.s0, dx[0], r.have);
            else if (p.dstate) store_part<E, V>((E*)p.dstate + ((size_t)r.b * (W - 1) + s + W - 1) * p.N + r.n, dx[0], r.have);
        }
        joined >>= 1;
#pragma unroll
        for (int j = 0; j < V; ++j) {
#pragma unroll
            for (int i = 0; i < W - 1; ++i) x[i][j] = x[i + 1][j], dx[i][j] = dx[i + 1][j];
            dx[W - 1][j] = x[W - 1][j] = 0.0f;
        }
    }
    float* part = p.part + ((size_t)r.run * p.B + r.b) * p.N * (W + 1);
#pragma unroll
    for (int j = 0; j < V; ++j)
        if (j < r.have) {
#pragma unroll
            for (int i = 0; i < W; ++i) part[(size_t)(r.n + j) * W + i] = dw[i][j];
            part[(size_t)p.N * W + r.n + j] = db[j];
        }
}

// dw and dbias from the runs' sums: columns by 64, the runs over 16 waves
__global__ void __launch_bounds__(1024) conv_sums_kernel(const float* part, long long rows, long long cols, long long first, float* dw,
                                                         long long nw, float* db) {
    __shared__ float red[16][64];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const long long c = (first + blockIdx.x) * 64 + lane;
    float s = 0.0f;
    if (c < cols)
        for (long long r = wv; r < rows; r += 16) s += part[r * cols + c];
    red[wv][lane] = s;
    __syncthreads();
    if (wv || c >= cols) return;
    for (int q = 1; q < 16; ++q) s += red[q][lane];
    if (c < nw) dw[c] = s;
    else if (db) db[c - nw] = s;
}

namespace {

template <class E>
constexpr int kVec = 4;

int conv_run_steps(int T, int B, int N) {
    (void)B; (void)N;
    return std::min(T, 32);
}

template <class E, int W>
void run_conv(CausalConv p, bool fwd, hipStream_t stream) {
    constexpr int V = kVec<E>;
    p.groups = (p.N + V - 1) / V;
    p.steps = conv_run_steps(p.T, p.B, p.N);
    p.runs = (p.T + p.steps - 1) / p.steps;
    const long long blocks = ((long long)p.runs * p.B * p.groups + 255) / 256;
    for (p.first = 0; p.first < blocks; p.first += kMostBlocks) {
        const dim3 grid((unsigned)std::min<long long>(blocks - p.first, kMostBlocks));
        if (fwd) hipLaunchKernelGGL((conv_fwd_kernel<E, V, W>), grid, dim3(256), 0, stream, p);
        else hipLaunchKernelGGL((conv_bwd_kernel<E, V, W>), grid, dim3(256), 0, stream, p);
    }
    if (fwd) return;
    const long long cols = (long long)p.N * (W + 1), cblocks = (cols + 63) / 64;
    for (long long first = 0; first < cblocks; first += kMostBlocks)
        hipLaunchKernelGGL(conv_sums_kernel, dim3((unsigned)std::min<long long>(cblocks - first, kMostBlocks)), dim3(1024), 0, stream, p.part,
                           (long long)p.runs * p.B, cols, first, p.dw, (long long)p.N * W, p.db);
}

template <class E>
void run_conv_w(const CausalConv& p, bool fwd, hipStream_t stream) {
    switch (p.W) {
        case 2: return run_conv<E, 2>(p, fwd, stream);
        case 3: return run_conv<E, 3>(p, fwd, stream);
        case 4: return run_conv<E, 4>(p, fwd, stream);
        case 5: return run_conv<E, 5>(p, fwd, stream);
        case 6: return run_conv<E, 6>(p, fwd, stream);
        case 7: return run_conv<E, 7>(p, fwd, stream);
        default: return run_conv<E, 8>(p, fwd, stream);
    }
}

}  // namespace

size_t conv_bwd_ws(int T, int B, int N, int W) {
    const int steps = conv_run_steps(T, B, N);
    return (size_t)((T + steps - 1) / steps) * B * N * (W + 1);
}

void launch_conv(const CausalConv& p, bool fwd, hipStream_t stream) {
    if (p.bf16) run_conv_w<__bf16>(p, fwd, stream);
    else run_conv_w<float>(p, fwd, stream);
}

}  // namespace delrec
