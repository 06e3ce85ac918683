// Gated linear recurrence over (T, B, N) sequences and its reverse pass.
//     k_t = sigmoid(-(f_t + bias)), h_t = h_{t-1} + k_t (z_t - h_{t-1})
// backwards, with lam_t = dh_t + c_{t+1} and c_t = (1 - k_t) lam_t (c_T = dlast):
//     dz_t = lam_t k_t, df_t = lam_t k_t (1 - k_t) (h_{t-1} - z_t), dh0 = c_0, db = sum df.
// Both are affine in what they carry, h -> A h + S and c -> A c + S with A the product of the
// leaks 1 - k, and affine maps compose: time is cut into pieces that run side by side.
//
// A workgroup takes 64 V channels (V consecutive ones a lane) and walks time in blocks of 64
// steps, eight per wave: each wave loads its steps, composes them from nothing into (A, S), the
// waves exchange these through LDS (one barrier a block, two buffers), every wave composes those
// before it onto the block's state, and runs its steps again from there, out of registers. So z
// and f are read once and h is written once, whatever T. With too few channels to fill the GPU
// time is cut a second time, over the grid: a first launch composes each range (reading its
// inputs once more), the second starts from the composition of the ranges before it.
//
// The forward keeps the state before every 64th step in 32 bits (1/16 byte a value and step); the
// backward starts its blocks there and recomputes the states between from z and f, which it needs
// anyway: exact in 32 bits where reading h back would bring its bf16 rounding into df, and two to
// four bytes a value less to read.
#include <algorithm>

#include "gated.h"
#include "kernels.h"

namespace delrec {

namespace {

constexpr int kBlk = DELREC_GATED_BLOCK;
constexpr int kSteps = 8;                    // steps of a wave in a block
constexpr int kWaves = kBlk / kSteps;

// A start inside a piece cuts what comes before it off, also where that is infinite: A = -1 says
// so (products of leaks are never negative). Only the masked forms have it.
template <bool MASK>
__device__ __forceinline__ float apply(float A, float S, float h) {
    if (MASK && A < 0.0f) return S;
    return fmaf(A, h, S);
}
template <bool MASK>
__device__ __forceinline__ float product(float A, float B) {
    if (MASK && (A < 0.0f || B < 0.0f)) return -1.0f;
    return A * B;
}

__device__ __forceinline__ int row_length(const GatedScan& p, int b) {
    if (!p.lengths) return p.T;
    const int64_t v = p.lengths[b];
    return v < 0 ? 0 : (v < p.T ? (int)v : p.T);
}

// the lane's channels: row b, columns n0 .. n0 + V - 1. The last lane of a row whose width is no
// multiple of V is moved back to end with it and repeats `skip` columns of the lane before (the
// same values, written twice). Lanes past the last row, and with 8-bit groups the lanes that fill
// a row's last group up, repeat valid columns and write nothing.
template <int V>
struct Lane {
    int b, n0, skip, group;                  // group: of its first own column
    bool on, first;                          // writes; first lane of its 8-bit group
    __device__ __forceinline__ Lane(const GatedScan& p, int per_row) {
        const long long c = (long long)blockIdx.x * 64 + (threadIdx.x & 63);
        const long long rows = c / per_row;
        b = rows < p.B ? (int)rows : p.B - 1;
        const int i = (int)(c - rows * per_row) * V;
        on = rows < p.B && i < p.N;
        first = on && i % kGroup8 == 0;
        n0 = i < p.N - V ? i : p.N - V;
        skip = on ? i - n0 : V;
        group = i / kGroup8;
    }
};

// the exchange: wave w's maps for the block, in LDS
template <int V>
struct Maps {
    float A[2][kWaves][64 * V], S[2][kWaves][64 * V];
    __device__ __forceinline__ void put(int buf, int w, int lane, const float* a, const float* s) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            A[buf][w][lane * V + j] = a[j];
            S[buf][w][lane * V + j] = s[j];
        }
    }
    template <bool MASK>
    __device__ __forceinline__ void run(int buf, int w, int lane, float* h) const {
#pragma unroll
        for (int j = 0; j < V; ++j) h[j] = apply<MASK>(A[buf][w][lane * V + j], S[buf][w][lane * V + j], h[j]);
    }
};

// The state that a range starts from: the maps of the ranges `from`, from + dir, .. (count of
// them) composed onto h by all waves together, through the exchange's first buffer.
template <int V, bool MASK>
__device__ __forceinline__ void enter_range(Maps<V>& m, const float* agg, size_t plane, size_t at, int from, int dir,
                                            int count, int w, int nw, int lane, float* h) {
    const int per = (count + nw - 1) / nw, q0 = min(w * per, count), q1 = min(q0 + per, count);
    float A[V], S[V];
#pragma unroll
    for (int j = 0; j < V; ++j) A[j] = 1.0f, S[j] = 0.0f;
    for (int q = q0; q < q1; ++q) {
        const float* a = agg + (size_t)(from + dir * q) * 2 * plane + at;
        const auto qa = vload<float, V>(a), qs = vload<float, V>(a + plane);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            S[j] = apply<MASK>(qa.get(j), qs.get(j), S[j]);
            A[j] = product<MASK>(A[j], qa.get(j));
        }
    }
    m.put(0, w, lane, A, S);
    barrier_lds();
    for (int q = 0; q < nw; ++q) m.template run<MASK>(0, q, lane, h);
    barrier_lds();                           // the buffer is free again
}

template <class S, int V>
struct Inputs {                              // a wave's steps of one block, as loaded
    Vec<S, V> z[kSteps], f[kSteps];
    uint8_t start[kSteps];
};

}  // namespace

// SUM: only the range's map, into p.ws. PACK: z and f also to 8 bits.
template <class S, int V, bool MASK, bool PACK, bool SUM>
__global__ void __launch_bounds__(512) gated_fwd_kernel(GatedScan p, int per_row, int range) {
    __shared__ Maps<V> maps;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = blockDim.x >> 6;
    const Lane<V> ln(p, per_row);
    const int T = p.T, N = p.N, B = p.B, b = ln.b, n0 = ln.n0;
    const size_t plane = (size_t)B * N, at = (size_t)b * N + n0;
    const int ts = blockIdx.y * range, te = min(ts + range, T);
    const S* zp = (const S*)p.z.data + b * p.z.s1 + n0;
    const S* fp = (const S*)p.f.data + b * p.f.s1 + n0;
    const int len = MASK ? row_length(p, b) : T;
    const int ng = (N + kGroup8 - 1) / kGroup8;
    float bias[V], h[V], sumA[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        bias[j] = p.bias ? p.bias[n0 + j] : 0.0f;
        h[j] = !SUM && p.h0 ? p.h0[at + j] : 0.0f;
        sumA[j] = 1.0f;
    }
    if (!SUM && blockIdx.y) enter_range<V, MASK>(maps, p.ws, plane, at, 0, 1, blockIdx.y, w, nw, lane, h);

    auto load = [&](Inputs<S, V>& in, int tb) {
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
            const int t = min(tb + w * kSteps + k, T - 1);
            in.z[k] = vload<S, V>(zp + t * p.z.s0);
            in.f[k] = vload<S, V>(fp + t * p.f.s0);
            if (MASK) in.start[k] = p.starts ? p.starts[(size_t)t * B + b] : 0;
        }
    };
    Inputs<S, V> in;
    load(in, ts);
    int buf = 0;
    for (int tb = ts; tb < te; tb += nw * kSteps, buf ^= 1) {
        const int t0 = tb + w * kSteps;
        float kk[kSteps][V], zz[kSteps][V], A[V], L[V];
        bool fresh[kSteps], live[kSteps];
#pragma unroll
        for (int j = 0; j < V; ++j) A[j] = 1.0f, L[j] = 0.0f;
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
            live[k] = t0 + k < (MASK ? len : T);
            fresh[k] = MASK && live[k] && in.start[k];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float z = in.z[k].get(j);
                kk[k][j] = live[k] ? gate_in(in.f[k].get(j) + bias[j]) : 0.0f;
                zz[k][j] = live[k] ? z : 0.0f;
                if (MASK && fresh[k]) L[j] = 0.0f;
                L[j] = fmaf(kk[k][j], zz[k][j] - L[j], L[j]);
                A[j] = fresh[k] ? -1.0f : product<MASK>(A[j], 1.0f - kk[k][j]);
            }
        }
        if constexpr (PACK) {
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                const int t = t0 + k;
                if (t >= T) break;
                float v[V];
                const size_t row = (size_t)t * B + b;
#pragma unroll
                for (int j = 0; j < V; ++j) v[j] = in.z[k].get(j);
                store8<V>(v, ln.skip, ln.first, p.z8.q + row * N + n0, p.z8.scale + row * ng + ln.group);
#pragma unroll
                for (int j = 0; j < V; ++j) v[j] = in.f[k].get(j);
                store8<V>(v, ln.skip, ln.first, p.f8.q + row * N + n0, p.f8.scale + row * ng + ln.group);
            }
        }
        maps.put(buf, w, lane, A, L);
        barrier_lds();
        if (tb + nw * kSteps < te) load(in, tb + nw * kSteps);
        if (!SUM && p.states && w == 0 && ln.on) vstore<float, V>(p.states + (size_t)(tb / kBlk) * plane + at, h);
        float g[V];
        for (int q = 0; q < nw; ++q) {
            if (q == w) {
#pragma unroll
                for (int j = 0; j < V; ++j) g[j] = h[j];
            }
            maps.template run<MASK>(buf, q, lane, h);
            if constexpr (SUM) {
#pragma unroll
                for (int j = 0; j < V; ++j) sumA[j] = product<MASK>(sumA[j], maps.A[buf][q][lane * V + j]);
            }
        }
        if constexpr (!SUM) {
            S* yp = (S*)p.h.data + b * p.h.s1 + n0;
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                if (t0 + k >= T) break;
                float y[V];
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    if (MASK && fresh[k]) g[j] = 0.0f;
                    g[j] = fmaf(kk[k][j], zz[k][j] - g[j], g[j]);
                    y[j] = live[k] ? g[j] : 0.0f;
                }
                if (ln.on) vstore<S, V>(yp + (t0 + k) * p.h.s0, y);
            }
        }
    }
    if (w || !ln.on) return;
    if constexpr (SUM) {
        float* a = p.ws + (size_t)blockIdx.y * 2 * plane + at;
        vstore<float, V>(a, sumA);
        vstore<float, V>(a + plane, h);
    } else if (te == T) {
        vstore<float, V>(p.h_last + at, h);
    }
}

// SUM: only the range's reverse map, from f and dh. PACK: z and f from their 8 bits.
template <class S, int V, bool MASK, bool PACK, bool SUM>
__global__ void __launch_bounds__(512) gated_bwd_kernel(GatedScan p, int per_row, int range, float* dbpart) {
    __shared__ Maps<V> fmap, rmap;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = blockDim.x >> 6;
    const Lane<V> ln(p, per_row);
    const int T = p.T, N = p.N, B = p.B, b = ln.b, n0 = ln.n0;
    const size_t plane = (size_t)B * N, at = (size_t)b * N + n0;
    const int ts = blockIdx.y * range, te = min(ts + range, T);
    const int ng = (N + kGroup8 - 1) / kGroup8;
    const S* zp = (const S*)p.z.data + b * p.z.s1 + n0;
    const S* fp = (const S*)p.f.data + b * p.f.s1 + n0;
    const S* dhp = (const S*)p.dh.data + b * p.dh.s1 + n0;
    const int len = MASK ? row_length(p, b) : T;
    float bias[V], c[V], sumA[V], db[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        bias[j] = p.bias ? p.bias[n0 + j] : 0.0f;
        c[j] = !SUM && p.dlast ? p.dlast[at + j] : 0.0f;
        sumA[j] = 1.0f;
        db[j] = 0.0f;
    }
    const int last = gridDim.y - 1;
    if (!SUM && (int)blockIdx.y < last)
        enter_range<V, MASK>(rmap, p.ws, plane, at, last, -1, last - blockIdx.y, w, nw, lane, c);

    int buf = 0;
    for (int tb = ts + (te - 1 - ts) / (nw * kSteps) * (nw * kSteps); tb >= ts; tb -= nw * kSteps, buf ^= 1) {
        const int t0 = tb + w * kSteps;
        float kk[kSteps][V], zz[kSteps][V], dh[kSteps][V];
        bool fresh[kSteps], live[kSteps];
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
            const int t = min(t0 + k, T - 1);
            live[k] = t0 + k < (MASK ? len : T);
            fresh[k] = MASK && live[k] && p.starts && p.starts[(size_t)t * B + b];
            const auto d = vload<S, V>(dhp + t * p.dh.s0);
            float f[V], z[V];
            if constexpr (PACK) {
                const size_t row = (size_t)t * B + b;
                const auto f8 = load8<V>(p.f8, row, n0, N, ng);
#pragma unroll
                for (int j = 0; j < V; ++j) f[j] = f8.get(j);
                if constexpr (!SUM) {
                    const auto z8 = load8<V>(p.z8, row, n0, N, ng);
#pragma unroll
                    for (int j = 0; j < V; ++j) z[j] = z8.get(j);
                }
            } else {
                const auto fv = vload<S, V>(fp + t * p.f.s0);
#pragma unroll
                for (int j = 0; j < V; ++j) f[j] = fv.get(j);
                if constexpr (!SUM) {
                    const auto zv = vload<S, V>(zp + t * p.z.s0);
#pragma unroll
                    for (int j = 0; j < V; ++j) z[j] = zv.get(j);
                }
            }
#pragma unroll
            for (int j = 0; j < V; ++j) {
                kk[k][j] = live[k] ? gate_in(f[j] + bias[j]) : 0.0f;
                dh[k][j] = live[k] ? d.get(j) : 0.0f;
                if (!SUM) zz[k][j] = live[k] ? z[j] : 0.0f;
            }
        }
        float A[V], L[V];
#pragma unroll
        for (int j = 0; j < V; ++j) A[j] = 1.0f, L[j] = 0.0f;
        if constexpr (!SUM) {
#pragma unroll
            for (int k = 0; k < kSteps; ++k)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    if (MASK && fresh[k]) L[j] = 0.0f;
                    L[j] = fmaf(kk[k][j], zz[k][j] - L[j], L[j]);
                    A[j] = fresh[k] ? -1.0f : product<MASK>(A[j], 1.0f - kk[k][j]);
                }
            fmap.put(buf, w, lane, A, L);
#pragma unroll
            for (int j = 0; j < V; ++j) A[j] = 1.0f, L[j] = 0.0f;
        }
#pragma unroll
        for (int k = kSteps - 1; k >= 0; --k)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float a = 1.0f - kk[k][j];
                L[j] = MASK && fresh[k] ? 0.0f : a * (dh[k][j] + L[j]);
                A[j] = fresh[k] ? -1.0f : product<MASK>(A[j], a);
            }
        rmap.put(buf, w, lane, A, L);
        barrier_lds();
        float g[V];
        for (int q = nw - 1; q >= 0; --q) {
            if (q == w) {
#pragma unroll
                for (int j = 0; j < V; ++j) g[j] = c[j];
            }
            rmap.template run<MASK>(buf, q, lane, c);
            if constexpr (SUM) {
#pragma unroll
                for (int j = 0; j < V; ++j) sumA[j] = product<MASK>(sumA[j], rmap.A[buf][q][lane * V + j]);
            }
        }
        if constexpr (!SUM) {
            float h[V], blk[V];
            const auto st = vload<float, V>(p.states + (size_t)(tb / kBlk) * plane + at);
#pragma unroll
            for (int j = 0; j < V; ++j) h[j] = st.get(j), blk[j] = 0.0f;
            for (int q = 0; q < w; ++q) fmap.template run<MASK>(buf, q, lane, h);
            // zz becomes h_{t-1} - z_t
#pragma unroll
            for (int k = 0; k < kSteps; ++k)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    if (MASK && fresh[k]) h[j] = 0.0f;
                    const float d = h[j] - zz[k][j];
                    h[j] = fmaf(-kk[k][j], d, h[j]);
                    zz[k][j] = live[k] ? d : 0.0f;
                }
            S* dzp = (S*)p.dz.data + b * p.dz.s1 + n0;
            S* dfp = (S*)p.df.data + b * p.df.s1 + n0;
#pragma unroll
            for (int k = kSteps - 1; k >= 0; --k) {
                float oz[V], of[V];
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float a = 1.0f - kk[k][j], lam = dh[k][j] + g[j];
                    oz[j] = live[k] ? lam * kk[k][j] : 0.0f;
                    of[j] = oz[j] * a * zz[k][j];
                    blk[j] += of[j];
                    g[j] = MASK && fresh[k] ? 0.0f : a * lam;
                }
                if (t0 + k < T && ln.on) {
                    vstore<S, V>(dzp + (t0 + k) * p.dz.s0, oz);
                    vstore<S, V>(dfp + (t0 + k) * p.df.s0, of);
                }
            }
            // the bias sum in two levels: within a block, then over blocks
#pragma unroll
            for (int j = 0; j < V; ++j) db[j] += blk[j];
        }
    }
    if constexpr (SUM) {
        if (w || !ln.on) return;
        float* a = p.ws + (size_t)blockIdx.y * 2 * plane + at;
        vstore<float, V>(a, sumA);
        vstore<float, V>(a + plane, c);
    } else {
        if (w == 0 && ln.on && ts == 0 && p.dh0) vstore<float, V>(p.dh0 + at, c);
        if (!dbpart) return;
        __syncthreads();
        float one[V];
#pragma unroll
        for (int j = 0; j < V; ++j) one[j] = 1.0f;
        rmap.put(0, w, lane, one, db);
        __syncthreads();
        if (w || !ln.on) return;
        for (int q = 1; q < nw; ++q)
#pragma unroll
            for (int j = 0; j < V; ++j) db[j] += rmap.S[0][q][lane * V + j];
        vstore<float, V>(dbpart + (size_t)blockIdx.y * plane + at, db);
    }
}

namespace {

struct Plan {
    int V, per_row, groups, waves, range, ranges;
};

// V = 4 wherever a row holds four columns. Time over the grid where the channels alone do not
// give every CU a workgroup.
Plan gated_plan(int T, int B, int N, bool pack) {
    Plan q;
    q.V = N >= 4 ? 4 : 1;
    q.per_row = pack ? (N + kGroup8 - 1) / kGroup8 * (kGroup8 / q.V) : (N + q.V - 1) / q.V;
    q.groups = (int)(((long long)B * q.per_row + 63) / 64);
    q.waves = T >= kBlk ? kWaves : (T + kSteps - 1) / kSteps;
    const int blocks = (T + kBlk - 1) / kBlk;
    int want = q.groups >= 256 ? 1 : (512 + q.groups - 1) / q.groups;
    if (want > 64) want = 64;
    if (want > blocks / 2) want = blocks / 2 < 1 ? 1 : blocks / 2;
    const int per = (blocks + want - 1) / want;
    q.range = per * kBlk;
    q.ranges = (blocks + per - 1) / per;
    return q;
}

size_t map_floats(const Plan& q, int B, int N) { return q.ranges > 1 ? (size_t)q.ranges * 2 * B * N : 0; }

template <class S, int V, bool MASK, bool PACK>
void run_gated(const GatedScan& p, const Plan& q, bool fwd, hipStream_t stream) {
    const dim3 block(64 * q.waves), grid(q.groups, q.ranges), inner(q.groups, q.ranges);
    if (fwd) {
        if (q.ranges > 1)
            hipLaunchKernelGGL((gated_fwd_kernel<S, V, MASK, false, true>), inner, block, 0, stream, p, q.per_row, q.range);
        hipLaunchKernelGGL((gated_fwd_kernel<S, V, MASK, PACK, false>), grid, block, 0, stream, p, q.per_row, q.range);
    } else {
        float* part = p.db ? p.ws + map_floats(q, p.B, p.N) : nullptr;
        if (q.ranges > 1)
            hipLaunchKernelGGL((gated_bwd_kernel<S, V, MASK, PACK, true>), inner, block, 0, stream, p, q.per_row, q.range, nullptr);
        hipLaunchKernelGGL((gated_bwd_kernel<S, V, MASK, PACK, false>), grid, block, 0, stream, p, q.per_row, q.range, part);
        if (p.db) launch_column_sums(part, q.ranges * p.B, p.N, p.N, p.db, nullptr, nullptr, stream);
    }
}

template <class S, int V>
void run_gated_m(const GatedScan& p, const Plan& q, bool fwd, hipStream_t stream) {
    const bool mask = p.starts || p.lengths;
    if (p.z8.q) mask ? run_gated<S, V, true, true>(p, q, fwd, stream) : run_gated<S, V, false, true>(p, q, fwd, stream);
    else mask ? run_gated<S, V, true, false>(p, q, fwd, stream) : run_gated<S, V, false, false>(p, q, fwd, stream);
}

void launch_gated(const GatedScan& p, bool fwd, hipStream_t stream) {
    const Plan q = gated_plan(p.T, p.B, p.N, p.z8.q != nullptr);
    if (p.bf16) q.V == 4 ? run_gated_m<__bf16, 4>(p, q, fwd, stream) : run_gated_m<__bf16, 1>(p, q, fwd, stream);
    else q.V == 4 ? run_gated_m<float, 4>(p, q, fwd, stream) : run_gated_m<float, 1>(p, q, fwd, stream);
}

}  // namespace

// floats of workspace: the ranges' maps, and the ranges' bias sums (the 8-bit form's wider rows
// give at most as many ranges)
size_t gated_fwd_ws(int T, int B, int N) {
    return std::max(map_floats(gated_plan(T, B, N, false), B, N), map_floats(gated_plan(T, B, N, true), B, N));
}
size_t gated_bwd_ws(int T, int B, int N) {
    const Plan a = gated_plan(T, B, N, false), b = gated_plan(T, B, N, true);
    return gated_fwd_ws(T, B, N) + (size_t)std::max(a.ranges, b.ranges) * B * N;
}

void launch_gated_fwd(const GatedScan& p, hipStream_t stream) { launch_gated(p, true, stream); }
void launch_gated_bwd(const GatedScan& p, hipStream_t stream) { launch_gated(p, false, stream); }

}  // namespace delrec
