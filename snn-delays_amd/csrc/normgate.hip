// Norms around a residual block, fused with its gate and residual scale, over rows of N:
//     r = 1/sqrt(mean o^2 + eps), y = o r w silu(g), x' = x + scale y,
//     r2 = 1/sqrt(mean x'^2 + eps), u = x' r2 w2.
// Backwards, with e = o r, e2 = x' r2, v2 = w2 du and the row means <.>:
//     dx = dx' + r2 (v2 - e2 <v2 e2>),  dn = scale dx silu(g),  v = w dn,
//     do = r (v - e <v e>),  dg = scale dx e w silu'(g),
//     dw2 = sum du e2,  dscale = sum dx y,  dw = sum dn e       (sums over the rows).
//
// Bound by memory: a row stays in registers between its loads and its stores, the two row sums
// are exchanges between its lanes. A row is 16, 64, 256 or 512 lanes, each with up to four vectors of
// four columns (16 lanes: four rows a wave, no LDS): forward 31 us for 32000 x 512 bf16 (5.2 TB/s).
// The backward recomputes x', e and the gate from o, g and x (or their 8 bits) and the two kept
// norms: one residual tensor is read, not two. Its column sums stay in registers over all the rows
// a workgroup takes; the workgroups' sums are added in a second launch, in a fixed order.
#include <algorithm>
#include <initializer_list>

#include "gated.h"
#include "kernels.h"

namespace delrec {

namespace {

// ---- rows of any width (two or three columns, or past 8192): one workgroup a row ----

constexpr int kNb = 256;

__device__ __forceinline__ float row_sum(float v, float* red) {
    v = group_sum_t<64>(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}

template <class T>
__device__ __forceinline__ T* row_ptr(const delrec_rows& x, long long row, int R1) {
    return (T*)x.data + (row / R1) * x.s0 + (row % R1) * x.s1;
}

__device__ __forceinline__ float sigm(float g) { return gate_in(-g); }

template <class S>
__device__ __forceinline__ float val8(const delrec_rows& x, const delrec_packed8& q, long long row, int n, int R1, int N) {
    if (!q.q) return to_f32(row_ptr<S>(x, row, R1)[n]);
    return (float)q.q[row * pitch8(N) + n] * q.scale[row * ((N + kGroup8 - 1) / kGroup8) + n / kGroup8];
}

}  // namespace

// the block's output at one position: o (or, in a step, the state's update), gate, residual
template <class S, class X>
__global__ void __launch_bounds__(kNb) norm_any_fwd_kernel(NormGate p) {
    __shared__ float red[4];
    const int N = p.N;
    const bool block = p.o.data || p.h;
    const long long rows = (long long)p.R0 * p.R1;
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
        const X* x = row_ptr<const X>(p.x, row, p.R1);
        float r = 0.0f, r2 = 0.0f, s = 0.0f;
        if (p.h) {
            for (int n = threadIdx.x; n < N; n += kNb) {
                const float f = to_f32(row_ptr<const S>(p.f, row, p.R1)[n]), z = to_f32(row_ptr<const S>(p.z, row, p.R1)[n]);
                const float m = gate_small2(fmaf(f, kLog2e, p.bias ? p.bias[n] * kLog2e : 0.0f)), h = p.h[row * N + n];
                p.h_out[row * N + n] = gate_step(m, h - z, h, z);
            }
            __syncthreads();
        }
        auto oval = [&](int n) { return p.h ? p.h_out[row * N + n] : to_f32(row_ptr<const S>(p.o, row, p.R1)[n]); };
        if (block) {
            for (int n = threadIdx.x; n < N; n += kNb) {
                const float o = oval(n);
                s += o * o;
            }
            r = 1.0f / sqrtf(row_sum(s, red) / (float)N + p.eps);
        }
        auto xval = [&](int n) {
            const float xv = to_f32(x[n]);
            if (!block) return xv;
            const float g = to_f32(row_ptr<const S>(p.g, row, p.R1)[n]);
            return fmaf(p.scale[n], oval(n) * r * p.w[n] * (g * sigm(g)), xv);
        };
        s = 0.0f;
        for (int n = threadIdx.x; n < N; n += kNb) {
            const float v = xval(n);
            if (block) ((X*)p.x_out)[row * N + n] = (X)v;
            s += v * v;
        }
        if (p.w2) {
            r2 = 1.0f / sqrtf(row_sum(s, red) / (float)N + p.eps);
            for (int n = threadIdx.x; n < N; n += kNb) ((S*)p.u)[row * N + n] = (S)(xval(n) * r2 * p.w2[n]);
        }
        if (p.stats && threadIdx.x == 0) {
            p.stats[2 * row] = r;
            p.stats[2 * row + 1] = r2;
        }
    }
}

template <class S, class X>
__global__ void __launch_bounds__(kNb) norm_any_bwd_kernel(NormGate p) {
    __shared__ float red[4];
    const int N = p.N, tid = threadIdx.x;
    const bool block = p.w != nullptr;
    float *dwp = p.part + (size_t)blockIdx.x * 3 * N, *dsp = dwp + N, *dw2p = dsp + N;
    for (int n = tid; n < N; n += kNb) dwp[n] = dsp[n] = dw2p[n] = 0.0f;
    __syncthreads();
    const long long rows = (long long)p.R0 * p.R1;
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
        const float r = p.stats[2 * row], r2 = p.stats[2 * row + 1];
        auto oval = [&](int n) { return val8<S>(p.o, p.o8, row, n, p.R1, N); };
        auto gval = [&](int n) { return val8<S>(p.g, p.g8, row, n, p.R1, N); };
        auto e2val = [&](int n) {
            float v = val8<X>(p.x, p.x8, row, n, p.R1, N);
            if (block) {
                const float g = gval(n);
                v = fmaf(p.scale[n], oval(n) * r * p.w[n] * (g * sigm(g)), v);
            }
            return v * r2;
        };
        auto duval = [&](int n) { return p.du.data ? to_f32(row_ptr<const S>(p.du, row, p.R1)[n]) : 0.0f; };
        float s = 0.0f, m2 = 0.0f;
        if (p.w2) {
            for (int n = tid; n < N; n += kNb) s += p.w2[n] * duval(n) * e2val(n);
            m2 = row_sum(s, red) / (float)N;
        }
        auto dxval = [&](int n) {
            const float up = p.dx_out.data ? to_f32(row_ptr<const X>(p.dx_out, row, p.R1)[n]) : 0.0f;
            return p.w2 ? up + r2 * (p.w2[n] * duval(n) - e2val(n) * m2) : up;
        };
        s = 0.0f;
        for (int n = tid; n < N; n += kNb) {
            const float dx = dxval(n);
            row_ptr<X>(p.dx, row, p.R1)[n] = (X)dx;
            if (p.w2) dw2p[n] += duval(n) * e2val(n);
            if (block) {
                const float g = gval(n), sg = sigm(g), si = g * sg, e = oval(n) * r, dn = p.scale[n] * dx * si;
                dwp[n] += dn * e;
                dsp[n] += dx * e * p.w[n] * si;
                row_ptr<S>(p.dg, row, p.R1)[n] = (S)(p.scale[n] * dx * e * p.w[n] * (sg + si * (1.0f - sg)));
                s += p.w[n] * dn * e;
            }
        }
        if (block) {
            const float m = row_sum(s, red) / (float)N;
            for (int n = tid; n < N; n += kNb) {
                const float g = gval(n), e = oval(n) * r, v = p.w[n] * p.scale[n] * dxval(n) * (g * sigm(g));
                row_ptr<S>(p.d_o, row, p.R1)[n] = (S)(r * (v - e * m));
            }
        }
        __syncthreads();
    }
}

// out_k[n] = sum over rows of part[row * pitch + k * N + n], k < 3, in a fixed order
__global__ void __launch_bounds__(1024) column_sums_kernel(const float* part, unsigned rows, int N, unsigned pitch, float* o0,
                                                           float* o1, float* o2) {
    __shared__ float red[16][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, k = blockIdx.y;
    float* out = k == 0 ? o0 : (k == 1 ? o1 : o2);
    for (long long n0 = blockIdx.x * 64LL; n0 < N; n0 += gridDim.x * 64LL) {
        const int n = (int)n0 + lane;
        // eight rows' loads in flight at a time (past the end the last row again, left out)
        float s8[8] = {};
        const float* at = part + (size_t)k * N + min(n, N - 1);
        for (unsigned r = w; r < rows; r += 128) {
            float v[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) v[q] = at[(size_t)min(r + 16 * q, rows - 1) * pitch];
#pragma unroll
            for (int q = 0; q < 8; ++q) s8[q] += r + 16 * q < rows ? v[q] : 0.0f;
        }
        float s = ((s8[0] + s8[1]) + (s8[2] + s8[3])) + ((s8[4] + s8[5]) + (s8[6] + s8[7]));
        red[w][lane] = s;
        __syncthreads();
        if (w == 0 && n < N && out) {
            s = red[0][lane];
            for (int q = 1; q < 16; ++q) s += red[q][lane];
            out[n] = s;
        }
        __syncthreads();
    }
}

void launch_column_sums(const float* part, unsigned rows, int N, unsigned pitch, float* o0, float* o1, float* o2, hipStream_t stream) {
    hipLaunchKernelGGL(column_sums_kernel, dim3(std::min((N - 1) / 64 + 1, kMostBlocks), pitch / N), dim3(1024), 0, stream, part, rows, N, pitch, o0, o1, o2);
}

// ---- rows of 4 to 8192 columns in registers ----

namespace {

template <int LPR>
constexpr int kRowBlock = LPR < 256 ? 256 : LPR;

// a sum over the row's lanes; `slot`: this call's LDS words (two sets, used in turn)
template <int LPR>
__device__ __forceinline__ float lanes_sum(float v, float* red, int slot) {
    v = group_sum_t<LPR < 64 ? LPR : 64>(v);
    if constexpr (LPR > 64) {
        constexpr int W = LPR / 64;
        if ((threadIdx.x & 63) == 0) red[slot * W + (threadIdx.x >> 6)] = v;
        barrier_lds();
        v = red[slot * W];
#pragma unroll
        for (int q = 1; q < W; ++q) v += red[slot * W + q];
    }
    return v;
}

// The lane's columns. The last lane of a row whose width is no multiple of 4 is moved back to end
// with it; lanes past the row repeat its last columns. Both compute and, where they store, store
// the values of columns that other lanes hold as well; sums leave the first `skip` out.
template <int LPR, int NE>
struct Cols {
    int n0[NE], skip[NE], group[NE], i[NE];
    bool on[NE], first[NE];
    __device__ __forceinline__ Cols(int lane, int N) {
#pragma unroll
        for (int e = 0; e < NE; ++e) {
            i[e] = (e * LPR + lane) * 4;
            on[e] = i[e] < N;
            n0[e] = min(i[e], N - 4);
            skip[e] = on[e] ? i[e] - n0[e] : 4;
            group[e] = min(i[e], N - 1) / kGroup8;
            first[e] = on[e] && i[e] % kGroup8 == 0;
        }
    }
};

template <class T>
__device__ __forceinline__ T* row_at(const delrec_rows& x, long long row, const NormGate& p) {
    if (p.flat) return (T*)x.data + row * x.s1;
    const unsigned r = (unsigned)row, i = r / (unsigned)p.R1, j = r - i * (unsigned)p.R1;
    return (T*)x.data + i * x.s0 + j * x.s1;
}

template <int NE>
__device__ __forceinline__ void load_cols(float (&v)[NE][4], const float* x, const int (&n0)[NE]) {
#pragma unroll
    for (int e = 0; e < NE; ++e) {
        const auto t = vload<float, 4>(x + n0[e]);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[e][j] = t.get(j);
    }
}

enum { kNormOnly = 0, kNormBlock = 1, kNormStep = 2 };

}  // namespace

template <class S, class X, int LPR, int NE, int FORM>
__global__ void __launch_bounds__(kRowBlock<LPR>) norm_gate_fwd_kernel(NormGate p) {
    __shared__ float red[2 * (LPR > 64 ? LPR / 64 : 1)];
    constexpr int RPW = kRowBlock<LPR> / LPR;
    const int lane = threadIdx.x % LPR, N = p.N, ng = (N + kGroup8 - 1) / kGroup8;
    const Cols<LPR, NE> c(lane, N);
    const long long rows = (long long)p.R0 * p.R1;
    float w[NE][4], sc[NE][4], w2[NE][4], bias[NE][4];
    if constexpr (FORM != kNormOnly) {
        load_cols<NE>(w, p.w, c.n0);
        load_cols<NE>(sc, p.scale, c.n0);
    }
    if (p.w2) load_cols<NE>(w2, p.w2, c.n0);
    if constexpr (FORM == kNormStep) {
        if (p.bias) load_cols<NE>(bias, p.bias, c.n0);
    }
    const float inv_n = 1.0f / (float)N;
    // rows past the end repeat the last one and store nothing (its lanes join the exchanges)
    for (long long r0 = (long long)blockIdx.x * RPW; r0 < rows; r0 += (long long)gridDim.x * RPW) {
        const long long mine = r0 + threadIdx.x / LPR, row = mine < rows ? mine : rows - 1;
        const bool live = mine < rows;
        Vec<X, 4> xv[NE];
        Vec<S, 4> ov[NE], gv[NE];
        float o[NE][4], x[NE][4], r = 0.0f, r2 = 0.0f, s = 0.0f;
        const X* xp = row_at<const X>(p.x, row, p);
#pragma unroll
        for (int e = 0; e < NE; ++e) xv[e] = vload<X, 4>(xp + c.n0[e]);
        if constexpr (FORM != kNormOnly) {
            const S* gp = row_at<const S>(p.g, row, p);
#pragma unroll
            for (int e = 0; e < NE; ++e) gv[e] = vload<S, 4>(gp + c.n0[e]);
            if constexpr (FORM == kNormBlock) {
                const S* op = row_at<const S>(p.o, row, p);
#pragma unroll
                for (int e = 0; e < NE; ++e) {
                    ov[e] = vload<S, 4>(op + c.n0[e]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[e][j] = ov[e].get(j);
                }
            } else {
                const S* zp = row_at<const S>(p.z, row, p);
                const S* fp = row_at<const S>(p.f, row, p);
#pragma unroll
                for (int e = 0; e < NE; ++e) {
                    const auto z = vload<S, 4>(zp + c.n0[e]);
                    const auto f = vload<S, 4>(fp + c.n0[e]);
                    const auto h = vload<float, 4>(p.h + row * N + c.n0[e]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float m = gate_small2(f.get_fma(j, kLog2e, p.bias ? bias[e][j] * kLog2e : 0.0f));
                        o[e][j] = gate_step(m, h.get(j) - z.get(j), h.get(j), z.get(j));
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < NE; ++e)
#pragma unroll
                for (int j = 0; j < 4; ++j) s += j >= c.skip[e] ? o[e][j] * o[e][j] : 0.0f;
            r = 1.0f / sqrtf(lanes_sum<LPR>(s, red, 0) * inv_n + p.eps);
            s = 0.0f;
        }
#pragma unroll
        for (int e = 0; e < NE; ++e) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[e][j] = xv[e].get(j);
                if constexpr (FORM != kNormOnly) {
                    const float g = gv[e].get(j);
                    x[e][j] = fmaf(sc[e][j], o[e][j] * r * w[e][j] * (g * sigm(g)), x[e][j]);
                }
                s += j >= c.skip[e] ? x[e][j] * x[e][j] : 0.0f;
            }
            if constexpr (FORM != kNormOnly) {
                if (live && c.on[e]) {
                    vstore<X, 4>((X*)p.x_out + row * N + c.n0[e], x[e]);
                    // in place: no lane may read a column of h that another has written. Every
                    // lane of the row has read its own before the first row sum.
                    if constexpr (FORM == kNormStep) vstore<float, 4>(p.h_out + row * N + c.n0[e], o[e]);
                }
            }
        }
        if (p.w2) {
            r2 = 1.0f / sqrtf(lanes_sum<LPR>(s, red, 1) * inv_n + p.eps);
#pragma unroll
            for (int e = 0; e < NE; ++e) {
                float u[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) u[j] = x[e][j] * r2 * w2[e][j];
                if (live && c.on[e]) vstore<S, 4>((S*)p.u + row * N + c.n0[e], u);
            }
        }
        // rows with one sum alone: its words are read before the next row's are written
        if constexpr (LPR > 64) {
            if (FORM == kNormOnly || !p.w2) barrier_lds();
        }
        if constexpr (FORM != kNormStep) {
            if (p.stats && live && lane == 0) {
                p.stats[2 * row] = r;
                p.stats[2 * row + 1] = r2;
            }
            if (p.x8.q) {
#pragma unroll
                for (int e = 0; e < NE; ++e) {
                    const Lane8<4> l8(c.i[e], c.skip[e], live && c.on[e], N);
                    const bool first = live && c.first[e];
                    const size_t q = row * pitch8(N), g = row * ng + c.group[e];
                    float v[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[j] = xv[e].get(j);
                    store8<4>(v, l8, first, p.x8.q + q, p.x8.scale + g);
                    if constexpr (FORM == kNormBlock) {
                        store8<4>(o[e], l8, first, p.o8.q + q, p.o8.scale + g);
#pragma unroll
                        for (int j = 0; j < 4; ++j) v[j] = gv[e].get(j);
                        store8<4>(v, l8, first, p.g8.q + q, p.g8.scale + g);
                    }
                }
            }
        }
    }
}

// PACK: o, g and x from their 8 bits. Up to two vectors a lane (N 4096), a row's values are loaded
// while the one before is computed, and the three column vectors are in LDS, read again in each
// half of a row. Each row's loads waited for in place, the columns in registers: 77 us for 32000 x
// 512 bf16 and 660 for 65536 x 2048 with 8 bits; so 50 (5.3 TB/s) and 485 (4.7 TB/s). With four
// vectors there are no registers for either.
template <class S, class X, int LPR, int NE, bool BLOCK, bool PACK>
__global__ void __launch_bounds__(kRowBlock<LPR>) norm_gate_bwd_kernel(NormGate p) {
    constexpr int RPW = kRowBlock<LPR> / LPR, W = LPR > 64 ? LPR / 64 : 1, ROW = LPR * NE * 4;
    constexpr bool SHARED = NE <= 2, AHEAD = NE <= 2;
    __shared__ float red[2 * W];
    __shared__ float slots[RPW > 1 ? RPW : 1][RPW > 1 ? ROW : 1];
    __shared__ float cols[SHARED ? 3 : 1][SHARED ? ROW : 1];
    const int lane = threadIdx.x % LPR, N = p.N, ng = (N + kGroup8 - 1) / kGroup8;
    const Cols<LPR, NE> c(lane, N);
    const long long rows = (long long)p.R0 * p.R1, step = (long long)gridDim.x * RPW;
    float held[SHARED ? 1 : 3][NE][4], acc[3][NE][4];
    auto fill = [&](int k, const float* src) {
#pragma unroll
        for (int e = 0; e < NE; ++e) {
            float v[4] = {};
            if (src) {
                const auto t = vload<float, 4>(src + c.n0[e]);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = t.get(j);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (SHARED) cols[k][(e * LPR + lane) * 4 + j] = v[j];
                else held[k][e][j] = v[j];
                acc[k][e][j] = 0.0f;
            }
        }
    };
    fill(0, BLOCK ? p.w : nullptr);
    fill(1, BLOCK ? p.scale : nullptr);
    fill(2, p.w2);
    __syncthreads();
    auto col = [&](int k, int e, int j) {
        if constexpr (SHARED) return cols[k][(e * LPR + lane) * 4 + j];
        else return held[k][e][j];
    };

    typedef typename std::conditional<PACK, Vec8<4>, Vec<S, 4>>::type SV;
    typedef typename std::conditional<PACK, Vec8<4>, Vec<X, 4>>::type XV;
    struct Raw {
        SV o[NE], g[NE];
        XV x[NE];
        Vec<X, 4> up[NE];
        Vec<S, 4> du[NE];
        float r, r2;
    } in;
    // rows past the end repeat the last one, with no gradient, and store nothing
    auto load = [&](long long r0) {
        const long long mine = r0 + threadIdx.x / LPR, row = mine < rows ? mine : rows - 1;
        const size_t q = (size_t)row * pitch8(N), s = (size_t)row * ng;
        in.r = p.stats[2 * row];
        in.r2 = p.stats[2 * row + 1];
#pragma unroll
        for (int e = 0; e < NE; ++e) {
            if constexpr (PACK) {
                const Lane8<4> l8(c.i[e], c.skip[e], c.on[e], N);
                if constexpr (BLOCK) {
                    in.o[e] = load8<4>(p.o8.q + q, p.o8.scale + s + c.group[e], l8);
                    in.g[e] = load8<4>(p.g8.q + q, p.g8.scale + s + c.group[e], l8);
                }
                in.x[e] = load8<4>(p.x8.q + q, p.x8.scale + s + c.group[e], l8);
            } else {
                if constexpr (BLOCK) {
                    in.o[e] = vload<S, 4>(row_at<const S>(p.o, row, p) + c.n0[e]);
                    in.g[e] = vload<S, 4>(row_at<const S>(p.g, row, p) + c.n0[e]);
                }
                in.x[e] = vload<X, 4>(row_at<const X>(p.x, row, p) + c.n0[e]);
            }
            if (p.dx_out.data) in.up[e] = vload<X, 4>(row_at<const X>(p.dx_out, row, p) + c.n0[e]);
            if (p.du.data) in.du[e] = vload<S, 4>(row_at<const S>(p.du, row, p) + c.n0[e]);
        }
    };
    const float inv_n = 1.0f / (float)N;
    long long r0 = (long long)blockIdx.x * RPW;
    if (AHEAD && r0 < rows) load(r0);
    for (; r0 < rows; r0 += step) {
        if (!AHEAD) load(r0);
        const long long mine = r0 + threadIdx.x / LPR, row = mine < rows ? mine : rows - 1;
        const bool live = mine < rows, has_up = live && p.dx_out.data, has_du = live && p.du.data;
        // (without a second norm r2 and x count as zeros, also where x is not finite)
        const float r = in.r, r2 = p.w2 ? in.r2 : 0.0f;
        float o[NE][4], g[NE][4], x[NE][4], up[NE][4], du[NE][4], sg[NE][4];
#pragma unroll
        for (int e = 0; e < NE; ++e)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (BLOCK) o[e][j] = in.o[e].get(j), g[e][j] = in.g[e].get(j);
                x[e][j] = in.x[e].get(j);
                up[e][j] = has_up ? in.up[e].get(j) : 0.0f;
                du[e][j] = has_du ? in.du[e].get(j) : 0.0f;
            }
        if (AHEAD && r0 + step < rows) load(r0 + step);
        // o becomes e = o r, x becomes e2 = x' r2
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < NE; ++e)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (BLOCK) {
                    o[e][j] *= r;
                    sg[e][j] = sigm(g[e][j]);
                    x[e][j] = fmaf(col(1, e, j), o[e][j] * col(0, e, j) * (g[e][j] * sg[e][j]), x[e][j]);
                }
                x[e][j] = p.w2 ? x[e][j] * r2 : 0.0f;
                s += j >= c.skip[e] ? col(2, e, j) * du[e][j] * x[e][j] : 0.0f;
            }
        const float m2 = lanes_sum<LPR>(s, red, 0) * inv_n;
        if constexpr (SHARED) asm volatile("" ::: "memory");   // the columns are read again, not kept
        s = 0.0f;
        X* dxp = row_at<X>(p.dx, row, p);
#pragma unroll
        for (int e = 0; e < NE; ++e) {
            float dg[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float dx = fmaf(r2, col(2, e, j) * du[e][j] - x[e][j] * m2, up[e][j]);
                acc[2][e][j] = fmaf(du[e][j], x[e][j], acc[2][e][j]);
                up[e][j] = dx;
                if constexpr (BLOCK) {
                    const float si = g[e][j] * sg[e][j], dxs = dx * si, dn = col(1, e, j) * dxs, ew = o[e][j] * col(0, e, j);
                    acc[0][e][j] = fmaf(dn, o[e][j], acc[0][e][j]);
                    acc[1][e][j] = fmaf(dxs, ew, acc[1][e][j]);
                    dg[j] = col(1, e, j) * dx * ew * fmaf(si, 1.0f - sg[e][j], sg[e][j]);
                    g[e][j] = col(0, e, j) * dn;   // v
                    s += j >= c.skip[e] ? g[e][j] * o[e][j] : 0.0f;
                }
            }
            if (live && c.on[e]) {
                vstore_own<X, 4>(dxp + c.n0[e], up[e], PACK ? c.skip[e] : 0);
                if constexpr (BLOCK) vstore_own<S, 4>(row_at<S>(p.dg, row, p) + c.n0[e], dg, PACK ? c.skip[e] : 0);
            }
        }
        if constexpr (BLOCK) {
            const float m = lanes_sum<LPR>(s, red, 1) * inv_n;
            S* dop = row_at<S>(p.d_o, row, p);
#pragma unroll
            for (int e = 0; e < NE; ++e) {
                float d[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) d[j] = r * (g[e][j] - o[e][j] * m);
                if (live && c.on[e]) vstore_own<S, 4>(dop + c.n0[e], d, PACK ? c.skip[e] : 0);
            }
        } else if constexpr (LPR > 64) {
            barrier_lds();
        }
    }
    float* part = p.part + (size_t)blockIdx.x * 3 * N;
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        if constexpr (RPW > 1) {
            __syncthreads();
#pragma unroll
            for (int e = 0; e < NE; ++e)
#pragma unroll
                for (int j = 0; j < 4; ++j) slots[threadIdx.x / LPR][(e * LPR + lane) * 4 + j] = acc[k][e][j];
            __syncthreads();
            if (threadIdx.x < LPR)
#pragma unroll
                for (int e = 0; e < NE; ++e)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        for (int q = 1; q < RPW; ++q) acc[k][e][j] += slots[q][(e * LPR + lane) * 4 + j];
        }
        if (threadIdx.x < LPR)
#pragma unroll
            for (int e = 0; e < NE; ++e)
                if (c.on[e]) vstore_own<float, 4>(part + (size_t)k * N + c.n0[e], acc[k][e], PACK ? c.skip[e] : 0);
    }
}

namespace {

bool in_registers(int N) { return N >= 4 && N <= 8192; }

// (lanes of a row, vectors of a lane): the fewest lanes that hold the row in two vectors; four where
// a wave or 512 lanes then do without more waves. Forward and backward of 33.5 million bf16 values
// in us, this plan's form and the next: N 64 66 + 102 with 16 lanes (192 + 293 with 64), N 128 63 +
// 106 with 16 x 2 (95 + 150 with 64), N 512 63 + 107 with 64 x 2 (115 + 156 with 256), N 1000 forward
// 61 with 64 x 4 (73 with 256), backward 112 with 256 (139 with 64 x 4, whose column sums leave no
// registers), N 2048 63 + 105 with 256 x 2 (71 + 101 with 512), N 4096 70 + 117 with 512 x 2 (68 + 146
// with 256 x 4), N 8192 101 + 137 (219 + 2243 as rows of any width).
struct RowPlan {
    int lanes, vecs, rpw;
};
RowPlan row_plan(int N, bool fwd) {
    RowPlan q{};
    if (N <= 64) q = {16, 1};
    else if (N <= 128) q = {16, 2};
    else if (N <= 256) q = {64, 1};
    else if (N <= 512) q = {64, 2};
    else if (N <= 1024) q = fwd ? RowPlan{64, 4} : RowPlan{256, 1};
    else if (N <= 2048) q = {256, 2};
    else if (N <= 4096) q = {512, 2};
    else q = {512, 4};
    q.rpw = q.lanes < 256 ? 256 / q.lanes : 1;
    return q;
}

// Workgroups of the backward, one set of column sums each: those that fit the GPU at once, each
// with its share of the rows (a second round of some of them leaves CUs idle: 32000 x 512 bf16, of
// which 768 fit: 50 us with 768, 59 with 1024).
constexpr int kMostParts = 1280;

long long row_groups(long long rows, int N) {
    if (!in_registers(N)) return rows;
    const int rpw = row_plan(N, false).rpw;
    return (rows + rpw - 1) / rpw;
}
int any_parts(long long rows) { return (int)std::min<long long>(rows, 512); }

int resident(const void* kernel, int block) {
    int per_cu = 0, dev = 0, cus = 0;
    if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&per_cu, kernel, block, 0) != hipSuccess || per_cu < 1) per_cu = 1;
    if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess)
        cus = 256;
    return std::min(per_cu * cus, kMostParts);
}

template <class S, class X, int LPR, int NE>
void run_fwd(const NormGate& p, hipStream_t stream) {
    const long long rows = (long long)p.R0 * p.R1;
    const int rpw = kRowBlock<LPR> / LPR;
    const dim3 grid((unsigned)std::min<long long>((rows + rpw - 1) / rpw, 4096)), block(kRowBlock<LPR>);
    if (p.h) hipLaunchKernelGGL((norm_gate_fwd_kernel<S, X, LPR, NE, kNormStep>), grid, block, 0, stream, p);
    else if (p.w) hipLaunchKernelGGL((norm_gate_fwd_kernel<S, X, LPR, NE, kNormBlock>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((norm_gate_fwd_kernel<S, X, LPR, NE, kNormOnly>), grid, block, 0, stream, p);
}

template <class S, class X, int LPR, int NE, bool BLOCK, bool PACK>
int run_bwd_k(const NormGate& p, hipStream_t stream) {
    static const int fit = resident((const void*)norm_gate_bwd_kernel<S, X, LPR, NE, BLOCK, PACK>, kRowBlock<LPR>);
    const int parts = (int)std::min<long long>(row_groups((long long)p.R0 * p.R1, p.N), fit);
    hipLaunchKernelGGL((norm_gate_bwd_kernel<S, X, LPR, NE, BLOCK, PACK>), dim3(parts), dim3(kRowBlock<LPR>), 0, stream, p);
    return parts;
}
template <class S, class X, int LPR, int NE>
int run_bwd(const NormGate& p, hipStream_t stream) {
    if (p.w) return p.x8.q ? run_bwd_k<S, X, LPR, NE, true, true>(p, stream) : run_bwd_k<S, X, LPR, NE, true, false>(p, stream);
    return p.x8.q ? run_bwd_k<S, X, LPR, NE, false, true>(p, stream) : run_bwd_k<S, X, LPR, NE, false, false>(p, stream);
}

// the workgroups of a backward (sets of column sums)
template <class S, class X>
int run_norm_gate(const NormGate& p, bool fwd, hipStream_t stream) {
    const long long rows = (long long)p.R0 * p.R1;
    if (!in_registers(p.N)) {
        if (fwd) {
            hipLaunchKernelGGL((norm_any_fwd_kernel<S, X>), dim3((unsigned)std::min<long long>(rows, kMostBlocks)), dim3(kNb), 0, stream, p);
            if (p.o8.q) launch_pack8({p.R0, p.R1, p.N, p.bf16, p.o, p.o8}, true, stream);
            if (p.g8.q) launch_pack8({p.R0, p.R1, p.N, p.bf16, p.g, p.g8}, true, stream);
            if (p.x8.q) launch_pack8({p.R0, p.R1, p.N, p.x_bf16, p.x, p.x8}, true, stream);
        } else {
            hipLaunchKernelGGL((norm_any_bwd_kernel<S, X>), dim3(any_parts(rows)), dim3(kNb), 0, stream, p);
        }
        return any_parts(rows);
    }
    const RowPlan q = row_plan(p.N, fwd);
    if (fwd) {
        if (q.lanes == 16) q.vecs == 1 ? run_fwd<S, X, 16, 1>(p, stream) : run_fwd<S, X, 16, 2>(p, stream);
        else if (q.lanes == 64) q.vecs == 1 ? run_fwd<S, X, 64, 1>(p, stream) : q.vecs == 2 ? run_fwd<S, X, 64, 2>(p, stream) : run_fwd<S, X, 64, 4>(p, stream);
        else if (q.lanes == 256) run_fwd<S, X, 256, 2>(p, stream);
        else q.vecs == 2 ? run_fwd<S, X, 512, 2>(p, stream) : run_fwd<S, X, 512, 4>(p, stream);
        return 0;
    }
    if (q.lanes == 16) return q.vecs == 1 ? run_bwd<S, X, 16, 1>(p, stream) : run_bwd<S, X, 16, 2>(p, stream);
    if (q.lanes == 64) return q.vecs == 1 ? run_bwd<S, X, 64, 1>(p, stream) : run_bwd<S, X, 64, 2>(p, stream);
    if (q.lanes == 256) return q.vecs == 1 ? run_bwd<S, X, 256, 1>(p, stream) : run_bwd<S, X, 256, 2>(p, stream);
    return q.vecs == 2 ? run_bwd<S, X, 512, 2>(p, stream) : run_bwd<S, X, 512, 4>(p, stream);
}

}  // namespace

size_t norm_gate_bwd_ws(long long rows, int N) {
    return (size_t)(in_registers(N) ? std::min<long long>(row_groups(rows, N), kMostParts) : any_parts(rows)) * 3 * N;
}

void launch_norm_gate(const NormGate& a, bool fwd, hipStream_t stream) {
    NormGate p = a;
    // without a gradient of u the second norm has no part in the backward (dw2 = 0)
    if (!fwd && !p.du.data) p.w2 = nullptr;
    // rows one pitch apart in every tensor need no division by R1
    p.flat = p.R0 == 1;
    if (!p.flat) {
        p.flat = 1;
        for (const delrec_rows* t : {&p.o, &p.g, &p.x, &p.dx_out, &p.du, &p.d_o, &p.dg, &p.dx})
            if (t->data && t->s0 != t->s1 * p.R1) p.flat = 0;
        if (p.R1 == 1) {
            p.flat = 1;
            for (delrec_rows* t : {&p.o, &p.g, &p.x, &p.dx_out, &p.du, &p.d_o, &p.dg, &p.dx}) t->s1 = t->s0;
            p.R1 = p.R0;
            p.R0 = 1;
        }
    }
    const int parts = !p.bf16 ? run_norm_gate<float, float>(p, fwd, stream)
                      : p.x_bf16 ? run_norm_gate<__bf16, __bf16>(p, fwd, stream)
                                 : run_norm_gate<__bf16, float>(p, fwd, stream);
    if (!fwd) launch_column_sums(p.part, parts, p.N, 3u * p.N, p.dw, p.dscale, p.dw2, stream);
}

}  // namespace delrec
