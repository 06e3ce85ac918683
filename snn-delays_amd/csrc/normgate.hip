// Norms around a residual block, fused with its gate and residual scale, over rows of N:
//     r = 1/sqrt(mean o^2 + eps), y = o r w silu(g), x' = x + scale y,
//     r2 = 1/sqrt(mean x'^2 + eps), u = x' r2 w2.
// Backwards, with e = o r, e2 = x' r2, v2 = w2 du and the row means <.>:
//     dx = dx' + r2 (v2 - e2 <v2 e2>),  dn = scale dx silu(g),  v = w dn,
//     do = r (v - e <v e>),  dg = scale dx e w silu'(g),
//     dw2 = sum du e2,  dscale = sum dx y,  dw = sum dn e       (sums over the rows).
#include "gated.h"
#include "kernels.h"

namespace delrec {

namespace {

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
    return (float)q.q[row * N + n] * q.scale[row * ((N + kGroup8 - 1) / kGroup8) + n / kGroup8];
}

}  // namespace

// the block's output at one position: o (or, in a step, the state's update), gate, residual
template <class S, class X>
__global__ void __launch_bounds__(kNb) norm_gate_fwd_kernel(NormGate p) {
    __shared__ float red[4];
    const long long row = blockIdx.x;
    const int N = p.N;
    const bool block = p.o.data || p.h;
    const X* x = row_ptr<const X>(p.x, row, p.R1);
    float r = 0.0f, r2 = 0.0f, s = 0.0f;
    if (p.h) {
        for (int n = threadIdx.x; n < N; n += kNb) {
            const float k = gate_in(to_f32(row_ptr<const S>(p.f, row, p.R1)[n]) + (p.bias ? p.bias[n] : 0.0f));
            const float h = p.h[row * N + n];
            p.h_out[row * N + n] = fmaf(k, to_f32(row_ptr<const S>(p.z, row, p.R1)[n]) - h, h);
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

template <class S, class X>
__global__ void __launch_bounds__(kNb) norm_gate_bwd_kernel(NormGate p) {
    __shared__ float red[4];
    const int N = p.N, tid = threadIdx.x;
    const bool block = p.w != nullptr;
    float* part = p.part + (size_t)blockIdx.x * 3 * N;
    for (int n = tid; n < 3 * N; n += kNb) part[n] = 0.0f;
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
            if (p.w2) part[2 * N + n] += duval(n) * e2val(n);
            if (block) {
                const float g = gval(n), sg = sigm(g), si = g * sg, e = oval(n) * r, dn = p.scale[n] * dx * si;
                part[n] += dn * e;
                part[N + n] += dx * e * p.w[n] * si;
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
__global__ void __launch_bounds__(1024) column_sums_kernel(const float* part, int rows, int N, int pitch, float* o0,
                                                           float* o1, float* o2) {
    __shared__ float red[16][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int n = blockIdx.x * 64 + lane, k = blockIdx.y;
    float* out = k == 0 ? o0 : (k == 1 ? o1 : o2);
    float s = 0.0f;
    if (n < N)
        for (int r = w; r < rows; r += 16) s += part[(size_t)r * pitch + (size_t)k * N + n];
    red[w][lane] = s;
    __syncthreads();
    if (w == 0 && n < N && out) {
        s = red[0][lane];
        for (int q = 1; q < 16; ++q) s += red[q][lane];
        out[n] = s;
    }
}

void launch_column_sums(const float* part, int rows, int N, int pitch, float* o0, float* o1, float* o2, hipStream_t stream) {
    hipLaunchKernelGGL(column_sums_kernel, dim3((N + 63) / 64, pitch / N), dim3(1024), 0, stream, part, rows, N, pitch, o0, o1, o2);
}

static int norm_gate_parts(long long rows) { return (int)(rows < 512 ? rows : 512); }
size_t norm_gate_bwd_ws(long long rows, int N) { return (size_t)norm_gate_parts(rows) * 3 * N; }

template <class S, class X>
static void launch_norm_gate_t(const NormGate& p, bool fwd, hipStream_t stream) {
    const long long rows = (long long)p.R0 * p.R1;
    if (fwd) hipLaunchKernelGGL((norm_gate_fwd_kernel<S, X>), dim3((unsigned)rows), dim3(kNb), 0, stream, p);
    else hipLaunchKernelGGL((norm_gate_bwd_kernel<S, X>), dim3(norm_gate_parts(rows)), dim3(kNb), 0, stream, p);
}

void launch_norm_gate(const NormGate& p, bool fwd, hipStream_t stream) {
    if (!p.bf16) launch_norm_gate_t<float, float>(p, fwd, stream);
    else if (p.x_bf16) launch_norm_gate_t<__bf16, __bf16>(p, fwd, stream);
    else launch_norm_gate_t<__bf16, float>(p, fwd, stream);
    if (fwd) {
        if (p.o8.q) launch_pack8({p.R0, p.R1, p.N, p.bf16, p.o, p.o8}, true, stream);
        if (p.g8.q) launch_pack8({p.R0, p.R1, p.N, p.bf16, p.g, p.g8}, true, stream);
        if (p.x8.q) launch_pack8({p.R0, p.R1, p.N, p.x_bf16, p.x, p.x8}, true, stream);
    } else {
        launch_column_sums(p.part, norm_gate_parts((long long)p.R0 * p.R1), p.N, 3 * p.N, p.dw, p.dscale, p.dw2, stream);
    }
}

}  // namespace delrec
