// Gated linear recurrence over (T, B, N) sequences and its reverse pass.
//     k_t = sigmoid(-(f_t + bias)), h_t = h_{t-1} + k_t (z_t - h_{t-1})
// backwards, with lam_t = dh_t + c_{t+1} and c_t = (1 - k_t) lam_t (c_T = dlast):
//     dz_t = lam_t k_t, df_t = lam_t k_t (1 - k_t) (h_{t-1} - z_t), dh0 = c_0, db = sum df.
// The state before every 64th step is kept by the forward; the backward recomputes those between.
#include "gated.h"
#include "kernels.h"

namespace delrec {

namespace {
constexpr int kBlk = DELREC_GATED_BLOCK;
}

__device__ __forceinline__ int row_length(const GatedScan& p, int b) {
    if (!p.lengths) return p.T;
    const int64_t v = p.lengths[b];
    return v < 0 ? 0 : (v < p.T ? (int)v : p.T);
}

template <class S>
__global__ void __launch_bounds__(256) gated_fwd_kernel(GatedScan p) {
    const long long c = (long long)blockIdx.x * 256 + threadIdx.x;
    if (c >= (long long)p.B * p.N) return;
    const int b = (int)(c / p.N), n = (int)(c % p.N);
    const S* z = (const S*)p.z.data + b * p.z.s1 + n;
    const S* f = (const S*)p.f.data + b * p.f.s1 + n;
    S* y = (S*)p.h.data + b * p.h.s1 + n;
    const float bias = p.bias ? p.bias[n] : 0.0f;
    const int len = row_length(p, b);
    float h = p.h0 ? p.h0[c] : 0.0f;
    for (int t = 0; t < p.T; ++t) {
        if (p.states && t % kBlk == 0) p.states[(size_t)(t / kBlk) * p.B * p.N + c] = h;
        float out = 0.0f;
        if (t < len) {
            if (p.starts && p.starts[(size_t)t * p.B + b]) h = 0.0f;
            const float k = gate_in(to_f32(f[t * p.f.s0]) + bias);
            h = fmaf(k, to_f32(z[t * p.z.s0]) - h, h);
            out = h;
        }
        y[t * p.h.s0] = (S)out;
    }
    p.h_last[c] = h;
}

// z, f of step t, row b, channel n: as given, or from the 8 bits kept of them
template <class S>
__device__ __forceinline__ float read8(const delrec_rows& x, const delrec_packed8& q, int t, int b, int n, int B, int N) {
    if (!q.q) return to_f32(((const S*)x.data)[t * x.s0 + b * x.s1 + n]);
    const size_t row = (size_t)t * B + b;
    return (float)q.q[row * N + n] * q.scale[row * ((N + kGroup8 - 1) / kGroup8) + n / kGroup8];
}

template <class S>
__global__ void __launch_bounds__(64) gated_bwd_kernel(GatedScan p) {
    __shared__ float before[kBlk][64];
    const long long c = (long long)blockIdx.x * 64 + threadIdx.x;
    if (c >= (long long)p.B * p.N) return;
    const int b = (int)(c / p.N), n = (int)(c % p.N), B = p.B, N = p.N;
    const float bias = p.bias ? p.bias[n] : 0.0f;
    const int len = row_length(p, b);
    const S* dh = (const S*)p.dh.data + b * p.dh.s1 + n;
    S* dz = (S*)p.dz.data + b * p.dz.s1 + n;
    S* df = (S*)p.df.data + b * p.df.s1 + n;
    float carry = p.dlast ? p.dlast[c] : 0.0f, db = 0.0f;
    for (int t0 = (p.T - 1) / kBlk * kBlk; t0 >= 0; t0 -= kBlk) {
        const int t1 = min(t0 + kBlk, p.T);
        float h = p.states[(size_t)(t0 / kBlk) * B * N + c];
        for (int t = t0; t < min(t1, len); ++t) {
            if (p.starts && p.starts[(size_t)t * B + b]) h = 0.0f;
            before[t - t0][threadIdx.x] = h;
            const float k = gate_in(read8<S>(p.f, p.f8, t, b, n, B, N) + bias);
            h = fmaf(k, read8<S>(p.z, p.z8, t, b, n, B, N) - h, h);
        }
        for (int t = t1 - 1; t >= t0; --t) {
            float oz = 0.0f, of = 0.0f;
            if (t < len) {
                const float k = gate_in(read8<S>(p.f, p.f8, t, b, n, B, N) + bias);
                const float z = read8<S>(p.z, p.z8, t, b, n, B, N);
                const float lam = to_f32(dh[t * p.dh.s0]) + carry;
                oz = lam * k;
                of = oz * (1.0f - k) * (before[t - t0][threadIdx.x] - z);
                carry = p.starts && p.starts[(size_t)t * B + b] ? 0.0f : lam * (1.0f - k);
                db += of;
            }
            dz[t * p.dz.s0] = (S)oz;
            df[t * p.df.s0] = (S)of;
        }
    }
    if (p.dh0) p.dh0[c] = carry;
    if (p.db) p.ws[c] = db;
}

size_t gated_fwd_ws(int, int, int) { return 0; }
size_t gated_bwd_ws(int, int B, int N) { return (size_t)B * N; }

void launch_gated_fwd(const GatedScan& p, hipStream_t stream) {
    const unsigned g = (unsigned)(((long long)p.B * p.N + 255) / 256);
    if (p.bf16) hipLaunchKernelGGL(gated_fwd_kernel<__bf16>, dim3(g), dim3(256), 0, stream, p);
    else hipLaunchKernelGGL(gated_fwd_kernel<float>, dim3(g), dim3(256), 0, stream, p);
    if (p.z8.q) {
        launch_pack8({p.T, p.B, p.N, p.bf16, p.z, p.z8}, true, stream);
        launch_pack8({p.T, p.B, p.N, p.bf16, p.f, p.f8}, true, stream);
    }
}

void launch_gated_bwd(const GatedScan& p, hipStream_t stream) {
    const unsigned g = (unsigned)(((long long)p.B * p.N + 63) / 64);
    if (p.bf16) hipLaunchKernelGGL(gated_bwd_kernel<__bf16>, dim3(g), dim3(64), 0, stream, p);
    else hipLaunchKernelGGL(gated_bwd_kernel<float>, dim3(g), dim3(64), 0, stream, p);
    if (p.db) launch_column_sums(p.ws, p.B, p.N, p.N, p.db, nullptr, nullptr, stream);
}

}  // namespace delrec
