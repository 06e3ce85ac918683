// A (rows, N) tensor to 8 bits and back: groups of 64 columns of a row share one 32-bit scale,
//     scale = max(amax / 127, 2^-126), q = rint(x / scale), x^ = q scale.
#include "gated.h"
#include "kernels.h"

namespace delrec {

template <class S>
__global__ void __launch_bounds__(256) pack8_kernel(Pack8 p) {
    const int lane = threadIdx.x & 63;
    const long long grp = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int ng = (p.N + kGroup8 - 1) / kGroup8;
    if (grp >= (long long)p.R0 * p.R1 * ng) return;
    const long long row = grp / ng;
    const int n = (int)(grp % ng) * kGroup8 + lane;
    const S* x = (const S*)p.x.data + (row / p.R1) * p.x.s0 + (row % p.R1) * p.x.s1;
    const float v = n < p.N ? to_f32(x[n]) : 0.0f;
    float m = fabsf(v);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, kWave));
    const float sc = scale8(m, __all(finite8(v)));
    if (n < p.N) p.p.q[row * p.N + n] = (int8_t)quant8(v, 1.0f / sc);
    if (lane == 0) p.p.scale[grp] = sc;
}

template <class S>
__global__ void __launch_bounds__(256) unpack8_kernel(Pack8 p) {
    const int ng = (p.N + kGroup8 - 1) / kGroup8;
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= (long long)p.R0 * p.R1 * p.N) return;
    const long long row = i / p.N;
    const int n = (int)(i % p.N);
    S* x = (S*)p.x.data + (row / p.R1) * p.x.s0 + (row % p.R1) * p.x.s1;
    x[n] = (S)((float)p.p.q[i] * p.p.scale[row * ng + n / kGroup8]);
}

void launch_pack8(const Pack8& p, bool pack, hipStream_t stream) {
    const long long rows = (long long)p.R0 * p.R1;
    if (pack) {
        const unsigned g = (unsigned)((rows * ((p.N + kGroup8 - 1) / kGroup8) + 3) / 4);
        if (p.bf16) hipLaunchKernelGGL(pack8_kernel<__bf16>, dim3(g), dim3(256), 0, stream, p);
        else hipLaunchKernelGGL(pack8_kernel<float>, dim3(g), dim3(256), 0, stream, p);
    } else {
        const unsigned g = (unsigned)((rows * p.N + 255) / 256);
        if (p.bf16) hipLaunchKernelGGL(unpack8_kernel<__bf16>, dim3(g), dim3(256), 0, stream, p);
        else hipLaunchKernelGGL(unpack8_kernel<float>, dim3(g), dim3(256), 0, stream, p);
    }
}

}  // namespace delrec
