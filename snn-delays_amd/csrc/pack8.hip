// A (rows, N) tensor to 8 bits and back: groups of 64 columns of a row share one 32-bit scale,
//     scale = max(amax / 127, 2^-126), q = rint(x / scale), x^ = q scale.
#include <algorithm>

#include "gated.h"
#include "kernels.h"

namespace delrec {

// one to three columns (one group): a wave a row
template <class S>
__global__ void __launch_bounds__(256) pack8_any_kernel(Pack8 p) {
    const int lane = threadIdx.x & 63;
    const long long rows = (long long)p.R0 * p.R1;
    for (long long row = blockIdx.x * 4LL + (threadIdx.x >> 6); row < rows; row += gridDim.x * 4LL) {
        const S* x = (const S*)p.x.data + (row / p.R1) * p.x.s0 + (row % p.R1) * p.x.s1;
        const float v = lane < p.N ? to_f32(x[lane]) : 0.0f;
        float m = fabsf(v);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, kWave));
        const float sc = scale8(m, __all(finite8(v)));
        if (lane < p.N) p.p.q[row * pitch8(p.N) + lane] = (int8_t)quant8(v, recip8(sc));
        if (lane == 0) p.p.scale[row] = sc;
    }
}

template <class S>
__global__ void __launch_bounds__(256) unpack8_any_kernel(Pack8 p) {
    const long long all = (long long)p.R0 * p.R1 * p.N;
    for (long long i = blockIdx.x * 256LL + threadIdx.x; i < all; i += gridDim.x * 256LL) {
        const long long row = i / p.N;
        const int n = (int)(i % p.N);
        S* x = (S*)p.x.data + (row / p.R1) * p.x.s0 + (row % p.R1) * p.x.s1;
        x[n] = (S)((float)p.p.q[row * pitch8(p.N) + n] * p.p.scale[row]);
    }
}

// Rows of four columns and more: LPR lanes a row, four columns a lane (16 lanes a group), kRows
// rows at once so that their loads are in flight together. The last lane of a row whose width is
// no multiple of 4 is moved back to end with it.
namespace {
constexpr int kRows = 4;

__device__ __forceinline__ long long row_offset(const Pack8& p, long long row) {
    if (p.R0 == 1) return row * p.x.s1;
    if (p.R1 == 1) return row * p.x.s0;
    const unsigned r = (unsigned)row, i = r / (unsigned)p.R1;
    return i * p.x.s0 + (r - i * (unsigned)p.R1) * p.x.s1;
}
}  // namespace

template <class S, int LPR, bool PACK>
__global__ void __launch_bounds__(256) pack8_kernel(Pack8 p) {
    constexpr int RPW = 256 / LPR;
    const int N = p.N, ng = (N + kGroup8 - 1) / kGroup8;
    const int i = (blockIdx.x * LPR + threadIdx.x % LPR) * 4, n0 = min(i, N - 4), group = min(i, N - 1) / kGroup8;
    const bool on = i < N, first = on && i % kGroup8 == 0;
    const long long rows = (long long)p.R0 * p.R1;
    for (long long r0 = (long long)blockIdx.y * RPW * kRows; r0 < rows; r0 += (long long)gridDim.y * RPW * kRows) {
        // rows past the end repeat the last one and store nothing
        long long row[kRows];
        bool live[kRows];
#pragma unroll
        for (int q = 0; q < kRows; ++q) {
            const long long mine = r0 + q * RPW + threadIdx.x / LPR;
            live[q] = mine < rows && on;
            row[q] = mine < rows ? mine : rows - 1;
        }
        if constexpr (PACK) {
            Vec<S, 4> v[kRows];
#pragma unroll
            for (int q = 0; q < kRows; ++q) v[q] = vload<S, 4>((const S*)p.x.data + row_offset(p, row[q]) + n0);
#pragma unroll
            for (int q = 0; q < kRows; ++q) {
                float x[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] = v[q].get(j);
                store8<4>(x, Lane8<4>(i, i - n0, live[q], N), live[q] && first, p.p.q + row[q] * pitch8(N), p.p.scale + row[q] * ng + group);
            }
        } else {
            Vec8<4> v[kRows];
#pragma unroll
            for (int q = 0; q < kRows; ++q) v[q] = load8<4>(p.p.q + row[q] * pitch8(N), p.p.scale + row[q] * ng + group, Lane8<4>(i, i - n0, on, N));
#pragma unroll
            for (int q = 0; q < kRows; ++q) {
                float x[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] = v[q].get(j);
                if (live[q]) vstore_own<S, 4>((S*)p.x.data + row_offset(p, row[q]) + n0, x, i - n0);
            }
        }
    }
}

// The fewest lanes, 16, 64 or 256, that hold a row's groups: packing and unpacking of 33.5 million bf16
// values take 20 + 16 us so; N 64 with 64 lanes 52 + 36, N 256 with 256 40 + 25 and with 16 22 + 21,
// N 2048 with 64 21 + 18.
template <class S, bool PACK>
static void run_pack8(const Pack8& p, hipStream_t stream) {
    const long long rows = (long long)p.R0 * p.R1;
    const int lanes = (p.N + kGroup8 - 1) / kGroup8 * (kGroup8 / 4);
    auto grid = [&](int lpr) {
        const int per = 256 / lpr * kRows;
        return dim3((lanes + lpr - 1) / lpr, (unsigned)std::min<long long>((rows + per - 1) / per, 16384));
    };
    if (lanes <= 16) hipLaunchKernelGGL((pack8_kernel<S, 16, PACK>), grid(16), dim3(256), 0, stream, p);
    else if (lanes <= 64) hipLaunchKernelGGL((pack8_kernel<S, 64, PACK>), grid(64), dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((pack8_kernel<S, 256, PACK>), grid(256), dim3(256), 0, stream, p);
}

template <class S>
static void run_pack8_any(const Pack8& p, bool pack, hipStream_t stream) {
    const long long rows = (long long)p.R0 * p.R1;
    if (p.N >= 4) return pack ? run_pack8<S, true>(p, stream) : run_pack8<S, false>(p, stream);
    if (pack) hipLaunchKernelGGL(pack8_any_kernel<S>, dim3((unsigned)std::min<long long>((rows + 3) / 4, kMostBlocks)), dim3(256), 0, stream, p);
    else hipLaunchKernelGGL(unpack8_any_kernel<S>, dim3((unsigned)std::min<long long>((rows * p.N + 255) / 256, kMostBlocks)), dim3(256), 0, stream, p);
}

void launch_pack8(const Pack8& p, bool pack, hipStream_t stream) {
    if (p.bf16) run_pack8_any<__bf16>(p, pack, stream);
    else run_pack8_any<float>(p, pack, stream);
}

}  // namespace delrec
