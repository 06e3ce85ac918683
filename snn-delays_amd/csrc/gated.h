// Shared device helpers of the gated-recurrence block's kernels (gated.hip, normgate.hip,
// pack8.hip): element types, the gate, the 8-bit groups.
#pragma once

#include "common.h"

namespace delrec {

typedef float gf4 __attribute__((ext_vector_type(4)));
typedef __bf16 gb4 __attribute__((ext_vector_type(4)));

// activations: float, or bf16 by the hardware's round to nearest even
template <class S>
__device__ __forceinline__ float to_f32(S v) { return (float)v; }

// k = sigmoid(-x) = 1 / (1 + e^x), through the hardware's 2^x and reciprocal (about 1 ulp each;
// the product x log2(e) adds 6e-8 |x| relative). k is computed by itself and not as 1 - a: at a
// leak near 1 that difference would lose the small k's digits.
__device__ __forceinline__ float gate_in(float x) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * 1.4426950408889634f));
}

// V consecutive activations of a row, at any alignment of the element (rows of odd width start
// anywhere): one 8- or 16-byte access for V = 4
typedef gf4 gf4u __attribute__((aligned(4)));
typedef gb4 gb4u __attribute__((aligned(2)));

template <class S, int V>
struct Vec {                       // V values as loaded
    S v[V];
    __device__ __forceinline__ float get(int j) const { return (float)v[j]; }
};
template <>
struct Vec<float, 4> {
    gf4 v;
    __device__ __forceinline__ float get(int j) const { return v[j]; }
};
template <>
struct Vec<__bf16, 4> {
    gb4 v;
    __device__ __forceinline__ float get(int j) const { return (float)v[j]; }
};

template <class S, int V>
__device__ __forceinline__ Vec<S, V> vload(const S* p) {
    Vec<S, V> r;
    if constexpr (V == 4 && sizeof(S) == 4) r.v = *(const gf4u*)p;
    else if constexpr (V == 4) r.v = *(const gb4u*)p;
    else
#pragma unroll
        for (int j = 0; j < V; ++j) r.v[j] = p[j];
    return r;
}
template <class S, int V>
__device__ __forceinline__ void vstore(S* p, const float* x) {
    if constexpr (V == 4) {
        const gf4 t = {x[0], x[1], x[2], x[3]};
        if constexpr (sizeof(S) == 4) *(gf4u*)p = t;
        else *(gb4u*)p = __builtin_convertvector(t, gb4);
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) p[j] = (S)x[j];
    }
}

// ---- 8-bit groups of 64 columns ----
constexpr int kGroup8 = DELREC_PACK8_GROUP;
constexpr float kInv127 = 1.0f / 127.0f;
constexpr float kMinScale8 = 0x1p-126f;

// a group's scale from its largest magnitude (NaN or infinite: NaN)
__device__ __forceinline__ float scale8(float amax, bool finite) {
    return finite ? fmaxf(amax * kInv127, kMinScale8) : __builtin_nanf("");
}
__device__ __forceinline__ bool finite8(float v) { return fabsf(v) < __builtin_inff(); }
// inv = 1 / scale rounded; |v| <= amax, so |v inv| < 127.5
__device__ __forceinline__ int quant8(float v, float inv) {
    const float q = rintf(v * inv);
    return q == q ? (int)q : 0;
}


// largest |bits| over the 64 / V lanes that hold a group: as unsigned numbers the bit patterns of
// magnitudes are in their order, infinities and NaN above all finite ones
template <int V>
__device__ __forceinline__ uint32_t group_umax(uint32_t m) {
    auto step = [&](int o) { m = max(m, (uint32_t)o); };
    step(__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xF, 0xF, false));
    step(__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xF, 0xF, false));
    step(__builtin_amdgcn_update_dpp(0, (int)m, 0x141, 0xF, 0xF, false));
    step(__builtin_amdgcn_update_dpp(0, (int)m, 0x140, 0xF, 0xF, false));
    if constexpr (V == 1) {
        step(__shfl_xor((int)m, 16, kWave));
        step(__shfl_xor((int)m, 32, kWave));
    }
    return m;
}
__device__ __forceinline__ float scale8_bits(uint32_t m) {
    return scale8(__uint_as_float(m), m < 0x7f800000u);
}

// V columns of a row whose 8-bit groups lie on the lanes in order: the lane's V values x (columns
// n0 .. n0 + V - 1, of which the first `skip` belong to the lane before, and all do when skip = V)
// go to q, the group's scale to *scale by its first lane. All lanes of the wave call it.
template <int V>
__device__ __forceinline__ void store8(const float* x, int skip, bool first, int8_t* q, float* scale) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) m = max(m, j >= skip ? __float_as_uint(x[j]) & 0x7fffffffu : 0u);
    const float sc = scale8_bits(group_umax<V>(m)), inv = 1.0f / sc;
    int b[V];
#pragma unroll
    for (int j = 0; j < V; ++j) b[j] = quant8(x[j], inv);
    if (V == 4 && skip == 0) {
        typedef uint32_t u32u __attribute__((aligned(1)));
        *(u32u*)q = (b[0] & 255) | (b[1] & 255) << 8 | (b[2 % V] & 255) << 16 | (uint32_t)b[3 % V] << 24;
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (j >= skip) q[j] = (int8_t)b[j];
    }
    if (first) *scale = sc;
}

// V columns from their 8 bits. A row's last lane may start in the group before its own (its
// columns are moved back to the row's end): both groups' scales.
template <int V>
struct Vec8 {
    uint32_t q;
    float s0, s1;
    int cut;                       // columns of the first group
    __device__ __forceinline__ float get(int j) const {
        return (float)((int32_t)(q << (24 - 8 * j)) >> 24) * (j < cut ? s0 : s1);
    }
};
template <int V>
__device__ __forceinline__ Vec8<V> load8(const delrec_packed8& p, size_t row, int n0, int N, int ng) {
    Vec8<V> r;
    const int8_t* q = p.q + row * N + n0;
    if constexpr (V == 4) {
        typedef uint32_t u32u __attribute__((aligned(1)));
        r.q = *(const u32u*)q;
    } else {
        r.q = (uint8_t)q[0];
    }
    const int g0 = n0 / kGroup8, g1 = (n0 + V - 1) / kGroup8;
    r.s0 = p.scale[row * ng + g0];
    r.s1 = p.scale[row * ng + g1];
    r.cut = g1 > g0 ? g1 * kGroup8 - n0 : V;
    return r;
}

}  // namespace delrec
