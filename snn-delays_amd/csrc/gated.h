// Shared device helpers of the gated-recurrence block's kernels (gated.hip, normgate.hip,
// pack8.hip): element types, the gate, the 8-bit groups.
#pragma once

#include <type_traits>

#include "common.h"

namespace delrec {

// Workgroups of a launch of up to 1024 threads each: a dimension has room for 2^32 threads. Kernels
// loop, or are launched again, over what is left.
constexpr int kMostBlocks = 1 << 20;

// activations: float, or bf16 by the hardware's round to nearest even
template <class S>
__device__ __forceinline__ float to_f32(S v) { return (float)v; }

// The gate k = sigmoid(-x) = 1 / (1 + e^x), as a factor of products.
constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float gate_in(float x) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * kLog2e));
}

// The recurrence needs the gate k and the leak a = 1 - k, each to its last digits: the one near 1
// comes from the other, which must not come from it. So the smaller of the two is kept, with its
// sign to say which: m = k where k <= a, m = -a elsewhere. From y = (f + bias) log2(e), with e =
// 2^-|y|, it is e / (1 + e), through the hardware's 2^y and reciprocal (about 1 ulp each; f and the
// bias are scaled apart, whose roundings add 6e-8 (|f + bias| + |bias|) relative). +0: nothing comes
// in, -0: nothing stays. With the leak as 1 - k, which is off by 1 % of itself at f + bias = -12 and
// gone at -17, the scan's kernels take 1 to 3 % less, with 8 bits 4 to 7 % (T1024 B64 N2048: 272 and
// 252 us instead of 283 and 269).
__device__ __forceinline__ float gate_small2(float y) {
    const float e = __builtin_amdgcn_exp2f(-fabsf(y));
    return copysignf(e * __builtin_amdgcn_rcpf(1.0f + e), y);
}
__device__ __forceinline__ bool leak_kept(float m) { return __float_as_int(m) < 0; }
// a x (-0: the summand that changes no product, its sign included)
__device__ __forceinline__ float leak_times(float m, float x) { return fmaf(-m, x, leak_kept(m) ? -0.0f : x); }
// the state after a step, a h + k z, from d = h - z
__device__ __forceinline__ float gate_step(float m, float d, float h, float z) { return fmaf(-m, d, leak_kept(m) ? z : h); }

// V consecutive activations of a row, at any alignment of the element (rows of odd width start
// anywhere): one access of up to 16 bytes
template <class S, int V>
struct Vec {
    typedef S type __attribute__((ext_vector_type(V)));
    typedef type unaligned __attribute__((aligned(sizeof(S))));
    type v;
    __device__ __forceinline__ float get(int j) const { return (float)v[j]; }
    // get(j) c + b, rounded once
    __device__ __forceinline__ float get_fma(int j, float c, float b) const { return fmaf(get(j), c, b); }
};
template <class S>
struct Vec<S, 1> {
    S v;
    __device__ __forceinline__ float get(int) const { return (float)v; }
    __device__ __forceinline__ float get_fma(int, float c, float b) const { return fmaf((float)v, c, b); }
};

template <class S, int V>
__device__ __forceinline__ Vec<S, V> vload(const S* p) {
    Vec<S, V> r;
    if constexpr (V > 1) r.v = *(const typename Vec<S, V>::unaligned*)p;
    else r.v = *p;
    return r;
}
template <class S, int V>
__device__ __forceinline__ void vstore(S* p, const float* x) {
    if constexpr (V > 1) {
        typename Vec<float, V>::type t;
#pragma unroll
        for (int j = 0; j < V; ++j) t[j] = x[j];
        *(typename Vec<S, V>::unaligned*)p = __builtin_convertvector(t, typename Vec<S, V>::type);
    } else {
        *p = (S)x[0];
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
// fl(1 / scale): one Newton step from the hardware's reciprocal (within 1 ulp) rounds correctly
// (Markstein), the all-ones mantissa aside; scales and reciprocals here are normal numbers.
__device__ __forceinline__ float recip8(float scale) {
    const float r = __builtin_amdgcn_rcpf(scale);
    return fmaf(fmaf(-scale, r, 1.0f), r, r);
}
// rint(v inv) in the low byte: |v inv| < 127.5, and at 1.5 * 2^23 a unit is the last place
__device__ __forceinline__ uint32_t quant8(float v, float inv) {
    return __float_as_uint(v * inv + 12582912.0f);
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
    if constexpr (V <= 2) step(__shfl_xor((int)m, 16, kWave));
    if constexpr (V == 1) step(__shfl_xor((int)m, 32, kWave));
    return m;
}
__device__ __forceinline__ float scale8_bits(uint32_t m) {
    return scale8(__uint_as_float(m), m < 0x7f800000u);
}

// A row's 8-bit columns are stored at a pitch of N rounded up to 4, so that a lane's V own columns
// (from its nominal column i on) are one aligned access, also in a row's last lane, whose values
// start `skip` columns before its own.
__host__ __device__ __forceinline__ int pitch8(int N) { return (N + 3) & ~3; }

template <int V>
struct Lane8 {
    uint32_t mask[V];              // of the bits of a magnitude: own columns only
    int at, shift;                 // first own column (clamped in lanes without one), 8 skip
    bool on;
    __device__ __forceinline__ Lane8(int i, int skip, bool on_, int N) : on(on_) {
#pragma unroll
        for (int j = 0; j < V; ++j) mask[j] = on && j >= skip ? 0x7fffffffu : 0u;
        at = on ? i : pitch8(N) - V;
        shift = on ? 8 * skip : 0;
    }
};

template <int V>
struct Word8 {
    typedef typename std::conditional<V == 4, uint32_t, typename std::conditional<V == 2, uint16_t, uint8_t>::type>::type type;
};

// the lane's V values as 8 bits, own columns from the low byte on, and their group's scale. The 64
// columns of a group lie on 64 / V neighbouring lanes; all lanes of the wave call it.
template <int V>
__device__ __forceinline__ uint32_t quantise8(const float* x, const Lane8<V>& ln, float* scale) {
    uint32_t m = 0, word, b[V];
#pragma unroll
    for (int j = 0; j < V; ++j) m = max(m, __float_as_uint(x[j]) & ln.mask[j]);
    *scale = scale8_bits(group_umax<V>(m));
    const float inv = recip8(*scale);
#pragma unroll
    for (int j = 0; j < V; ++j) b[j] = quant8(x[j], inv);
    if constexpr (V == 4)
        word = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400) | __builtin_amdgcn_perm(b[3], b[2], 0x04000c0c);
    else if constexpr (V == 2) word = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400);
    else word = b[0];
    return word >> ln.shift;
}
// and stored: own columns, the scale by the group's first lane (`first`)
template <int V>
__device__ __forceinline__ void store8(const float* x, const Lane8<V>& ln, bool first, int8_t* qrow, float* scale) {
    float sc;
    const uint32_t word = quantise8<V>(x, ln, &sc);
    if (ln.on) *(typename Word8<V>::type*)(qrow + ln.at) = (typename Word8<V>::type)word;
    if (first) *scale = sc;
}

// V columns from their 8 bits, by the scale of the lane's own group; columns before its own come as
// zeros (a lane must not store what it computes of them).
template <int V>
struct Vec8 {
    uint32_t q;
    float scale;
    __device__ __forceinline__ float whole(int j) const { return (float)((int32_t)(q << (24 - 8 * j)) >> 24); }
    __device__ __forceinline__ float get(int j) const { return whole(j) * scale; }
    __device__ __forceinline__ float get_fma(int j, float c, float b) const { return fmaf(whole(j), scale * c, b); }
};
template <int V>
__device__ __forceinline__ Vec8<V> load8(const int8_t* qrow, const float* scale, const Lane8<V>& ln) {
    Vec8<V> r;
    r.q = (uint32_t)*(const typename Word8<V>::type*)(qrow + ln.at) << ln.shift;
    r.scale = *scale;
    return r;
}

// V results of a lane, without the first `skip`
template <class S, int V>
__device__ __forceinline__ void vstore_own(S* p, const float* x, int skip) {
    if (skip == 0) {
        vstore<S, V>(p, x);
    } else {
#pragma unroll
        for (int j = 1; j < V; ++j)
            if (j >= skip) p[j] = (S)x[j];
    }
}

}  // namespace delrec
