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

}  // namespace delrec
