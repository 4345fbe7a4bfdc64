// Activations of the fused GEMM epilogues, fp32 in and out.
//
// Each is written in the form that keeps its relative accuracy where the result is small (a sum like 1 + erf(v) or 1 + tanh(u)
// cancels there): gelu through erfc, the tanh form as v * sigmoid(2u) = v / (1 + exp(-2u)).  NaN stays NaN and infinities follow
// the formulas: silu and the tanh form of -inf are -inf / inf = NaN.
#pragma once

#include "common.cuh"

namespace hkb {

inline bool act_known(int act) { return act >= HKB_ACT_NONE && act <= HKB_ACT_SILU; }

// v / (1 + exp(-z)), for negative z as v * exp(z) / (1 + exp(z)): exp(-z) itself overflows while the quotient is still a normal
// number, and the denominator stays in [1, 2], where __fdividef is good to 2 ulp.  __expf loses |z| * 2^-24 of its result.
__device__ __forceinline__ float times_sigmoid(float v, float z) {
    const float t = __expf(-fabsf(z));
    return __fdividef(z >= 0.0f ? v : v * t, 1.0f + t);
}

__device__ __forceinline__ float act_relu(float v) { return v < 0.0f ? 0.0f : v; }
__device__ __forceinline__ float act_gelu(float v) { return 0.5f * v * erfcf(-0.70710678118654752f * v); }
__device__ __forceinline__ float act_gelu_tanh(float v) {
    // 2 * sqrt(2 / pi) * (v + 0.044715 v^3)
    return times_sigmoid(v, v * __fmaf_rn(0.0713548162726f, v * v, 1.59576912160573f));
}
__device__ __forceinline__ float act_silu(float v) { return times_sigmoid(v, v); }

// NV values through the same activation: one branch for all of them (`act` is uniform over the launch).
template <int NV>
__device__ __forceinline__ void apply_act(float* v, int act) {
    if (act == HKB_ACT_RELU) {
#pragma unroll
        for (int j = 0; j < NV; ++j) v[j] = act_relu(v[j]);
    } else if (act == HKB_ACT_GELU) {
#pragma unroll
        for (int j = 0; j < NV; ++j) v[j] = act_gelu(v[j]);
    } else if (act == HKB_ACT_GELU_TANH) {
#pragma unroll
        for (int j = 0; j < NV; ++j) v[j] = act_gelu_tanh(v[j]);
    } else if (act == HKB_ACT_SILU) {
#pragma unroll
        for (int j = 0; j < NV; ++j) v[j] = act_silu(v[j]);
    }
}

}  // namespace hkb
