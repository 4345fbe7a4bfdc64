// Activations of the fused GEMM epilogues, fp32 in and out.
//
// Each is written in the form that keeps its relative accuracy where the result is small (a sum like 1 + erf(v) or 1 + tanh(u)
// cancels there): gelu through erfc, the tanh form as v * sigmoid(2u) = v / (1 + exp(-2u)).  NaN stays NaN and infinities follow
// the formulas: silu and both forms of gelu of -inf are -inf * 0 = NaN.
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
// v * Phi(v), two values at a time on the packed fp32 pipe.  For a = |v|, Phi(-a) = erfc(a / sqrt 2) / 2 = exp(-a^2 / 2) t P(t) with
// t = 1 / (1 + 0.36 a): the scaled function is smooth in t on (0, 1], and P, of degree 6, is a minimax fit of its relative error over
// 0 <= a <= 14 (8.7e-7; with the roundings 2^-19.5 for a <= 3, 2^-18.7 for a <= 6, 2^-17 at 13, where the exponent's argument rounds).
// 2000 x 14336 x 4096 with bias, us: this 98, erfcf() 118 (its 50 instructions per value outlast the main loop), no activation 95.
__device__ __forceinline__ float2 act_gelu2(float2 v) {
    const float2 a = make_float2(fabsf(v.x), fabsf(v.y));
    const float2 d = __ffma2_rn(a, make_float2(0.36f, 0.36f), make_float2(1.0f, 1.0f));
    float2 t, e;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t.x) : "f"(d.x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t.y) : "f"(d.y));
    auto c2 = [](float c) { return make_float2(c, c); };
    float2 q = __ffma2_rn(c2(4.705620929598808e-2f), t, c2(-1.7976443469524384e-1f));
    q = __ffma2_rn(q, t, c2(1.8095368146896362e-1f));
    q = __ffma2_rn(q, t, c2(2.6549549773335457e-2f));
    q = __ffma2_rn(q, t, c2(1.397191882133484e-1f));
    q = __ffma2_rn(q, t, c2(1.4177246391773224e-1f));
    q = __ffma2_rn(q, t, c2(1.4371304214000702e-1f));
    const float2 x = __fmul2_rn(__fmul2_rn(v, v), c2(-0.72134752044448170f));            // -a^2 / 2 in powers of two
    asm("ex2.approx.f32 %0, %1;" : "=f"(e.x) : "f"(x.x));
    asm("ex2.approx.f32 %0, %1;" : "=f"(e.y) : "f"(x.y));
    q = __fmul2_rn(__fmul2_rn(q, t), e);
    return __fmul2_rn(v, make_float2(v.x >= 0.0f ? 1.0f - q.x : q.x, v.y >= 0.0f ? 1.0f - q.y : q.y));
}
__device__ __forceinline__ float act_gelu_tanh(float v) {
    // 2 * sqrt(2 / pi) * (v + 0.044715 v^3)
    return times_sigmoid(v, v * __fmaf_rn(0.0713548162726f, v * v, 1.59576912160573f));
}
__device__ __forceinline__ float act_silu(float v) { return times_sigmoid(v, v); }

// NV values through the same activation: one branch for all of them (`act` is uniform over the launch).
template <int NV>      // even
__device__ __forceinline__ void apply_act(float* v, int act) {
    if (act == HKB_ACT_RELU) {
#pragma unroll
        for (int j = 0; j < NV; ++j) v[j] = act_relu(v[j]);
    } else if (act == HKB_ACT_GELU) {
#pragma unroll
        for (int j = 0; j < NV; j += 2) {
            const float2 r = act_gelu2(make_float2(v[j], v[j + 1]));
            v[j] = r.x;
            v[j + 1] = r.y;
        }
    } else if (act == HKB_ACT_GELU_TANH) {
#pragma unroll
        for (int j = 0; j < NV; ++j) v[j] = act_gelu_tanh(v[j]);
    } else if (act == HKB_ACT_SILU) {
#pragma unroll
        for (int j = 0; j < NV; ++j) v[j] = act_silu(v[j]);
    }
}

}  // namespace hkb
