// Activations of the fused GEMM epilogues, fp32 in and out.
//
// Each is written in the form that keeps its relative accuracy where the result is small (a sum like 1 + erf(v) or 1 + tanh(u)
// cancels there): gelu through erfc, the tanh form as v * sigmoid(2u) = v / (1 + exp(-2u)).  NaN stays NaN and infinities follow
// the formulas: silu and both forms of gelu of -inf are -inf * 0 = NaN.
#pragma once

#include "common.cuh"

namespace hkb {

inline bool act_known(int act) { return act >= HKB_ACT_NONE && act <= HKB_ACT_SILU; }

__device__ __forceinline__ float2 twice(float c) { return make_float2(c, c); }

// v / (1 + exp(-z)), for negative z as v * exp(z) / (1 + exp(z)): exp(-z) itself overflows while the quotient is still a normal
// number.  Two values at a time on the packed fp32 pipe.  exp(-|z|) is the square of exp(-|z| / 2), which stays a normal number
// until the square is zero: the exponential needs no care for small results, the product has it anyway.  The denominators x and y are
// in [1, 2], so one reciprocal of the special-function pipe does for both: 1 / (xy) times y and times x.  A NaN would reach the other
// value through it; it becomes 2 there and stays in the numerator.  Measured, silu: off by 2^-20.4 of the value for
// |z| <= 8, 2^-18 at 60 (the exponent's rounding, |z| * 2^-23.4).  4096 x 4096 x 1024 with bias, us, block scales / per-token: this 42.8 /
// 31.4, a reciprocal each 43.8 / 32.5, __expf and __fdividef 43.7 / 33.0, no activation 34.8 / 24.8.
__device__ __forceinline__ float2 times_sigmoid2(float2 v, float2 z) {
    constexpr float c = -0.72134752044448170f;             // powers of two in half a unit of exp
    float2 h;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(h.x) : "f"(fabsf(z.x) * c));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(h.y) : "f"(fabsf(z.y) * c));
    const float2 d = __ffma2_rn(h, h, twice(1.0f)), x = make_float2(fminf(d.x, 2.0f), fminf(d.y, 2.0f)), vt = __fmul2_rn(v, __fmul2_rn(h, h));
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x.x * x.y));
    return __fmul2_rn(make_float2(z.x >= 0.0f ? v.x : vt.x, z.y >= 0.0f ? v.y : vt.y), __fmul2_rn(twice(r), make_float2(x.y, x.x)));
}

__device__ __forceinline__ float act_relu(float v) { return v < 0.0f ? 0.0f : v; }
// v * Phi(v), two values at a time on the packed fp32 pipe.  For a = |v|, Phi(-a) = erfc(a / sqrt 2) / 2 = exp(-a^2 / 2) t P(t) with
// t = 1 / (1 + 0.36 a): the scaled function is smooth in t on (0, 1], and P, of degree 6, is a minimax fit of its relative error over
// 0 <= a <= 14 (8.7e-7; with the roundings 2^-19.4 for a <= 3, 2^-18.7 for a <= 6, 2^-17 at 13, where the exponent's argument rounds).
// One reciprocal for both values (as above) was 2 % behind here: the polynomial keeps the other pipes busy.
// 2000 x 14336 x 4096 with bias, us: this 98, erfcf() 118 (its 50 instructions per value outlast the main loop), no activation 95.
__device__ __forceinline__ float2 act_gelu2(float2 v) {
    const float2 a = make_float2(fabsf(v.x), fabsf(v.y));
    const float2 d = __ffma2_rn(a, twice(0.36f), twice(1.0f));
    float2 t, e;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t.x) : "f"(d.x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t.y) : "f"(d.y));
    float2 q = __ffma2_rn(twice(4.705620929598808e-2f), t, twice(-1.7976443469524384e-1f));
    q = __ffma2_rn(q, t, twice(1.8095368146896362e-1f));
    q = __ffma2_rn(q, t, twice(2.6549549773335457e-2f));
    q = __ffma2_rn(q, t, twice(1.397191882133484e-1f));
    q = __ffma2_rn(q, t, twice(1.4177246391773224e-1f));
    q = __ffma2_rn(q, t, twice(1.4371304214000702e-1f));
    const float2 x = __fmul2_rn(__fmul2_rn(v, v), twice(-0.36067376022224085f));        // -a^2 / 4 in powers of two
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(x.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(x.y));
    e = __fmul2_rn(e, e);
    q = __fmul2_rn(__fmul2_rn(q, t), e);
    return __fmul2_rn(v, make_float2(v.x >= 0.0f ? 1.0f - q.x : q.x, v.y >= 0.0f ? 1.0f - q.y : q.y));
}
__device__ __forceinline__ float2 act_gelu_tanh2(float2 v) {
    // 2 * sqrt(2 / pi) * (v + 0.044715 v^3); measured: off by 2^-19.6 for v >= -3, 2^-17.7 at -6, 2^-15.7 at -13 (z is -180 there)
    return times_sigmoid2(v, __fmul2_rn(v, __ffma2_rn(twice(0.0713548162726f), __fmul2_rn(v, v), twice(1.59576912160573f))));
}
__device__ __forceinline__ float2 act_silu2(float2 v) { return times_sigmoid2(v, v); }

// NV values (an even number) through the same activation: one branch for all of them (`act` is uniform over the launch).
template <int NV>
__device__ __forceinline__ void apply_act(float* v, int act) {
    auto pairs = [&](auto f) {
#pragma unroll
        for (int j = 0; j < NV; j += 2) {
            const float2 r = f(make_float2(v[j], v[j + 1]));
            v[j] = r.x;
            v[j + 1] = r.y;
        }
    };
    if (act == HKB_ACT_NONE) return;
    if (act == HKB_ACT_RELU) pairs([](float2 x) { return make_float2(act_relu(x.x), act_relu(x.y)); });
    else if (act == HKB_ACT_GELU) pairs([](float2 x) { return act_gelu2(x); });
    else if (act == HKB_ACT_GELU_TANH) pairs([](float2 x) { return act_gelu_tanh2(x); });
    else pairs([](float2 x) { return act_silu2(x); });
}

}  // namespace hkb
