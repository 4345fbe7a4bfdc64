// Residual addition + RMSNorm + FP8 (e4m3fn) quantization in one pass over the rows.
//
//   h = bf16(x + residual)                     the new residual stream, stored
//   y = h * rsqrt(mean(h^2) + eps) * w         fp32, never stored
//   scale = max(amax|y| / 448, 1e-10), q = e4m3fn_rne(clamp(y / scale, +-448)), amax over 128 columns or over the row (CodeDivider)
//
// h is rounded to bf16 before it is normalised, because the stored stream is what every later layer sees: the result is that of
// an addition into the stream followed by the norm of the stream.  Sums, statistics and y stay in fp32.
//
// HBM bounds it: 2 + 2 bytes in and 2 + 1 out per element, and nothing is read twice, because a thread keeps its part of h in
// registers from the sum to the codes.  A NaN, or an infinity in a row, comes out as the formula says: the maxima propagate NaN
// into the scales (fmaxf would drop it and leave finite codes).
#include "tc_common.cuh"

namespace hkb {
namespace {

constexpr float kFp8Max = 448.0f;
constexpr float kScaleFloor = 1e-10f;
constexpr int kThreads = 256;          // of the flat kernel, and of a CTA of several teams
constexpr int kMaxWarps = 16;          // of a team

// EL bf16 (8 or 16) of one row.  Plain loads, not the read-only path: residual_out may be x or residual.
template <int EL> struct Chunk { uint32_t w[EL / 2]; };
__device__ __forceinline__ void load(Chunk<16>& c, const __nv_bfloat16* p) {
    asm volatile("ld.global.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(c.w[0]), "=r"(c.w[1]), "=r"(c.w[2]), "=r"(c.w[3]), "=r"(c.w[4]), "=r"(c.w[5]), "=r"(c.w[6]), "=r"(c.w[7]) : "l"(p));
}
__device__ __forceinline__ void load(Chunk<8>& c, const __nv_bfloat16* p) {
    asm volatile("ld.global.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(c.w[0]), "=r"(c.w[1]), "=r"(c.w[2]), "=r"(c.w[3]) : "l"(p));
}
__device__ __forceinline__ void store(__nv_bfloat16* p, const Chunk<16>& c) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                 ::"l"(p), "r"(c.w[0]), "r"(c.w[1]), "r"(c.w[2]), "r"(c.w[3]), "r"(c.w[4]), "r"(c.w[5]), "r"(c.w[6]), "r"(c.w[7]) : "memory");
}
__device__ __forceinline__ void store(__nv_bfloat16* p, const Chunk<8>& c) { *reinterpret_cast<uint4*>(p) = make_uint4(c.w[0], c.w[1], c.w[2], c.w[3]); }
__device__ __forceinline__ void store_codes(uint8_t* p, const uint32_t (&o)[4]) { *reinterpret_cast<uint4*>(p) = make_uint4(o[0], o[1], o[2], o[3]); }
__device__ __forceinline__ void store_codes(uint8_t* p, const uint32_t (&o)[2]) { *reinterpret_cast<uint2*>(p) = make_uint2(o[0], o[1]); }

struct AddNormParams {
    const __nv_bfloat16 *x, *residual, *w;
    __nv_bfloat16* sum;
    uint8_t* q;
    float* scales;
    int64_t M;
    int D;
    float eps;
    int warps;             // of a team
};

// A team of `warps` warps has a row (blockDim / team rows per CTA), a thread holds NW chunks of EL elements, chunk index t + i * team.
// The 128 columns of a scale group lie in 128 / EL neighbouring lanes of one i.  Teams of a CTA meet on their own named barrier only.
template <int EL, int NW, bool kRowScale>
__global__ void __launch_bounds__(32 * kMaxWarps)
add_rmsnorm_quant_kernel(const AddNormParams p) {
    pdl_trigger();
    pdl_wait();
    const int team = 32 * p.warps, r_in = (int)threadIdx.x / team, t = (int)threadIdx.x - r_in * team;
    const int64_t row = (int64_t)blockIdx.x * ((int)blockDim.x / team) + r_in;
    const bool live = row < p.M;
    const int chunks = p.D / EL;
    const int64_t base = row * p.D;

    __shared__ float s_part[2][kMaxWarps];
    auto row_reduce = [&](int which, float v, auto op) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
        if (p.warps > 1) {
            float* const part = s_part[which] + r_in * p.warps;
            if ((t & 31) == 0) part[t >> 5] = v;
            asm volatile("bar.sync %0, %1;" ::"r"(1 + r_in), "r"(team) : "memory");
            v = part[0];
            for (int k = 1; k < p.warps; ++k) v = op(v, part[k]);
        }
        return v;
    };

    Chunk<EL> h[NW];
    {
        Chunk<EL> a[NW];
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            const int c = t + i * team;
            if (live && c < chunks) {
                load(a[i], p.x + base + (int64_t)c * EL);
                load(h[i], p.residual + base + (int64_t)c * EL);
            } else {
#pragma unroll
                for (int j = 0; j < EL / 2; ++j) a[i].w[j] = h[i].w[j] = 0;
            }
        }
#pragma unroll
        for (int i = 0; i < NW; ++i)
#pragma unroll
            for (int j = 0; j < EL / 2; ++j) {
                const float2 u = bf16x2_to_f2(a[i].w[j]), v = bf16x2_to_f2(h[i].w[j]);
                const __nv_bfloat162 s = __floats2bfloat162_rn(u.x + v.x, u.y + v.y);
                h[i].w[j] = *reinterpret_cast<const uint32_t*>(&s);
            }
    }
    float2 ss2 = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < NW; ++i) {
        const int c = t + i * team;
        if (live && c < chunks) store(p.sum + base + (int64_t)c * EL, h[i]);
#pragma unroll
        for (int j = 0; j < EL / 2; ++j) { const float2 f = bf16x2_to_f2(h[i].w[j]); ss2 = __ffma2_rn(f, f, ss2); }
    }
    const float ss = row_reduce(0, ss2.x + ss2.y, [](float a, float b) { return a + b; });
    const float rinv = rsqrtf(ss / (float)p.D + p.eps);
    const float2 rinv2 = make_float2(rinv, rinv);

    // y of chunk i; the gain comes from L1 / L2
    auto normed = [&](int i, float2 (&y)[EL / 2]) {
        const int c = t + i * team;
        uint4 w[EL / 8];
#pragma unroll
        for (int k = 0; k < EL / 8; ++k)
            w[k] = c < chunks ? __ldg(reinterpret_cast<const uint4*>(p.w + (int64_t)c * EL) + k) : make_uint4(0, 0, 0, 0);
        const uint32_t* const ww = reinterpret_cast<const uint32_t*>(w);
        float am = 0.0f;
#pragma unroll
        for (int j = 0; j < EL / 2; ++j) {
            y[j] = __fmul2_rn(__fmul2_rn(bf16x2_to_f2(h[i].w[j]), rinv2), bf16x2_to_f2(ww[j]));
            am = max_nan(am, max_nan(fabsf(y[j].x), fabsf(y[j].y)));
        }
        return am;
    };
    // The quotient is rounded as a division rounds it.  y * RN(1/scale) is within an fp32 ulp of that, but h and w have few bits, so many
    // quotients lie between two codes exactly, and that ulp decides them: of 16384 x 8192 codes 11967 were not those of 64 bits, now 10977
    // (the order of the sum of squares decides the rest).  1000 x 4096 with block scales 4.8 -> 4.9 us, 16384 x 8192 no difference.
    auto emit = [&](int i, const float2 (&y)[EL / 2], const CodeDivider& codes) {
        const int c = t + i * team;
        uint32_t o[EL / 4];
#pragma unroll
        for (int j = 0; j < EL / 4; ++j) o[j] = codes(y[2 * j], y[2 * j + 1]);
        if (live && c < chunks) store_codes(p.q + base + (int64_t)c * EL, o);
    };

    if constexpr (kRowScale) {
        // y stays in registers for the second pass instead of h; with 48 of them that costs a CTA of the SM, so there it is computed again.
        // Again / kept, us: 1000 x 4104 6.4 / 6.0, 2000 x 16384 52.9 / 37.6, 4000 x 32768 155.6 / 153.7; 4000 x 8200 (48) 44.0 / 48.5.
        constexpr bool kKeep = EL * NW != 48;
        float2 y[kKeep ? NW : 1][EL / 2];
        float am = 0.0f;
#pragma unroll
        for (int i = 0; i < NW; ++i) am = max_nan(am, normed(i, y[kKeep ? i : 0]));
        am = row_reduce(1, am, [](float a, float b) { return max_nan(a, b); });
        const float scale = max_nan(__fdiv_rn(am, kFp8Max), kScaleFloor);
        const CodeDivider codes(scale);
        if (live && t == 0) p.scales[row] = scale;
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            if constexpr (!kKeep) normed(i, y[0]);
            emit(i, y[kKeep ? i : 0], codes);
        }
    } else {
        constexpr int LANES = 128 / EL;
        float2 y[EL / 2];
        float* const sr = p.scales + row * (p.D / 128);
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            float am = normed(i, y);
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) am = max_nan(am, __shfl_xor_sync(0xFFFFFFFFu, am, o));
            const float scale = max_nan(__fdiv_rn(am, kFp8Max), kScaleFloor);
            emit(i, y, CodeDivider(scale));
            const int c = t + i * team;
            if (live && c < chunks && t % LANES == 0) sr[c / LANES] = scale;
        }
    }
}

// Chunks per thread.  Few rows, where only latency counts: one, as many warps per row as it takes.  Else 32 elements per thread (24 in
// 8-element chunks) in teams of up to 16 (8) warps, more only for rows that need it.  us in a replayed graph with 1 / 2 / 3 / 4 chunks of
// 16, block scales: 300 x 4096 3.3 / 3.5 / 3.9 / 4.2, 1000 x 4096 5.4 / 5.1 / 6.8 / 5.4, 1000 x 5120 6.2 / 6.4 / 7.4 / 7.8, 4096 x 4096
// 22.1 / 18.6 / 21.0 / 20.2, 4096 x 5120 25.7 / 25.5 / 28.5 / 29.8, 16384 x 8192 146 / 137 / 152 / 140; row scales 1000 x 4096 6.0 / 5.1 /
// 7.6 / 5.2, 16384 x 8192 189 / 136 / 169 / 144.  With 1 / 2 / 3 / 4 / 6 / 8 chunks of 8, row scales: 8000 x 1032 25.5 / 16.0 / 11.5 / 14.0 /
// 13.4 / 12.5, 8000 x 2056 33.1 / 30.9 / 21.3 / 22.2 / 27.4 / 27.2, 4000 x 16376 - / - / - / 105 / 113 / 77.  4000 x 8200, the narrowest
// rows with six, would be ahead with fewer: - / - / 40.9 / 40.4 / 44.7 / 42.7.
template <int EL, bool kRowScale>
int dispatch_add_norm(AddNormParams p, cudaStream_t st) {
    const int chunks = p.D / EL, most = (chunks + 31) / 32, sms = sm_count();
    HKB_REQUIRE(sms > 0, HKB_ERR_CUDA, "no CUDA device");
    int nw;
    if (most == 1 || (most <= kMaxWarps && p.M * most <= 16 * (int64_t)sms)) nw = 1;
    else if constexpr (EL == 16) nw = most <= 2 * kMaxWarps ? 2 : 4;
    else nw = most <= 3 * 8 ? 3 : most <= 6 * 8 ? 6 : 8;
    void (*kern)(AddNormParams) = add_rmsnorm_quant_kernel<EL, 1, kRowScale>;
    if constexpr (EL == 16) {
        if (nw == 2) kern = add_rmsnorm_quant_kernel<EL, 2, kRowScale>;
        if (nw == 4) kern = add_rmsnorm_quant_kernel<EL, 4, kRowScale>;
    } else {
        if (nw == 3) kern = add_rmsnorm_quant_kernel<EL, 3, kRowScale>;
        if (nw == 6) kern = add_rmsnorm_quant_kernel<EL, 6, kRowScale>;
        if (nw == 8) kern = add_rmsnorm_quant_kernel<EL, 8, kRowScale>;
    }
    p.warps = (most + nw - 1) / nw;                  // at most kMaxWarps: D <= 32768
    const int teams = p.warps >= kThreads / 32 ? 1 : kThreads / 32 / p.warps;
    HKB_CUDA(launch_dependent(true, kern, (unsigned)((p.M + teams - 1) / teams), 32 * p.warps * teams, 0, 0, st, p));
    return check_launch("add_rmsnorm_quant_kernel");
}

// fp32 groups of 128 -> codes and scales: eight lanes per group, 16 elements each.
__global__ void __launch_bounds__(kThreads)
quant_f32_1x128_kernel(const float* __restrict__ y, uint8_t* __restrict__ q, float* __restrict__ scales, int64_t groups) {
    pdl_trigger();
    pdl_wait();
    const int64_t g = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / 8;
    const int sub = threadIdx.x & 7;
    float v[16];
    float am = 0.0f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float4 f = g < groups ? *reinterpret_cast<const float4*>(y + g * 128 + sub * 16 + 4 * k) : make_float4(0, 0, 0, 0);
        v[4 * k] = f.x; v[4 * k + 1] = f.y; v[4 * k + 2] = f.z; v[4 * k + 3] = f.w;
    }
#pragma unroll
    for (int k = 0; k < 16; ++k) am = max_nan(am, fabsf(v[k]));
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) am = max_nan(am, __shfl_xor_sync(0xFFFFFFFFu, am, o));
    const float scale = max_nan(__fdiv_rn(am, kFp8Max), kScaleFloor);
    if (g < groups) {
        const CodeDivider codes(scale);
        uint32_t o[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = codes(make_float2(v[4 * k], v[4 * k + 1]), make_float2(v[4 * k + 2], v[4 * k + 3]));
        *reinterpret_cast<uint4*>(q + g * 128 + sub * 16) = make_uint4(o[0], o[1], o[2], o[3]);
        if (sub == 0) scales[g] = scale;
    }
}

}  // namespace

int launch_quant_f32_1x128(const float* y, void* q, float* scales, int64_t groups, cudaStream_t st) {
    HKB_CUDA(launch_dependent(true, quant_f32_1x128_kernel, (unsigned)((groups * 8 + kThreads - 1) / kThreads), kThreads, 0, 0, st, y, (uint8_t*)q, scales, groups));
    return check_launch("quant_f32_1x128_kernel");
}

}  // namespace hkb

extern "C" int hkb_add_rmsnorm_quant_fp8(const void* x, const void* residual, const void* w, void* q, float* scales, void* residual_out,
                                         int64_t M, int64_t D, int64_t group, float eps, void* stream) {
    using namespace hkb;
    HKB_REQUIRE(M >= 0 && M <= 0x7FFFFFFFLL && D > 0 && D <= 32768 && D % 8 == 0, HKB_ERR_BAD_SHAPE,
                "add_rmsnorm_quant_fp8: need D %% 8 == 0 and 0 < D <= 32768, got M=%lld D=%lld", (long long)M, (long long)D);
    HKB_REQUIRE(group == D || (group == 128 && D % 128 == 0), HKB_ERR_BAD_SHAPE,
                "add_rmsnorm_quant_fp8: one scale per 128 columns (D %% 128 == 0) or per row, got group %lld of D=%lld", (long long)group, (long long)D);
    if (M == 0) return HKB_OK;               // an empty tensor has no address
    HKB_REQUIRE(x && residual && w && q && scales && residual_out, HKB_ERR_BAD_ARG, "add_rmsnorm_quant_fp8: null pointer");
    HKB_REQUIRE(aligned16(x) && aligned16(residual) && aligned16(w) && aligned16(residual_out) && ((uintptr_t)q & 7) == 0 && ((uintptr_t)scales & 3) == 0,
                HKB_ERR_BAD_ALIGN, "add_rmsnorm_quant_fp8: x, residual, w and residual_out must be 16-byte, q 8-byte, scales 4-byte aligned");
    const AddNormParams p{(const __nv_bfloat16*)x, (const __nv_bfloat16*)residual, (const __nv_bfloat16*)w, (__nv_bfloat16*)residual_out,
                          (uint8_t*)q, scales, M, (int)D, eps, 0};
    // 32-byte chunks where every row of every tensor starts on one
    const bool wide = D % 16 == 0 && aligned32(x) && aligned32(residual) && aligned32(residual_out) && aligned16(q);
    cudaStream_t st = (cudaStream_t)stream;
    if (group == D) return wide ? dispatch_add_norm<16, true>(p, st) : dispatch_add_norm<8, true>(p, st);
    return wide ? dispatch_add_norm<16, false>(p, st) : dispatch_add_norm<8, false>(p, st);
}
