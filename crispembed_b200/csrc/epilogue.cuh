// epilogue.cuh -- what the kernels of the linear layers share behind the products: Q4_K
// nibbles as floats, activations, and values of the three activation types.
#pragma once

#include "../../include/ceb_ops.h"
#include "common.cuh"

namespace ceb_epi {

CEB_DEV float nib_f(uint32_t v, int byte) {
    return __uint_as_float(0x4B000000u | ((v >> (8 * byte)) & 0xFFu)) - 8388608.0f;
}

// erf-GELU 0.5 x (1 + erf(x / sqrt 2)) with erf from Abramowitz & Stegun 7.1.26
// (|error| <= 1.5e-7 on erf), far below the fp16/fp32 rounding of the output:
//   z = |x|/sqrt2, t = 1/(1 + p z), erf(z) = 1 - t(a1 + t(a2 + t(a3 + t(a4 + t a5)))) exp(-z^2).
// The reciprocal and the exponential use the MUFU approximations (rel. error ~2^-22),
// exp(-z^2) as 2^(-(z sqrt(log2 e))^2) with the scaling folded into one constant.
CEB_DEV float rcp_approx(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
CEB_DEV float ex2_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
CEB_DEV float gelu_as(float x) {
    constexpr float kZ = 0.70710678118654752f;             // 1/sqrt(2)
    constexpr float kE = 0.84932180028801904f;             // sqrt(log2 e) / sqrt(2)
    const float ax = fabsf(x);
    const float t = rcp_approx(fmaf(0.3275911f * kZ, ax, 1.0f));
    float p = fmaf(1.061405429f, t, -1.453152027f);
    p = fmaf(p, t, 1.421413741f);
    p = fmaf(p, t, -0.284496736f);
    p = fmaf(p, t, 0.254829592f);
    const float u = ax * kE;
    const float e = ex2_approx(-u * u);                     // exp(-x^2/2)
    const float erf_abs = fmaf(-p * t, e, 1.0f);            // erf(|x|/sqrt2)
    const float h = 0.5f * x;
    return fmaf(fabsf(h), erf_abs, h);                      // 0.5x + 0.5|x| erf(|x|/sqrt2)
}

// Activations of the extended epilogue.  silu(x) = x / (1 + exp(-x)); the tanh form of GELU
// is the same with 2 sqrt(2/pi) (x + 0.044715 x^3) in the exponent, since
// (1 + tanh u) / 2 = 1 / (1 + exp(-2u)).  Exponential and reciprocal are the MUFU
// approximations (relative error ~2^-22, below the fp32 sums in front of them).
template <int ACT>
CEB_DEV float ex_act1(float x) {
    if (ACT == CEB_FN_GELU) return gelu_as(x);
    if (ACT == CEB_FN_RELU) return x < 0.0f ? 0.0f : x;  // NaN stays
    if (ACT == CEB_FN_NONE) return x;
    constexpr float kL = 1.4426950408889634f, kG = 2.0f * 0.79788456080286536f;
    const float u = ACT == CEB_FN_SILU ? x : kG * fmaf(0.044715f * x * x, x, x);
    return x * rcp_approx(1.0f + ex2_approx(-kL * u));
}
template <int ACT>
CEB_DEV void ex_act_all(float* x) {
#pragma unroll
    for (int j = 0; j < 32; ++j) x[j] = ex_act1<ACT>(x[j]);
}
// 32 values: one branch for all
CEB_DEV void ex_act(float* x, int act) {
    if (act == CEB_FN_SILU) ex_act_all<CEB_FN_SILU>(x);
    else if (act == CEB_FN_GELU) ex_act_all<CEB_FN_GELU>(x);
    else if (act == CEB_FN_GELU_TANH) ex_act_all<CEB_FN_GELU_TANH>(x);
    else if (act == CEB_FN_RELU) ex_act_all<CEB_FN_RELU>(x);
}
// one value of type CEB_ACT_* at element `i` of `p`
CEB_DEV float load1(const void* p, int type, int64_t i) {
    if (type == CEB_ACT_F32) return static_cast<const float*>(p)[i];
    if (type == CEB_ACT_F16) return __half2float(static_cast<const __half*>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
// two values as the packed 16-bit pair of type `type`
CEB_DEV uint32_t pack2(float a, float b, int type) {
    if (type == CEB_ACT_F16) return h2_as_u32(__floats2half2_rn(a, b));
    __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&r);
}
CEB_DEV void store1(void* p, int type, int64_t i, float v) {
    if (type == CEB_ACT_F32) static_cast<float*>(p)[i] = v;
    else if (type == CEB_ACT_F16) static_cast<__half*>(p)[i] = __float2half_rn(v);
    else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}
CEB_DEV float ex_act_one(float x, int act) {
    return act == CEB_FN_SILU        ? ex_act1<CEB_FN_SILU>(x)
           : act == CEB_FN_GELU      ? ex_act1<CEB_FN_GELU>(x)
           : act == CEB_FN_GELU_TANH ? ex_act1<CEB_FN_GELU_TANH>(x)
           : act == CEB_FN_RELU      ? ex_act1<CEB_FN_RELU>(x)
                                     : x;
}

}  // namespace ceb_epi
