// The activations of a gated dense layer and their slopes.
#pragma once

#include "camel_tensor_b200.h"

#include <cstdint>

namespace ct {

// Both sides of the logistic function with their full relative precision: 1 - sigmoid(g) is sigmoid(-g), not a difference.
// exp(-|g|) = 2^t (1 + r ln 2), t the rounded -|g| log2(e) and r what it lacks, to 2^-22 of itself; 1 / (1 + e), of a number from 1 to 2, by
// a reciprocal and a Newton step.  No branches: in the epilogue of a product the division's and expf's cost a tile as much as half of its MMAs.
__device__ __forceinline__ void sigmoids(float g, float &s, float &other) {
    const float kLog2e = 1.44269502162933349609375f, kLog2eRest = 1.925963033500011079e-8f;
    float x, e, a;
    asm("min.NaN.f32 %0, %1, 0f42D00000;" : "=f"(x) : "f"(fabsf(g))); // 104, where exp(-x) is no float any more
    const float t = __fmul_rn(-x, kLog2e);
    const float r = __fmaf_rn(-x, kLog2eRest, __fmaf_rn(-x, kLog2e, -t));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
    e             = __fmaf_rn(__fmul_rn(e, r), 0.693147182464599609375f, e);
    const float d = __fadd_rn(1.0f, e);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(a) : "f"(d));
    a             = __fmaf_rn(a, __fmaf_rn(-d, a, 1.0f), a);
    const float b = __fmul_rn(e, a);
    s     = g >= 0.0f ? a : b;
    other = g >= 0.0f ? b : a;
}

template <int GATE> __device__ __forceinline__ float gate_value(float g) {
    if (GATE == CT_GATE_RELU)
        return __fmul_rn(g, g > 0.0f ? 1.0f : 0.0f);
    if (GATE == CT_GATE_GELU)
        return __fmul_rn(g, normcdff(g));
    float s, other;
    sigmoids(g, s, other);
    return GATE == CT_GATE_SILU ? __fmul_rn(g, s) : s;
}

// gate(g) and gate'(g)
template <int GATE> __device__ __forceinline__ void gate_slope(float g, float &value, float &slope) {
    if (GATE == CT_GATE_RELU) {
        const float on = g > 0.0f ? 1.0f : 0.0f;
        value = __fmul_rn(g, on), slope = on;
    } else if (GATE == CT_GATE_GELU) {
        const float cdf = normcdff(g), pdf = __fmul_rn(0.3989422804f, expf(__fmul_rn(-0.5f, __fmul_rn(g, g))));
        value = __fmul_rn(g, cdf), slope = __fmaf_rn(g, pdf, cdf);
    } else {
        float s, other;
        sigmoids(g, s, other);
        value = GATE == CT_GATE_SILU ? __fmul_rn(g, s) : s;
        slope = GATE == CT_GATE_SILU ? __fmul_rn(s, __fmaf_rn(g, other, 1.0f)) : __fmul_rn(s, other);
    }
}

inline bool valid_gate(int gate) { return gate >= CT_GATE_SIGMOID && gate <= CT_GATE_GELU; }

// f(std::integral_constant<int, GATE>)
template <typename F> auto with_gate(int gate, F &&f) {
    switch (gate) {
    case CT_GATE_SIGMOID:
        return f(std::integral_constant<int, CT_GATE_SIGMOID>{});
    case CT_GATE_RELU:
        return f(std::integral_constant<int, CT_GATE_RELU>{});
    case CT_GATE_SILU:
        return f(std::integral_constant<int, CT_GATE_SILU>{});
    default:
        return f(std::integral_constant<int, CT_GATE_GELU>{});
    }
}

} // namespace ct
