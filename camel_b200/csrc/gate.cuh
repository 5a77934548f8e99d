// The activations of a gated dense layer and their slopes.
#pragma once

#include "camel_tensor_b200.h"

#include <cstdint>

namespace ct {

// Both sides of the logistic function with their full relative precision: 1 - sigmoid(g) is sigmoid(-g), not a difference.
__device__ __forceinline__ void sigmoids(float g, float &s, float &other) {
    const float e = expf(-fabsf(g));
    const float a = __fdiv_rn(1.0f, __fadd_rn(1.0f, e)), b = __fmul_rn(e, a);
    s     = g >= 0.0f ? a : b;
    other = g >= 0.0f ? b : a;
    if (g != g)
        s = other = g;
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
