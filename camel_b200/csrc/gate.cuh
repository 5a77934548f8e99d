// The activations of a gated dense layer and their slopes.
#pragma once

#include "camel_tensor_b200.h"

#include <cstdint>

namespace ct {

// Both sides of the logistic function with their full relative precision: 1 - sigmoid(g) is sigmoid(-g), not a difference; the smaller one is 0
// below 2^-126 (|g| beyond 87.3).
// exp(-|g|) = 2^t (1 + r ln 2), t the rounded -|g| log2(e) and r what it lacks, to 2^-22 of itself; 1 / (1 + e), of a number from 1 to 2, by
// a reciprocal and a Newton step.  No branches: in the epilogue of a product the division's and expf's cost a tile as much as half of its MMAs.
__device__ __forceinline__ void sigmoids(float g, float &s, float &other) {
    const float kLog2e = 1.44269502162933349609375f, kLog2eRest = 1.925963033500011079e-8f;
    float x, e, a;
    asm("min.NaN.f32 %0, %1, 0f42D00000;" : "=f"(x) : "f"(fabsf(g))); // 104: e is 0 from 87.3 on, and stays it
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

// The normal distribution function and its density over that of 0, both from one exponential: cdf(-x) = exp(-x^2 / 2) E(x), and E(x) (1 + c x),
// c = 0.35, is a polynomial of t = 1 / (1 + c x) to 2^-24.9 of itself for x up to 14.5, beyond which cdf(-x) is no float any more.
// (Coefficients: least squares in t at 600 Chebyshev nodes of (0, 1], weights raised where the relative error was largest until it was level.)
// x^2 is taken with what its rounding lost, or exp's error would grow with it.  To 2^-21 of the smaller of cdf and 1 - cdf.  No branches, as
// above: with normcdff (as far off, 2^-21.4) and expf 8192 x 512 x 5504 took 317 us, so 271, its gradient with k = 64 470, so 441.
__device__ __forceinline__ void normal(float g, float &cdf, float &exponential) {
    const float kHalfLog2e = 0.7213475108146667480f, kHalfLog2eRest = 9.629815167e-9f;
    float x, e, t;
    asm("min.NaN.f32 %0, %1, 0f41700000;" : "=f"(x) : "f"(fabsf(g))); // 15
    const float p = __fmul_rn(x, x), rest = __fmaf_rn(x, x, -p), y = __fmul_rn(-p, kHalfLog2e);
    const float r = __fmaf_rn(-rest, kHalfLog2e, __fmaf_rn(-p, kHalfLog2eRest, __fmaf_rn(-p, kHalfLog2e, -y)));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(y));
    e             = __fmaf_rn(__fmul_rn(e, r), 0.693147182464599609375f, e);
    const float d = __fmaf_rn(0.35f, x, 1.0f);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(d));
    t       = __fmaf_rn(t, __fmaf_rn(-d, t, 1.0f), t);
    float q = -2.915788442e-02f;
    q = __fmaf_rn(q, t, 1.440309137e-01f), q = __fmaf_rn(q, t, -2.558390200e-01f), q = __fmaf_rn(q, t, 1.593197286e-01f);
    q = __fmaf_rn(q, t, -2.321236767e-02f), q = __fmaf_rn(q, t, 1.055525094e-01f), q = __fmaf_rn(q, t, 1.198212877e-01f);
    q = __fmaf_rn(q, t, 1.398635060e-01f), q = __fmaf_rn(q, t, 1.396213025e-01f);
    const float tail = __fmul_rn(e, __fmul_rn(q, t));
    cdf         = g >= 0.0f ? __fsub_rn(1.0f, tail) : tail;
    exponential = e;
}

template <int GATE> __device__ __forceinline__ float gate_value(float g) {
    if (GATE == CT_GATE_RELU)
        return __fmul_rn(g, g > 0.0f ? 1.0f : 0.0f);
    if (GATE == CT_GATE_GELU) {
        float cdf, e;
        normal(g, cdf, e);
        return __fmul_rn(g, cdf);
    }
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
        float cdf, e;
        normal(g, cdf, e);
        value = __fmul_rn(g, cdf), slope = __fmaf_rn(g, __fmul_rn(0.3989422804f, e), cdf);
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
