// act.h — activations and their slopes in f32 (linear.hip, linear_grad.hip).
#pragma once
#include "../../include/anneal_hip.h"
#include "ah_common.h"

namespace ah {

constexpr float kLog2e = 1.44269504088896340736f;

// e^x: the product with log2 e carries what its rounding loses, which at x = -10 is 3e-7 of the result.
__device__ __forceinline__ float exp_of(float x) {
    const float t = x * kLog2e, low = fmaf(x, kLog2e, -t) + x * 1.925963033500e-8f;   // log2 e less its f32 value
    const float r = __builtin_amdgcn_exp2f(t);
    return t > -126.0f ? fmaf(r, low * 0.69314718f, r) : r;   // -inf stays away from the correction
}

// silu(z) = z s(z) and gelu_tanh(z) = z s(2 k z (1 + 0.044715 z^2)), s(t) = 1 / (1 + e^-t), k = sqrt(2/pi): one form, z s(z (a + b z^2)).
constexpr float kTanhA = 1.5957691216057308f, kTanhB = kTanhA * 0.044715f;

// s(t) and s(t) (1 - s(t)), both without cancellation.
__device__ __forceinline__ float sigmoid(float t, float &slope) {
    const float e = exp_of(-fabsf(t)), r = __builtin_amdgcn_rcpf(1.0f + e);
    slope = e * r * r;
    return t < 0.0f ? e * r : r;
}

// The normal distribution: its density g at z, and the probability below z. FAST: t P(t) e^(-z^2/2), t = 1 / (1 + 0.305 |z|), for the tail,
// with a fit of the degree-7 P in the least maximal error: within 2e-7 of 1 anywhere and 4e-7 of the tail's value, to which the exponent's rounding
// adds up to 2^-24 z^2 (3e-6 at z = -8), for results that are rounded to f16.
template <bool FAST>
__device__ __forceinline__ float normal(float z, float &g) {
    const float e = FAST ? __builtin_amdgcn_exp2f(-0.5f * kLog2e * z * z) : exp_of(-0.5f * z * z);
    g = 0.3989422804014327f * e;
    if constexpr (FAST) {
        const float t = __builtin_amdgcn_rcpf(fmaf(0.305f, fabsf(z), 1.0f));
        float p = fmaf(t, 0.036699004f, -0.15298754f);
        p = fmaf(t, p, 0.18571551f);
        p = fmaf(t, p, -0.037975427f);
        p = fmaf(t, p, 0.12102083f);
        p = fmaf(t, p, 0.10342117f);
        p = fmaf(t, p, 0.12246676f);
        p = fmaf(t, p, 0.12163974f);
        p *= t * e;
        return z > 0.0f ? 1.0f - p : p;
    } else {
        return 0.5f * erfcf(-0.7071067811865476f * z);
    }
}

// FAST forms, for results that are rounded to f16: s(t) = 1 / (1 + 2^(-t log2 e)) without the exponent's correction and folding of signs
// (within 2^-20 up to |t| = 16, past which s is 0 or 1 to 2^-22), and 1 - s by subtraction (off by 2^-24 of 1).
template <bool FAST>
__device__ __forceinline__ float gate_of(int act, float z, float &q) {   // s(z (a + q)), q = b z^2
    const float a = act == AH_ACT_SILU ? 1.0f : kTanhA, b = act == AH_ACT_SILU ? 0.0f : kTanhB;
    if constexpr (FAST) {
        q = b * (z * z);
        return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * (fmaf(z * z, -kLog2e * b, -kLog2e * a))));
    } else {
        float unused;
        q = b * fminf(z * z, 1e30f);   // (0 times an infinite square would be NaN)
        return sigmoid(z * (a + q), unused);
    }
}

// act(z). NaN stays NaN under each of them. FAST takes z of at most 2^63.
template <bool FAST>
__device__ __forceinline__ float act_of(int act, float z) {
    float unused;
    if (act <= AH_ACT_RELU) return act == AH_ACT_RELU && z < 0.0f ? 0.0f : z;
    if (act == AH_ACT_GELU) return z * normal<FAST>(z, unused);
    return z * gate_of<FAST>(act, z, unused);
}

// act(z) and act'(z). Past |z| = 1e4 the slopes of both GELUs are 0 and 1 exactly, and their formulas would meet infinities.
template <bool FAST>
__device__ __forceinline__ float act_slope(int act, float z, float &slope) {
    if (act <= AH_ACT_RELU) {
        const bool off = act == AH_ACT_RELU && !(z > 0.0f);
        slope = off ? 0.0f : 1.0f;
        return off && z == z ? 0.0f : z;
    }
    if (act == AH_ACT_GELU) {
        float g;
        const float p = normal<FAST>(z, g);
        slope = g > 0.0f ? fmaf(z, g, p) : p;
        return z * p;
    }
    const float a = act == AH_ACT_SILU ? 1.0f : kTanhA;
    if constexpr (FAST) {
        float q;
        const float s = gate_of<true>(act, z, q);
        slope = fmaf(z * (s - s * s), fmaf(3.0f, q, a), s);
        return z * s;
    } else {
        const float b = act == AH_ACT_SILU ? 0.0f : kTanhB, q = b * fminf(z * z, 1e8f);
        float s1;
        const float s = sigmoid(z * (a + q), s1);
        slope = s1 > 0.0f ? fmaf(z * s1, fmaf(3.0f, q, a), s) : s;
        return z * s;
    }
}

// No act's slope is larger than this: the GELUs' largest is 1.129, SiLU's 1.0999.
__device__ __forceinline__ float slope_bound(int act) { return act <= AH_ACT_RELU ? 1.0f : 1.13f; }

}  // namespace ah
