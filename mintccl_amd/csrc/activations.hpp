// Activations and their slopes, of gates (norms.hpp) and of products (dense.hip), in 32 bits.  Which one is uniform over a
// launch.  No counterpart in the reference.
#pragma once
#include "operators.hpp"

#include <cfloat>

namespace mint {

// e^x: 2^p of the rounded product p = x log2(e), and what the rounding left over to the first order; a few units of 2^-24 off, in
// eight instructions.  From |p| = 126 on (|x| = 87.3) nothing is put right, since 2^p may be infinite: up to |p| = 128 it is off by the rounding of p, 44 units at most.  Beyond
// the range it is infinite, or 0.
__device__ __forceinline__ float exponential(float x) {
    constexpr float kLog2e = 0x1.715476p+0f, kRest = 0x1.4ae0c0p-26f, kLn2 = 0x1.62e430p-1f;
    const float p = x * kLog2e, left = fmaf(x, kRest, fmaf(x, kLog2e, -p)), power = __builtin_amdgcn_exp2f(p);
    return fabsf(p) < 126.0f ? fmaf(power, left * kLn2, power) : power;
}
__device__ __forceinline__ float reciprocal(float x) { return __builtin_amdgcn_rcpf(x); }
__device__ __forceinline__ float logistic(float x) { return reciprocal(1.0f + exponential(-x)); }
// Near 0, where 1 - 2 / (1 + e^2x) cancels, the first terms of its series: x^11 is less than 2^-29 of x there.
__device__ __forceinline__ float tangent(float x) {
    const float s = x * x, near = x * fmaf(fmaf(fmaf(fmaf(0.0218694885f, s, -0.0539682540f), s, 0.133333333f), s, -0.333333333f), s, 1.0f);
    const float far = copysignf(1.0f - 2.0f * reciprocal(1.0f + exponential(2.0f * fabsf(x))), x);
    return fabsf(x) < 0.25f ? near : far;
}
// 1 - tanh^2 = 1 / cosh^2, without a difference that cancels where tanh is near 1
__device__ __forceinline__ float tangent_slope(float x) {
    const float e = exponential(-2.0f * fabsf(x)), r = reciprocal(1.0f + e);
    return 4.0f * e * r * r;
}
// P(N > x) of a normal N for x >= 0: Abramowitz and Stegun, 7.1.26 (1.5e-7 off at most, for twice of it), with e^(-x^2 / 2) as `power`.
__device__ __forceinline__ float normal_above(float x, float power) {
    const float t = reciprocal(fmaf(0.3275911f * 0.70710678f, x, 1.0f));
    const float poly = fmaf(fmaf(fmaf(fmaf(1.061405429f, t, -1.453152027f), t, 1.421413741f), t, -0.284496736f), t, 0.254829592f) * t;
    return 0.5f * poly * power;
}

// MINT_ACT_GELU is x * P(N <= x) of a normal N, MINT_ACT_GELU_TANH the approximation of it by a hyperbolic tangent: 1 + tanh(u) = 2 logistic(2 u).
template <int N>
__device__ __forceinline__ void activate(int kind, float (&v)[N]) {
    switch (kind) {
        case MINT_ACT_RELU:
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = v[i] > 0.0f || v[i] != v[i] ? v[i] : 0.0f;
            break;
        case MINT_ACT_SILU:
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] *= logistic(v[i]);
            break;
        case MINT_ACT_SIGMOID:
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = logistic(v[i]);
            break;
        case MINT_ACT_TANH:
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = tangent(v[i]);
            break;
        case MINT_ACT_GELU:
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float above = normal_above(fabsf(v[i]), exponential(-0.5f * v[i] * v[i]));
                v[i] *= v[i] < 0.0f ? above : 1.0f - above;
            }
            break;
        case MINT_ACT_GELU_TANH:
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] *= logistic(1.5957691f * fmaf(0.044715f * v[i], v[i] * v[i], v[i]));
            break;
        default: break;
    }
}
// the largest number of its sign in the place of an infinity: times 0 it is 0
__device__ __forceinline__ float finite(float x) { return __builtin_amdgcn_fmed3f(x, -FLT_MAX, FLT_MAX); }
// ... v becomes the activation's slope there, at an infinity its limit (what is kept of a product in 16 bits may have left their range)
template <int N>
__device__ __forceinline__ void slopes(int kind, float (&v)[N]) {
    switch (kind) {
        case MINT_ACT_RELU:
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = v[i] > 0.0f ? 1.0f : v[i] != v[i] ? v[i] : 0.0f;
            break;
        case MINT_ACT_SILU:
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float s = logistic(v[i]);
                v[i] = s * fmaf(finite(v[i]), 1.0f - s, 1.0f);
            }
            break;
        case MINT_ACT_SIGMOID:
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float e = exponential(-fabsf(v[i])), r = reciprocal(1.0f + e);      // (of either sign without a difference that cancels)
                v[i] = e * r * r;
            }
            break;
        case MINT_ACT_TANH:
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = tangent_slope(v[i]);
            break;
        case MINT_ACT_GELU:
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float power = exponential(-0.5f * v[i] * v[i]), above = normal_above(fabsf(v[i]), power), below = v[i] < 0.0f ? above : 1.0f - above;
                v[i] = power == 0.0f ? below : fmaf(v[i], 0.39894228f * power, below);
            }
            break;
        case MINT_ACT_GELU_TANH:
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float x = v[i], s = logistic(1.5957691f * fmaf(0.044715f * x, x * x, x));
                const float inner = s * (1.0f - s);              // (0 where x is far out: then so is what it is multiplied with)
                v[i] = inner == 0.0f ? s : fmaf(x * inner, 1.5957691f * fmaf(3.0f * 0.044715f * x, x, 1.0f), s);
            }
            break;
        default:
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = 1.0f;
            break;
    }
}
inline bool activation_known(int kind) { return kind >= MINT_ACT_NONE && kind <= MINT_ACT_GELU_TANH; }

// Of a gate: none, sigmoid, tanh or silu, in as little code as that takes (it stands in many kernels).  At infinities silu and its slope are their limits: a gate
// of -inf shuts.
__device__ __forceinline__ float gate_value(int kind, float g) {
    if (kind == MINT_ACT_NONE) return g;
    if (kind == MINT_ACT_TANH) return tangent(g);
    return logistic(g) * (kind == MINT_ACT_SILU ? fmaxf(g, -FLT_MAX) : 1.0f);
}
__device__ __forceinline__ float gate_slope(int kind, float g) {
    if (kind == MINT_ACT_NONE) return 1.0f;
    if (kind == MINT_ACT_TANH) return tangent_slope(g);
    const float e = exponential(-fabsf(g)), r = reciprocal(1.0f + e), s = (g < 0.0f ? e : 1.0f) * r, slope = e * r * r;
    return kind == MINT_ACT_SILU ? (slope == 0.0f ? s : fmaf(g, slope, s)) : slope;
}
inline bool gate_known(int kind) { return kind == MINT_ACT_NONE || kind == MINT_ACT_SIGMOID || kind == MINT_ACT_TANH || kind == MINT_ACT_SILU; }

}  // namespace mint
