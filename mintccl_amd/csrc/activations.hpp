// Activations and their slopes, of gates (norms.hip) and of products (dense.hip), in 32 bits.  Which one is uniform over a
// launch.  No counterpart in the reference.
#pragma once
#include "operators.hpp"

namespace mint {

__device__ __forceinline__ float logistic(float x) { return 1.0f / (1.0f + expf(-x)); }

// MINT_ACT_GELU is x * P(N <= x) of a normal N, MINT_ACT_GELU_TANH the approximation of it by a hyperbolic tangent.
__device__ __forceinline__ float activated(int kind, float x) {
    switch (kind) {
        case MINT_ACT_RELU: return x > 0.0f || x != x ? x : 0.0f;
        case MINT_ACT_SILU: return x * logistic(x);
        case MINT_ACT_SIGMOID: return logistic(x);
        case MINT_ACT_TANH: return tanhf(x);
        case MINT_ACT_GELU: return 0.5f * x * erfcf(-0.70710678f * x);
        case MINT_ACT_GELU_TANH: return 0.5f * x * (1.0f + tanhf(0.79788456f * (x + 0.044715f * x * x * x)));
        default: return x;
    }
}
__device__ __forceinline__ float slope_of(int kind, float x) {
    switch (kind) {
        case MINT_ACT_RELU: return x > 0.0f ? 1.0f : x != x ? x : 0.0f;
        case MINT_ACT_SILU: {
            const float s = logistic(x);
            return s * (1.0f + x * (1.0f - s));
        }
        case MINT_ACT_SIGMOID: {
            const float e = expf(-fabsf(x));             // (of either sign without a difference that cancels)
            return e / ((1.0f + e) * (1.0f + e));
        }
        case MINT_ACT_TANH: {
            const float t = tanhf(x);
            return 1.0f - t * t;
        }
        case MINT_ACT_GELU: return 0.5f * erfcf(-0.70710678f * x) + x * (0.39894228f * expf(-0.5f * x * x));
        case MINT_ACT_GELU_TANH: {
            const float t = tanhf(0.79788456f * (x + 0.044715f * x * x * x));
            return 0.5f * (1.0f + t) + 0.5f * x * (1.0f - t * t) * (0.79788456f * (1.0f + 3.0f * 0.044715f * x * x));
        }
        default: return 1.0f;
    }
}
// Of a gate: none, sigmoid, tanh or silu, in as little code as that takes (it stands in many kernels).
__device__ __forceinline__ float gate_value(int kind, float g) {
    if (kind == MINT_ACT_NONE) return g;
    if (kind == MINT_ACT_TANH) return tanhf(g);
    return logistic(g) * (kind == MINT_ACT_SILU ? g : 1.0f);
}
__device__ __forceinline__ float gate_slope(int kind, float g) {
    if (kind == MINT_ACT_NONE) return 1.0f;
    if (kind == MINT_ACT_TANH) {
        const float t = tanhf(g);
        return 1.0f - t * t;
    }
    const float e = expf(-fabsf(g)), s = (g < 0.0f ? e : 1.0f) / (1.0f + e), slope = e / ((1.0f + e) * (1.0f + e));
    return kind == MINT_ACT_SILU ? fmaf(g, slope, s) : slope;
}
inline bool gate_known(int kind) { return kind == MINT_ACT_NONE || kind == MINT_ACT_SIGMOID || kind == MINT_ACT_TANH || kind == MINT_ACT_SILU; }
inline bool activation_known(int kind) { return kind >= MINT_ACT_NONE && kind <= MINT_ACT_GELU_TANH; }

}  // namespace mint
