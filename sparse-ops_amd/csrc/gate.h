// The gated block's elementwise part: activations and their slopes in fp32.
#pragma once
#include "elements.h"
#include "so_internal.h"

namespace so_gate {

static inline bool known(int act) { return act >= SO_ACT_NONE && act <= SO_ACT_GELU_TANH; }

// 1 / (1 + exp(-v)) and what is left to 1, both to full relative precision.
struct Share { float of, rest; };
__device__ __forceinline__ Share logistic(float v)
{
    const float e = expf(-fabsf(v)), r = 1.0f / (1.0f + e), s = e * r;
    return v >= 0.0f ? Share{r, s} : v < 0.0f ? Share{s, r} : Share{v, v};      // NaN stays
}

constexpr float kRootHalf = 0.70710678f, kRootTwoOverPi = 0.79788456f, kCubic = 0.044715f, kNormal = 0.39894228f;      // 1 / sqrt(2), sqrt(2 / pi), 1 / sqrt(2 pi)

__device__ __forceinline__ float tanh_argument(float v) { return kRootTwoOverPi * fmaf(kCubic * v * v, v, v); }

// g[e] = act(g[e]) u[e].  The activation is the same for a whole launch, so that the branch on it costs a few scalar instructions.
template <int V>
__device__ __forceinline__ void apply(int act, float (&g)[V], const float (&u)[V])
{
    const auto each = [&](auto &&f) {
#pragma unroll
        for (int e = 0; e < V; ++e) g[e] = f(g[e]) * u[e];
    };
    switch (act) {
    case SO_ACT_RELU: return each([](float v) { return v <= 0.0f ? 0.0f : v; });
    case SO_ACT_SIGMOID: return each([](float v) { return logistic(v).of; });
    case SO_ACT_TANH: return each([](float v) { return tanhf(v); });
    case SO_ACT_SILU: return each([](float v) { return v * logistic(v).of; });
    case SO_ACT_GELU: return each([](float v) { return 0.5f * v * erfcf(-kRootHalf * v); });
    case SO_ACT_GELU_TANH: return each([](float v) { return v * logistic(2.0f * tanh_argument(v)).of; });
    default: return each([](float v) { return v; });
    }
}

struct Both { float value, slope; };
__device__ __forceinline__ Both value_and_slope(int act, float v)
{
    switch (act) {
    case SO_ACT_RELU: return {v <= 0.0f ? 0.0f : v, v <= 0.0f ? 0.0f : v > 0.0f ? 1.0f : v};
    case SO_ACT_SIGMOID: {
        const Share p = logistic(v);
        return {p.of, p.of * p.rest};
    }
    case SO_ACT_TANH: {
        const Share p = logistic(2.0f * v);
        return {tanhf(v), 4.0f * p.of * p.rest};
    }
    case SO_ACT_SILU: {
        const Share p = logistic(v);
        return {v * p.of, p.of * fmaf(v, p.rest, 1.0f)};
    }
    case SO_ACT_GELU: {
        const float below = 0.5f * erfcf(-kRootHalf * v), bell = kNormal * expf(-0.5f * v * v);
        return {v * below, bell == 0.0f ? below : fmaf(v, bell, below)};
    }
    case SO_ACT_GELU_TANH: {
        const Share p = logistic(2.0f * tanh_argument(v));
        const float both = p.of * p.rest;
        return {v * p.of, both == 0.0f ? p.of : fmaf(2.0f * v * both, kRootTwoOverPi * fmaf(3.0f * kCubic * v, v, 1.0f), p.of)};
    }
    default: return {v, 1.0f};
    }
}

} // namespace so_gate
