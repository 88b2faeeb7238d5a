// The gated block's elementwise part: activations and their slopes in fp32.
#pragma once
#include <type_traits>

#include "elements.h"
#include "so_internal.h"

namespace so_gate {

static inline bool known(int act) { return act >= SO_ACT_NONE && act <= SO_ACT_GELU_TANH; }

constexpr float kLog2e = 1.44269504f, kRootHalf = 0.70710678f, kRootTwoOverPi = 0.79788456f, kCubic = 0.044715f, kNormal = 0.39894228f;      // 1 / sqrt(2), sqrt(2 / pi), 1 / sqrt(2 pi)

// 1 / (1 + exp(-v)).  For results of 16 bits by the exponential and the reciprocal of the vector unit, a step each.  Rounding v log2 e costs |v| steps of the exponential, which matter only where that is small
// beside 1 (v > 0) or the result is as small as it (v < 0): v times it is within 2^-23 for all v.  expf and a division, 25 instructions more, made the forward pass of 8192 x 4096 x 4096 bf16
// 45 us slower.  For fp32, whose results are to be right to their own last bits, those, and of a negative v the exponential that cannot overflow.
template <bool HALF>
__device__ __forceinline__ float logistic(float v)
{
    if constexpr (HALF) return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2e * v));
    const float e = expf(-fabsf(v));
    return (v < 0.0f ? e : 1.0f) / (1.0f + e);
}

// That and what is left to 1, both to a few steps of their own.
struct Share { float of, rest; };
template <bool HALF>
__device__ __forceinline__ Share shares(float v)
{
    float r, s;
    if constexpr (HALF) {
        const float e = __builtin_amdgcn_exp2f(-kLog2e * fabsf(v));
        r = __builtin_amdgcn_rcpf(1.0f + e);
        s = e * r;
    } else {
        const float e = expf(-fabsf(v));
        r = 1.0f / (1.0f + e);
        s = e / (1.0f + e);
    }
    return v >= 0.0f ? Share{r, s} : Share{s, r};
}

__device__ __forceinline__ float tanh_argument(float v) { return kRootTwoOverPi * fmaf(kCubic * v * v, v, v); }

// The normal distribution.  For results of 16 bits its tail exp(-z^2) q(t) / 2, t = 1 / (1 + 3 z / 8), z = |v| / sqrt(2), with the polynomial q of degree 7 without a constant that is nearest to exp(z^2) erfc(z) relative
// to it for z up to 10 (least squares whose weights follow the error): within 2^-19.9 of itself as fp32 evaluates it, so that gelu of numbers far below 0 is right to its own last bit too.
template <bool HALF>
__device__ __forceinline__ float normal(float v)
{
    if constexpr (!HALF) return 0.5f * erfcf(-kRootHalf * v);
    const float z = kRootHalf * fabsf(v), t = __builtin_amdgcn_rcpf(fmaf(0.375f, z, 1.0f));
    const float q = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, -0.13509569f, 0.38793707f), -0.12959625f), 0.2830608f), 0.16666485f), 0.21568912f), 0.21133946f);
    const float tail = 0.5f * q * __builtin_amdgcn_exp2f(-kLog2e * z * z);
    return v > 0.0f ? 1.0f - tail : tail;
}

// Its density.  In fp32 what rounding v v leaves, v^2 / 2 steps of the exponential, is put back.
template <bool HALF>
__device__ __forceinline__ float bell(float v)
{
    if constexpr (HALF) return kNormal * __builtin_amdgcn_exp2f(-0.5f * kLog2e * v * v);
    const float square = v * v, e = expf(-0.5f * square);
    return e == 0.0f ? 0.0f : kNormal * fmaf(-0.5f * fmaf(v, v, -square), e, e);
}

// f(function of v) for the activation, the same for a whole launch, so that the branch on it costs a few scalar instructions.
template <bool HALF, class F>
__device__ __forceinline__ void with(int act, F &&f)
{
    switch (act) {
    case SO_ACT_RELU: return f([](float v) { return v <= 0.0f ? 0.0f : v; });
    case SO_ACT_SIGMOID: return f([](float v) { return logistic<HALF>(v); });
    case SO_ACT_TANH: return f([](float v) { return tanhf(v); });
    case SO_ACT_SILU: return f([](float v) { return v * logistic<HALF>(v); });
    case SO_ACT_GELU: return f([](float v) { return v * normal<HALF>(v); });
    case SO_ACT_GELU_TANH: return f([](float v) { return v * logistic<HALF>(2.0f * tanh_argument(v)); });
    default: return f([](float v) { return v; });
    }
}

// g[e] = act(g[e]) u[e], for results of type T.
template <class T, int V>
__device__ __forceinline__ void apply(int act, float (&g)[V], const float (&u)[V])
{
    with<sizeof(T) == 2>(act, [&](auto value) {
#pragma unroll
        for (int e = 0; e < V; ++e) g[e] = value(g[e]) * u[e];
    });
}

// The same with slopes: f(function of v).
struct Both { float value, slope; };
template <bool HALF, class F>
__device__ __forceinline__ void with_slope(int act, F &&f)
{
    switch (act) {
    case SO_ACT_RELU: return f([](float v) { return Both{v <= 0.0f ? 0.0f : v, v <= 0.0f ? 0.0f : v > 0.0f ? 1.0f : v}; });
    case SO_ACT_SIGMOID: return f([](float v) {
        const Share p = shares<HALF>(v);
        return Both{p.of, p.of * p.rest};
    });
    case SO_ACT_TANH: return f([](float v) {
        const Share p = shares<HALF>(2.0f * v);
        return Both{tanhf(v), 4.0f * p.of * p.rest};
    });
    case SO_ACT_SILU: return f([](float v) {
        const Share p = shares<HALF>(v);
        return Both{v * p.of, p.of * fmaf(v, p.rest, 1.0f)};
    });
    case SO_ACT_GELU: return f([](float v) {
        const float below = normal<HALF>(v), beside = bell<HALF>(v);
        return Both{v * below, beside == 0.0f ? below : fmaf(v, beside, below)};
    });
    case SO_ACT_GELU_TANH: return f([](float v) {
        const Share p = shares<HALF>(2.0f * tanh_argument(v));
        const float both = p.of * p.rest;
        return Both{v * p.of, both == 0.0f ? p.of : fmaf(2.0f * v * both, kRootTwoOverPi * fmaf(3.0f * kCubic * v, v, 1.0f), p.of)};
    });
    default: return f([](float v) { return Both{v, 1.0f}; });
    }
}

} // namespace so_gate
