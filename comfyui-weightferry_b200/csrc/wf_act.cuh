// The dense linear layer's activations and their slopes, in float32.
#pragma once

#include "wf_common.cuh"

namespace wf {
namespace {

constexpr float kSqrtHalf = 0.70710678f;       // 1 / sqrt(2)
constexpr float kInvSqrt2Pi = 0.39894228f;     // 1 / sqrt(2 pi)
constexpr float kSqrt2OverPi = 0.79788456f;    // sqrt(2 / pi)
constexpr float kGeluCubic = 0.044715f;

// 1 / (1 + exp(-v)); exp's overflow to infinity gives the right limit, 0
__device__ __forceinline__ float sigmoid(float v) { return __fdividef(1.0f, 1.0f + __expf(-v)); }

// act(v). relu keeps NaN; gelu is the erf form; gelu_tanh is 0.5 v (1 + tanh(u)) = v sigmoid(2 u).
template <int ACT>
__device__ __forceinline__ float act(float v) {
    if constexpr (ACT == WF_ACT_RELU) return v < 0.f ? 0.f : v;
    else if constexpr (ACT == WF_ACT_SILU) return v * sigmoid(v);
    else if constexpr (ACT == WF_ACT_GELU) return 0.5f * v * (1.0f + erff(v * kSqrtHalf));
    else if constexpr (ACT == WF_ACT_GELU_TANH) return v * sigmoid(2.0f * kSqrt2OverPi * fmaf(kGeluCubic * v * v, v, v));
    else return v;
}

// act(v) and act'(v)
template <int ACT>
__device__ __forceinline__ void act_slope(float v, float &h, float &slope) {
    if constexpr (ACT == WF_ACT_RELU) {
        h = v < 0.f ? 0.f : v;
        slope = v > 0.f ? 1.f : 0.f;
    } else if constexpr (ACT == WF_ACT_SILU) {
        const float p = sigmoid(v);
        h = v * p;
        slope = fmaf(h, 1.f - p, p);
    } else if constexpr (ACT == WF_ACT_GELU) {
        const float cdf = fmaf(0.5f, erff(v * kSqrtHalf), 0.5f);
        h = v * cdf;
        slope = fmaf(v * kInvSqrt2Pi, __expf(-0.5f * v * v), cdf);
    } else if constexpr (ACT == WF_ACT_GELU_TANH) {
        const float p = sigmoid(2.0f * kSqrt2OverPi * fmaf(kGeluCubic * v * v, v, v));
        h = v * p;
        const float v2 = fminf(v * v, 1e8f);  // past |v| = 1e4 the slope is p alone; the square must not overflow to 0 * inf
        slope = fmaf(h * (1.f - p), 2.0f * kSqrt2OverPi * fmaf(3.0f * kGeluCubic, v2, 1.f), p);
    } else {
        h = v;
        slope = 1.f;
    }
}

}  // namespace
}  // namespace wf
