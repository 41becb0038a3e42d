// The dense linear layer's activations and their slopes, in float32.
#pragma once

#include "wf_common.cuh"
#include "wf_pairs.cuh"

namespace wf {
namespace {

constexpr float kInvSqrt2Pi = 0.39894228f;     // 1 / sqrt(2 pi)
constexpr float kSqrt2OverPi = 0.79788456f;    // sqrt(2 / pi)
constexpr float kGeluCubic = 0.044715f;

// 1 / x and exp(x) by the hardware's approximations (a step or two of float32; tiny results flush to 0, and 1 / infinity
// is 0: the limits that the formulas below want)
__device__ __forceinline__ float fast_rcp(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float fast_exp(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x * 1.44269504f));
    return r;
}

// 1 / (1 + exp(-v))
__device__ __forceinline__ float sigmoid(float v) { return fast_rcp(1.0f + fast_exp(-v)); }

// The normal distribution function of two values: 0.5 + v g(v^2), g the minimax polynomial (weighted by v) of degree 14
// in s = 2 (v / 5.25)^2 - 1, fitted on |v| <= 5.25. Off by at most 1.1e-7, evaluated in float32, over all v (0.5 (1 + erf)
// in float32: 0.6e-7); relative to the value that is 4e-4 at -3.5, 1.5e-3 at -4 and 1.8e-2 at -4.5. Past 5.25
// its leading term drives the sum out of [0, 1], where it is clamped. Packed multiply-adds alone: erff, or an exp and a
// reciprocal (16 cycles a warp on the special-function unit), held up the product (8192 x 512 x 8192 with gelu: 137 us
// with them).
__device__ __forceinline__ void normal_cdf2(float v0, float v1, float &c0, float &c1) {
    constexpr float c[15] = {0.13465934991836548f,   -0.0671268180012703f,   0.04964578524231911f,  -0.03976341336965561f,
                             0.03203143924474716f,   -0.025041932240128517f, 0.018538648262619972f, -0.012775249779224396f,
                             0.008417869918048382f,  -0.005448520183563232f, 0.002892362419515848f, -0.0010395343415439129f,
                             0.0006647314294241369f, -0.0006565839285030961f, 0.0002399503719061613f};
    const uint64_t v = pack_f2(v0, v1);
    const uint64_t s = fma_f2(mul_f2(v, v), pack_f2(0.07256235927343369f, 0.07256235927343369f), pack_f2(-1.f, -1.f));
    uint64_t g = pack_f2(c[14], c[14]);
#pragma unroll
    for (int i = 13; i >= 0; --i) g = fma_f2(g, s, pack_f2(c[i], c[i]));
    float g0, g1;
    unpack_f2(g, g0, g1);
    c0 = __saturatef(fmaf(v0, g0, 0.5f));
    c1 = __saturatef(fmaf(v1, g1, 0.5f));
}

// act(v) of two values. relu keeps NaN; gelu is the erf form; gelu_tanh is 0.5 v (1 + tanh(u)) = v sigmoid(2 u).
template <int ACT>
__device__ __forceinline__ void act2(float &v0, float &v1) {
    if constexpr (ACT == WF_ACT_RELU) {
        v0 = v0 < 0.f ? 0.f : v0;
        v1 = v1 < 0.f ? 0.f : v1;
    } else if constexpr (ACT == WF_ACT_SILU) {
        v0 *= sigmoid(v0);
        v1 *= sigmoid(v1);
    } else if constexpr (ACT == WF_ACT_GELU) {
        float c0, c1;
        normal_cdf2(v0, v1, c0, c1);
        v0 *= c0;
        v1 *= c1;
    } else if constexpr (ACT == WF_ACT_GELU_TANH) {
        v0 *= sigmoid(2.0f * kSqrt2OverPi * fmaf(kGeluCubic * v0 * v0, v0, v0));
        v1 *= sigmoid(2.0f * kSqrt2OverPi * fmaf(kGeluCubic * v1 * v1, v1, v1));
    }
}

// act(v) and act'(v) of two values
template <int ACT>
__device__ __forceinline__ void act_slope2(const float (&v)[2], float (&h)[2], float (&slope)[2]) {
    if constexpr (ACT == WF_ACT_GELU) {
        float c[2];
        normal_cdf2(v[0], v[1], c[0], c[1]);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            h[i] = v[i] * c[i];
            slope[i] = fmaf(v[i] * kInvSqrt2Pi, fast_exp(-0.5f * v[i] * v[i]), c[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if constexpr (ACT == WF_ACT_RELU) {
                h[i] = v[i] < 0.f ? 0.f : v[i];
                slope[i] = v[i] > 0.f ? 1.f : 0.f;
            } else if constexpr (ACT == WF_ACT_SILU) {
                const float p = sigmoid(v[i]);
                h[i] = v[i] * p;
                slope[i] = fmaf(h[i], 1.f - p, p);
            } else if constexpr (ACT == WF_ACT_GELU_TANH) {
                const float v2 = v[i] * v[i], p = sigmoid(2.0f * kSqrt2OverPi * fmaf(kGeluCubic * v2, v[i], v[i]));
                h[i] = v[i] * p;
                // past |v| = 1e4 the slope is p alone; the square must not overflow to 0 * infinity
                slope[i] = fmaf(h[i] * (1.f - p), 2.0f * kSqrt2OverPi * fmaf(3.0f * kGeluCubic, fminf(v2, 1e8f), 1.f), p);
            } else {
                h[i] = v[i];
                slope[i] = 1.f;
            }
        }
    }
}

}  // namespace
}  // namespace wf
