// The gated block's activations, their slopes, and where their numbers come from.
//
//   silu       g s(g)                              s(z) = 1 / (1 + exp(-z))
//   gelu       g P(g)                              P the normal distribution's function, (1 + erf(g / sqrt 2)) / 2
//   gelu_tanh  g s(z),  z = sqrt(8 / pi) (g + 0.044715 g^3), since (1 + tanh(z / 2)) / 2 = s(z)
//
// In fp32 with the exponential and reciprocal instructions, within a few ulp: results are rounded to 16 bits.
#pragma once

#include <hip/hip_runtime.h>

namespace feather {

enum Activation : int { kSilu = 0, kGelu = 1, kGeluTanh = 2 };

struct Slope {
    float value, slope;
};

// s(z) and 1 - s(z), each from exp(-|z|), so that neither loses its bits where it is small.
struct Logistic {
    float s, c;
};

__device__ __forceinline__ Logistic logistic(float z) {
    const float root = __expf(-0.5f * fabsf(z));   // squared: its square reaches below the least normal with all its bits
    const float t = root * root;
    const float q = __builtin_amdgcn_rcpf(1.0f + t);
    const float tq = t * q;
    return z < 0.0f ? Logistic{tq, q} : Logistic{q, tq};
}

// a * s for a factor s that may be 0 where a is infinite or the type's lowest value: 0 and not NaN.
__device__ __forceinline__ float faded(float a, float s) { return s == 0.0f ? 0.0f * s : a * s; }

constexpr float kTanhSlope = 1.5957691216057308f;   // sqrt(8 / pi)
constexpr float kTanhCube = 0.044715f;
constexpr float kRootHalf = 0.70710678118654752f;
constexpr float kNormalDensity = 0.39894228040143268f;   // 1 / sqrt(2 pi)

// P(g), without the cancellation of 1 + erf at negative g.
__device__ __forceinline__ float normal_function(float g) { return 0.5f * erfcf(-g * kRootHalf); }

template <int kAct>
__device__ __forceinline__ float activate(float g) {
    if constexpr (kAct == kSilu) return faded(g, logistic(g).s);
    if constexpr (kAct == kGelu) return faded(g, normal_function(g));
    const float z = kTanhSlope * (g + kTanhCube * g * g * g);
    return faded(g, logistic(z).s);
}

template <int kAct>
__device__ __forceinline__ Slope activate_with_slope(float g) {
    if constexpr (kAct == kSilu) {
        const Logistic l = logistic(g);
        const float value = faded(g, l.s);
        return {value, l.s + faded(value, l.c)};
    }
    if constexpr (kAct == kGelu) {
        const float p = normal_function(g);
        return {faded(g, p), p + faded(g, kNormalDensity * __expf(-0.5f * g * g))};
    }
    const float z = kTanhSlope * (g + kTanhCube * g * g * g);
    const Logistic l = logistic(z);
    return {faded(g, l.s), l.s + faded(g * kTanhSlope * (1.0f + 3.0f * kTanhCube * g * g), l.s * l.c)};
}

}  // namespace feather
