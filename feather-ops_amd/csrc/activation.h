// The gated block's activations, their slopes, and where their numbers come from.
//
//   silu       g s(g)                              s(z) = 1 / (1 + exp(-z))
//   gelu       g P(g)                              P the normal distribution's function, (1 + erf(g / sqrt 2)) / 2
//   gelu_tanh  g s(z),  z = sqrt(8 / pi) (g + 0.044715 g^3), since (1 + tanh(z / 2)) / 2 = s(z)
//
// In fp32 with the exponential and reciprocal instructions; results are rounded to 16 bits. What errs most is the rounding of an
// exponential's argument, which grows with it: relative to their value s(z) is off by 2^-20.5 at most down to z = -8, 2^-19 to -40
// and 2^-18 to -86, P(g) by 2^-19.3 down to g = -3, 2^-18.7 to -6 and 2^-17 to -13 (the steps emulated in fp32 against 64 bits). At the
// end of a 256 x 256 tile one wave a SIMD does this for 128 values a lane, with nothing beside it. gelu by the library's erfc, some
// 60 instructions: 4097 x 2576 -> 5000 242 us, by the polynomial below 230.
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

// a * s for a factor s that may be 0 where a is infinite: 0 and not NaN.
__device__ __forceinline__ float faded(float a, float s) { return (s == 0.0f ? 0.0f : a) * s; }

constexpr float kTanhSlope = 1.5957691216057308f;   // sqrt(8 / pi)
constexpr float kTanhCube = 0.044715f;
constexpr float kNormalDensity = 0.39894228040143268f;   // 1 / sqrt(2 pi)

struct Normal {
    float p, density;   // P(g) and P'(g)
};

// With t = |g|, P(-t) exp(t^2 / 2) is smooth and falls from 1 / 2 like 1 / t: a polynomial in u = 1 / (1 + 0.36 t) without a
// constant, fitted to the least relative error over t up to 14.5 (1e-6 before fp32's roundings), where the exponential ends.
__device__ __forceinline__ Normal normal(float g) {
    const float t = fabsf(g);
    const float root = __expf(-0.25f * t * t);
    const float e = root * root;
    const float u = __builtin_amdgcn_rcpf(__builtin_fmaf(0.36f, t, 1.0f));
    float r = 0.04678545892238617f;
    r = __builtin_fmaf(r, u, -0.1788369119167328f);
    r = __builtin_fmaf(r, u, 0.17969179153442383f);
    r = __builtin_fmaf(r, u, 0.02741684578359127f);
    r = __builtin_fmaf(r, u, 0.13940362632274628f);
    r = __builtin_fmaf(r, u, 0.1418297439813614f);
    r = __builtin_fmaf(r, u, 0.14370901882648468f);
    const float tail = r * u * e;
    return {g < 0.0f ? tail : 1.0f - tail, kNormalDensity * e};
}

template <int kAct>
__device__ __forceinline__ float activate(float g) {
    if constexpr (kAct == kSilu) return faded(g, logistic(g).s);
    if constexpr (kAct == kGelu) return faded(g, normal(g).p);
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
        const Normal n = normal(g);
        return {faded(g, n.p), n.p + faded(g, n.density)};
    }
    const float z = kTanhSlope * (g + kTanhCube * g * g * g);
    const Logistic l = logistic(z);
    return {faded(g, l.s), l.s + faded(g * kTanhSlope * (1.0f + 3.0f * kTanhCube * g * g), l.s * l.c)};
}

}  // namespace feather
