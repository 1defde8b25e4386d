// The activations of the fully connected layer and their slopes, in fp32.
#pragma once
#include <hip/hip_runtime.h>

#include "swc_hip.h"

namespace swc_hip {

#if __HIP_DEVICE_COMPILE__
// Where the result is rounded to bfloat16 (FAST) the exponential, the reciprocal and Phi are good to some 5e-7 of
// themselves, on the exponential and reciprocal instructions; in fp32 they are the library functions.
//
// 1 / (1 + e^-x).  e^-x overflows to infinity for x < -88, where the quotient is the right 0.
template <bool FAST> __device__ __forceinline__ float sigmoid(float x) {
    if (FAST) return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * -1.44269504088896340736f));
    return 1.f / (1.f + expf(-x));
}

// The normal distribution Phi(z) and e^(-z^2/2).  For x = |z|: Phi(-x) = e^(-x^2/2) P(t), t = 1 / (1 + 0.31 x), with P of
// degree 8 fitted to the scaled complementary error function on [0, 15] (weighted least squares until the relative error
// levels out: 1.7e-7, 4.6e-7 evaluated in fp32); Phi(z) = 1 - Phi(-z) on the right keeps both tails.
template <bool FAST> __device__ __forceinline__ float normal_cdf(float z, float &bell) {
    if (FAST) {
        const float x = fabsf(z);
        bell = __builtin_amdgcn_exp2f(z * z * -0.72134752044448170368f);
        const float t = __builtin_amdgcn_rcpf(fmaf(0.31f, x, 1.f));
        float p = 0.03589478135108948f;
        p = fmaf(p, t, -0.14183589816093445f);
        p = fmaf(p, t, 0.15548671782016754f);
        p = fmaf(p, t, -0.015310253947973251f);
        p = fmaf(p, t, 0.11033819615840912f);
        p = fmaf(p, t, 0.10769762098789215f);
        p = fmaf(p, t, 0.12407287955284119f);
        p = fmaf(p, t, 0.12365604192018509f);
        p = p * t * bell;
        return z < 0.f ? p : 1.f - p;
    }
    bell = expf(-0.5f * z * z);
    return 0.5f * (1.f + erff(z * 0.7071067811865476f));
}

constexpr float kGeluC = 0.7978845608028654f;    // sqrt(2 / pi)
constexpr float kGeluA = 0.044715f;

// gelu(z) = z Phi(z); its tanh form 0.5 z (1 + tanh u) = z sigmoid(2 u), u = c (z + a z^3).
template <int ACT, bool FAST> __device__ __forceinline__ float act_value(float z) {
    if (ACT == SWC_HIP_ACT_RELU) return z > 0.f ? z : 0.f;
    if (ACT == SWC_HIP_ACT_GELU) {
        float bell;
        return z * normal_cdf<FAST>(z, bell);
    }
    if (ACT == SWC_HIP_ACT_GELU_TANH) return z * sigmoid<FAST>(2.f * kGeluC * (z + kGeluA * z * z * z));
    if (ACT == SWC_HIP_ACT_SILU) return z * sigmoid<FAST>(z);
    return z;
}

// The slope of a smooth activation at z.  The second terms vanish long before |z| = 40; z is held there so that infinities times zero do not
// make them NaN.
template <int ACT, bool FAST> __device__ __forceinline__ float act_slope(float z) {
    static_assert(ACT >= SWC_HIP_ACT_GELU, "the others have no slope to compute");
    const float y = fminf(fmaxf(z, -40.f), 40.f);
    float s = 1.f;
    if (ACT == SWC_HIP_ACT_GELU) {
        float bell;
        const float p = normal_cdf<FAST>(y, bell);
        s = p + y * bell * 0.3989422804014327f;
    } else if (ACT == SWC_HIP_ACT_GELU_TANH) {
        const float p = sigmoid<FAST>(2.f * kGeluC * (y + kGeluA * y * y * y));
        s = p + y * p * (1.f - p) * (2.f * kGeluC * (1.f + 3.f * kGeluA * y * y));
    } else {
        const float p = sigmoid<FAST>(y);
        s = p * (1.f + y * (1.f - p));
    }
    return z == z ? s : z;   // (fminf and fmaxf drop a NaN)
}

// The gradient g of a value, taken to its argument z.  An inactive ReLU passes nothing on, not even infinities and NaN (as
// reluGrad_f): in the products behind it one of them would fill a row and a column.
template <int ACT, bool FAST> __device__ __forceinline__ float act_grad_value(float z, float g) {
    if constexpr (ACT == SWC_HIP_ACT_RELU) return z > 0.f ? g : 0.f;
    else return g * act_slope<ACT, FAST>(z);
}
#endif

inline bool known_act(int act) { return act >= SWC_HIP_ACT_NONE && act <= SWC_HIP_ACT_SILU; }

// Calls f with the activation as a compile-time constant.
template <class F> int with_act(int act, F f) {
    switch (act) {
    case SWC_HIP_ACT_RELU: return f.template operator()<SWC_HIP_ACT_RELU>();
    case SWC_HIP_ACT_GELU: return f.template operator()<SWC_HIP_ACT_GELU>();
    case SWC_HIP_ACT_GELU_TANH: return f.template operator()<SWC_HIP_ACT_GELU_TANH>();
    case SWC_HIP_ACT_SILU: return f.template operator()<SWC_HIP_ACT_SILU>();
    default: return f.template operator()<SWC_HIP_ACT_NONE>();
    }
}

} // namespace swc_hip
