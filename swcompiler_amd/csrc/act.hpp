// The activations of the fully connected layer and their slopes, in fp32.
#pragma once
#include <hip/hip_runtime.h>

#include "swc_hip.h"

namespace swc_hip {

#if __HIP_DEVICE_COMPILE__
// 1 / (1 + e^-x).  e^-x overflows to infinity for x < -88, where the quotient is the right 0.
__device__ __forceinline__ float sigmoid(float x) { return 1.f / (1.f + expf(-x)); }

constexpr float kGeluC = 0.7978845608028654f;    // sqrt(2 / pi)
constexpr float kGeluA = 0.044715f;

// gelu(z) = z Phi(z); its tanh form 0.5 z (1 + tanh u) = z sigmoid(2 u), u = c (z + a z^3).
__device__ __forceinline__ float act_value(float z, int act) {
    switch (act) {
    case SWC_HIP_ACT_RELU: return z > 0.f ? z : 0.f;
    case SWC_HIP_ACT_GELU: return 0.5f * z * (1.f + erff(z * 0.7071067811865476f));
    case SWC_HIP_ACT_GELU_TANH: return z * sigmoid(2.f * kGeluC * (z + kGeluA * z * z * z));
    case SWC_HIP_ACT_SILU: return z * sigmoid(z);
    default: return z;
    }
}

// The slope at z.  The second terms vanish long before |z| = 40; z is held there so that infinities times zero do not
// make them NaN.
__device__ __forceinline__ float act_slope(float z, int act) {
    const float y = fminf(fmaxf(z, -40.f), 40.f);
    float s = 1.f;
    switch (act) {
    case SWC_HIP_ACT_RELU: return z > 0.f ? 1.f : 0.f;
    case SWC_HIP_ACT_GELU:
        s = 0.5f * (1.f + erff(y * 0.7071067811865476f)) + y * expf(-0.5f * y * y) * 0.3989422804014327f;
        break;
    case SWC_HIP_ACT_GELU_TANH: {
        const float p = sigmoid(2.f * kGeluC * (y + kGeluA * y * y * y));
        s = p + y * p * (1.f - p) * (2.f * kGeluC * (1.f + 3.f * kGeluA * y * y));
        break;
    }
    case SWC_HIP_ACT_SILU: {
        const float p = sigmoid(y);
        s = p * (1.f + y * (1.f - p));
        break;
    }
    default: return 1.f;
    }
    return z == z ? s : z;   // (fminf and fmaxf drop a NaN)
}
#endif

} // namespace swc_hip
