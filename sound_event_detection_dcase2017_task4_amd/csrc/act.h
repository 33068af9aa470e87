#pragma once
#include <hip/hip_runtime.h>

// Activations of the group norm and of the matrix products (SED_ACT_* of sed_hip.h) and their derivatives, on the hardware's exp2 and
// reciprocal (1 ulp each).  GELU is z Phi(z) with the error function by formula 7.1.26 of Abramowitz and Stegun (|error| <= 1.5e-7):
// one exponential, which the derivative Phi(z) + z phi(z) shares.
__device__ __forceinline__ float sed_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }
__device__ __forceinline__ float sed_sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + sed_exp(-z)); }
__device__ __forceinline__ float sed_phi_cdf(float z, float e) {          // Phi(z), e = exp(-z^2 / 2)
    const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f * 0.70710678118654752f, fabsf(z), 1.f));
    float q = fmaf(t, 1.061405429f, -1.453152027f);
    q = fmaf(t, q, 1.421413741f);
    q = fmaf(t, q, -0.284496736f);
    q = fmaf(t, q, 0.254829592f);
    q *= 0.5f * t * e;                                                   // (1 - erf(|z| / sqrt(2))) / 2
    return z < 0.f ? q : 1.f - q;
}
template <int ACT> __device__ __forceinline__ float sed_act(float z) {
    if (ACT == 1) return z > 0.f ? z : (z == z ? 0.f : z);
    if (ACT == 2) return z * sed_sigmoid(z);
    if (ACT == 3) return z * sed_phi_cdf(z, sed_exp(-0.5f * z * z));
    return z;
}
template <int ACT> __device__ __forceinline__ float sed_act_grad(float z) {
    if (ACT == 1) return z > 0.f ? 1.f : 0.f;
    if (ACT == 2) {
        const float s = sed_sigmoid(z);
        return s * fmaf(z, 1.f - s, 1.f);
    }
    if (ACT == 3) {
        const float e = sed_exp(-0.5f * z * z);
        return fmaf(z * e, 0.39894228040143268f, sed_phi_cdf(z, e));
    }
    return 1.f;
}
