#pragma once
#include <hip/hip_runtime.h>

// Activations of the group norm and of the matrix products (SED_ACT_* of sed_hip.h) and their derivatives, on the hardware's exp2 and
// reciprocal (1 ulp each).  GELU is z Phi(z) with Phi(-u) = t P(t) exp(-u^2 / 2), t = 1 / (1 + 0.35 u): one exponential, which the derivative
// Phi(z) + z phi(z) shares.  P is the polynomial of degree 8 with the least largest relative error from u = 0 to 14, fitted here in 64 bits
// (3.2e-8); in 32 bits z Phi(z) is off by 0.9e-7 at most for negative z, by 2e-6 of itself down to z = -6, and by 5e-7 of itself for positive z.
__device__ __forceinline__ float sed_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }
__device__ __forceinline__ float sed_sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + sed_exp(-z)); }
__device__ __forceinline__ float sed_phi_cdf(float z, float e) {          // Phi(z), e = exp(-z^2 / 2)
    const float t = __builtin_amdgcn_rcpf(fmaf(0.35f, fabsf(z), 1.f));
    float q = fmaf(t, -0.0291456636f, 0.143970504f);
    q = fmaf(t, q, -0.255711973f);
    q = fmaf(t, q, 0.159171775f);
    q = fmaf(t, q, -0.0231083408f);
    q = fmaf(t, q, 0.105507433f);
    q = fmaf(t, q, 0.119833f);
    q = fmaf(t, q, 0.139861852f);
    q = fmaf(t, q, 0.139621407f);
    q *= t * e;
    return z < 0.f ? q : 1.f - q;
}
template <int ACT> __device__ __forceinline__ float sed_act(float z) {
    if (ACT == 1) return z > 0.f ? z : (z == z ? 0.f : z);
    if (ACT == 2) return z * sed_sigmoid(z);
    if (ACT == 3) return z * sed_phi_cdf(z, sed_exp(-0.5f * z * z));
    return z;
}
template <int ACT> __device__ __forceinline__ float sed_act_grad(float z) {
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
// gy act'(z).  ReLU selects: an infinite gy is 0 where z is not positive, and passes where z is NaN, as in torch
template <int ACT> __device__ __forceinline__ float sed_act_gz(float gy, float z) {
    if (ACT == 1) return z <= 0.f ? 0.f : gy;
    return gy * sed_act_grad<ACT>(z);
}
