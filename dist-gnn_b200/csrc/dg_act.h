// Activations of the linear layer and their derivatives, in fp32.
#pragma once
#include "dist_gnn_b200.h"

namespace dg {

// gelu(z) = z Phi(z) with the distribution function of the normal distribution, silu(z) = z / (1 + exp(-z)).
template <int ACT> __device__ __forceinline__ float act_value(float z)
{
    if (ACT == DG_ACT_RELU) return z > 0.f || z != z ? z : 0.f;       // a NaN stays
    if (ACT == DG_ACT_GELU) return z * fmaf(0.5f, erff(z * 0.70710678f), 0.5f);
    if (ACT == DG_ACT_SILU) return z * __frcp_rn(1.f + __expf(-z));
    return z;
}
// d act / dz:  Phi + z phi,  s (1 + z (1 - s)).
template <int ACT> __device__ __forceinline__ float act_slope(float z)
{
    if (ACT == DG_ACT_RELU) return z > 0.f ? 1.f : 0.f;
    if (ACT == DG_ACT_GELU) return fmaf(0.5f, erff(z * 0.70710678f), 0.5f) + z * 0.39894228f * __expf(-0.5f * z * z);
    if (ACT == DG_ACT_SILU) {
        const float s = __frcp_rn(1.f + __expf(-z));
        return s * fmaf(z, 1.f - s, 1.f);
    }
    return 1.f;
}

}  // namespace dg
