// Activations of the linear layer and their derivatives, in fp32.
#pragma once
#include "dist_gnn_b200.h"
#include "dg_pair.h"

namespace dg {

// Phi(z) and e = exp(-z^2 / 2) by Hastings' formula (Abramowitz and Stegun, Handbook of Mathematical Functions, 7.1.26): Phi(-|z|) = t (a1 + t (a2 + ... a5)) e / 2
// with t = 1 / (1 + p |z| / sqrt 2), off by at most 7.5e-8.  No branches, and the density that the derivative needs comes with it: against erff, whose two
// branches diverge, the forward pass of 2,449,029 x 256 -> 256 bf16 went from 1,329 us to 975 and the gradient's pass from 1,101 to 874.
__device__ __forceinline__ float normal_cdf(float z, float* e)
{
    const float t = reciprocal(fmaf(0.3275911f * 0.70710678f, fabsf(z), 1.f));
    float p = fmaf(t, 0.5f * 1.061405429f, 0.5f * -1.453152027f);
    p = fmaf(t, p, 0.5f * 1.421413741f);
    p = fmaf(t, p, 0.5f * -0.284496736f);
    p = fmaf(t, p, 0.5f * 0.254829592f);
    *e = exp2_approx(z * z * -0.72134752f);
    const float tail = p * t * *e;
    return z > 0.f ? 1.f - tail : tail;
}
__device__ __forceinline__ float sigmoid(float z)
{
    return reciprocal(1.f + exp2_approx(z * -1.44269504f));
}
// z within [low, high]; a NaN stays one.  SiLU multiplies its sigmoid by a z so bounded: beyond, an s that is a rounding away from 0 or 1 would count |z| times.
__device__ __forceinline__ float bounded(float z, float low, float high)
{
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(z) : "f"(low));
    asm("min.NaN.f32 %0, %0, %1;" : "+f"(z) : "f"(high));
    return z;
}
__device__ __forceinline__ float at_least(float z, float low)
{
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(z) : "f"(low));
    return z;
}

// gelu(z) = z Phi(z) with the distribution function of the normal distribution, silu(z) = z / (1 + exp(-z)).
template <int ACT> __device__ __forceinline__ float act_value(float z)
{
    if (ACT == DG_ACT_RELU) return z > 0.f || z != z ? z : 0.f;       // a NaN stays
    if (ACT == DG_ACT_GELU) {
        float e;
        return z * normal_cdf(z, &e);
    }
    if (ACT == DG_ACT_SILU) return at_least(z, -104.f) * sigmoid(z);      // -infinity gives zero, as do numbers from -104 on
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
        return s * fmaf(bounded(z, -104.f, 60.f), 1.f - s, 1.f);
    }
    return 1.f;
}

// The same two at a time for results of 16 bits, by packed operations and with fewer of the special-function unit's, 16 a clock and SM, which bound
// the pair above.  With a = |z| and e = exp(-z^2 / 2):  gelu(z) = max(z, 0) - a e R(a),  gelu'(z) = w + 1 for z > 0, else -w, with w = e (a / sqrt(2 pi) - R(a)),
// where R(a) = Phi(-a) / e is a polynomial, fitted on [0, 5.6] for the least largest max(1, a) |e R - Phi(-a)|: 1.8e-6, a 250th of half a step of fp16.
// Beyond 16 the polynomial is held and e is zero.  SiLU takes one reciprocal for a pair: 1 / u = v / (u v).
// 2,449,029 x 256 -> 256 bf16, forward alone (scalar -> pairs, and 8 -> 16 epilogue warps): GELU 741 us -> 595, SiLU 555 -> 478.
// -e R(a), or with SLOPE  e (a / sqrt(2 pi) - R(a))
template <bool SLOPE> __device__ __forceinline__ float_pair normal_tail(float_pair z, float_pair a)
{
    const float2 s = halves(mul2(mul2(z, both(-0.72134752f)), z));
    const float_pair e = pair_of(exp2_approx(s.x), exp2_approx(s.y));
    float_pair p = fma2(a, both(-3.0133221e-05f), both(0.000520282793f));
    p = fma2(a, p, both(-0.00394014047f));
    p = fma2(a, p, both(0.0177029971f));
    p = fma2(a, p, both(-0.0546821583f));
    p = fma2(a, p, both(0.128968935f));
    p = fma2(a, p, both(-0.248956095f));
    p = fma2(a, p, both(SLOPE ? 0.398837851f + 0.39894228f : 0.398837851f));
    p = fma2(a, p, both(-0.49999825f));
    return mul2(p, e);
}
// SiLU's sigmoid stands at 2^-60 below z = -41.6 and z at -60, which leaves 6e-17 of the true value.
__device__ __forceinline__ float_pair sigmoid2(float_pair z)
{
    const float2 s = halves(mul2(z, both(-1.44269504f)));
    const float_pair u = add2(pair_of(exp2_approx(fminf(s.x, 60.f)), exp2_approx(fminf(s.y, 60.f))), both(1.f));      // the product stays finite
    const float2 d = halves(u);
    return mul2(pair_of(d.y, d.x), both(reciprocal(d.x * d.y)));
}
template <int ACT> __device__ __forceinline__ float_pair act_value2(float_pair z)
{
    const float2 f = halves(z);
    if (ACT == DG_ACT_RELU) return pair_of(act_value<ACT>(f.x), act_value<ACT>(f.y));
    if (ACT == DG_ACT_GELU) {
        const float_pair a = pair_of(fminf(fabsf(f.x), 16.f), fminf(fabsf(f.y), 16.f));
        return fma2(a, normal_tail<false>(z, a), pair_of(fmaxf(f.x, 0.f), fmaxf(f.y, 0.f)));
    }
    if (ACT == DG_ACT_SILU) return mul2(pair_of(at_least(f.x, -60.f), at_least(f.y, -60.f)), sigmoid2(z));
    return z;
}
template <int ACT> __device__ __forceinline__ float_pair act_slope2(float_pair z)
{
    if (ACT == DG_ACT_GELU) {
        const float2 f = halves(z);
        const float_pair a = pair_of(fminf(fabsf(f.x), 16.f), fminf(fabsf(f.y), 16.f));
        const float2 w = halves(normal_tail<true>(z, a));
        return pair_of(f.x > 0.f ? w.x + 1.f : -w.x, f.y > 0.f ? w.y + 1.f : -w.y);
    }
    if (ACT == DG_ACT_SILU) {
        const float2 f = halves(z);
        const float_pair s = sigmoid2(z), rest = fma2(s, both(-1.f), both(1.f)), near = pair_of(bounded(f.x, -60.f, 60.f), bounded(f.y, -60.f, 60.f));
        return mul2(s, fma2(near, rest, both(1.f)));
    }
    return both(1.f);
}

}  // namespace dg
