// Activations of the linear layer and their derivatives, in fp32.
#pragma once
#include "dist_gnn_b200.h"
#include "dg_pair.h"

namespace dg {

// A NaN stays one in both.
__device__ __forceinline__ float at_least(float z, float low)
{
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(z) : "f"(low));
    return z;
}
__device__ __forceinline__ float at_most(float z, float high)
{
    asm("min.NaN.f32 %0, %0, %1;" : "+f"(z) : "f"(high));
    return z;
}
// SiLU multiplies its sigmoid by a z within bounds: beyond them a sigmoid that is a rounding away from 0 or 1 would count |z| times.
__device__ __forceinline__ float bounded(float z, float low, float high) { return at_most(at_least(z, low), high); }

// Phi(-a) = e R(a) with e = exp(-a^2 / 2) and R(a) = t P(t), t = 1 / (1 + 0.23 a): the form of Hastings (Approximations for Digital Computers, 1955), with a
// polynomial of degree 7 fitted for the least largest error over [0, 14], relative to R and to 4e-8 of the value at once: within 5e-7 of R everywhere, so that the small values of
// GELU's tail are as exact as the large ones, and 1.3e-7 / 4e-8 of Phi / z Phi.  No branches, and the density that the derivative needs comes with it: against erff, whose two
// branches diverge, the forward pass of 2,449,029 x 256 -> 256 bf16 went from 1,329 us to 975 and the gradient's pass from 1,101 to 874.
// a is held at 16, where e is zero.
__device__ __forceinline__ float normal_tail(float a, float* e)
{
    const float t = reciprocal(fmaf(a, 0.23f, 1.f));
    float p = fmaf(t, -0.07433278f, 0.27045143f);
    p = fmaf(t, p, -0.23720871f);
    p = fmaf(t, p, 0.255083f);
    p = fmaf(t, p, -0.0011804379f);
    p = fmaf(t, p, 0.10612199f);
    p = fmaf(t, p, 0.08916063f);
    p = fmaf(t, p, 0.0919049f);
    *e = exp2_approx(a * a * -0.72134752f);
    return p * t * *e;
}
__device__ __forceinline__ float sigmoid(float z)
{
    return reciprocal(1.f + exp2_approx(z * -1.44269504f));
}
// gelu(z) = z Phi(z) with the distribution function of the normal distribution, silu(z) = z / (1 + exp(-z)).
template <int ACT> __device__ __forceinline__ float act_value(float z)
{
    if (ACT == DG_ACT_RELU) return z > 0.f || z != z ? z : 0.f;       // a NaN stays
    if (ACT == DG_ACT_GELU) {
        float e;
        const float a = at_most(fabsf(z), 16.f), tail = normal_tail(a, &e);
        return fmaf(-a, tail, fmaxf(z, 0.f));                         // -infinity gives zero
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
        const float a = at_most(fabsf(z), 16.f), w = normal_tail(a, &e) - a * 0.39894228f * e;
        return z > 0.f ? 1.f - w : w;
    }
    if (ACT == DG_ACT_SILU) {
        const float s = sigmoid(z);
        return s * fmaf(bounded(z, -104.f, 60.f), 1.f - s, 1.f);
    }
    return 1.f;
}

// The same two at a time for results of 16 bits, by packed operations and with fewer of the special-function unit's, 16 a clock and SM, which bound
// the pair above.  With a = |z| and e = exp(-z^2 / 2):  gelu(z) = max(z, 0) - a e R(a),  gelu'(z) = w + 1 for z > 0, else -w, with w = e (a / sqrt(2 pi) - R(a)).
// R(a) = t P(t) as above, t = 1 / (1 + 0.3 a) and P of degree 5: within 1.8e-5 of R everywhere on [0, 14], a 27th of half a step of fp16, and 3e-7 of the value.  (A polynomial in
// a, fitted for the value alone, was 11 % off at gelu(-4.5) and several times the value below -5.)  SiLU and GELU take one reciprocal for a pair: 1 / u = v / (u v).
// 2,449,029 x 256 -> 256 bf16, forward alone (scalar -> pairs, and 8 -> 16 epilogue warps): GELU 741 us -> 584, SiLU 555 -> 507.
__device__ __forceinline__ float_pair reciprocals(float_pair u)      // of numbers whose product is within fp32's range
{
    const float2 d = halves(u);
    return mul2(pair_of(d.y, d.x), both(reciprocal(d.x * d.y)));
}
// -e R(a), or with SLOPE  e (a / sqrt(2 pi) - R(a))
template <bool SLOPE> __device__ __forceinline__ float_pair normal_tail(float_pair z, float_pair a)
{
    const float2 s = halves(mul2(mul2(z, both(-0.72134752f)), z));
    const float_pair e = pair_of(exp2_approx(s.x), exp2_approx(s.y)), t = reciprocals(fma2(a, both(0.3f), both(1.f)));
    float_pair p = fma2(t, both(0.07944028f), both(-0.22236827f));
    p = fma2(t, p, both(0.023232138f));
    p = fma2(t, p, both(-0.14699727f));
    p = fma2(t, p, both(-0.11319609f));
    p = fma2(t, p, both(-0.12011052f));
    p = SLOPE ? fma2(t, p, mul2(a, both(0.39894228f))) : mul2(t, p);
    return mul2(p, e);
}
// SiLU's sigmoid stands at 2^-60 below z = -41.6 and z at -60, which leaves 6e-17 of the true value.
__device__ __forceinline__ float_pair sigmoid2(float_pair z)
{
    const float2 s = halves(mul2(z, both(-1.44269504f)));
    const float_pair u = add2(pair_of(exp2_approx(fminf(s.x, 60.f)), exp2_approx(fminf(s.y, 60.f))), both(1.f));      // the product stays finite
    return reciprocals(u);
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
