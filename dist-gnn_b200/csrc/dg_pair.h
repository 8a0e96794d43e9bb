// Two fp32 numbers in a register pair: packed operations, each lane rounded by itself, and the special-function unit's approximations.
#pragma once
#include <cstdint>

namespace dg {

using float_pair = unsigned long long;
__device__ __forceinline__ float_pair pair_of(float a, float b)
{
    float_pair r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 halves(float_pair v)
{
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ float_pair fma2(float_pair a, float_pair b, float_pair c)
{
    float_pair r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ float_pair mul2(float_pair a, float_pair b)
{
    float_pair r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float_pair add2(float_pair a, float_pair b)
{
    float_pair r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float_pair both(float v) { return pair_of(v, v); }
__device__ __forceinline__ float reciprocal(float v)      // within a unit in the last place
{
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float exp2_approx(float v)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

}  // namespace dg
