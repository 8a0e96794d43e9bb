// One AdamW step over all tensors of a model, states in 32 bits or in 8, and the norm of all gradients that clips them.
//
//   g' = g min(1, max_norm / (|g| + 1e-6)),  m = b1 m + (1 - b1) g',  v = b2 v + (1 - b2) g'^2,  r = sqrt(v)
//   p  = p (1 - lr wd) - lr / (1 - b1^t)  m / (r / sqrt(1 - b2^t) + eps)
//
// All of it in fp32, whatever the type of p and g, each operation rounded by itself, p rounded once to its type.  In 8 bits m and r are kept (r, not
// v: its range is half as many octaves) as e4m3 numbers times a scale for every 256 elements, the block's largest magnitude / 448.  Rounding to
// nearest would freeze such an average, which moves by 0.05 % of itself a step on a grid of 6 to 12 %; so the rounding is random, up with the probability
// of the distance to the neighbour below, with numbers that are a function of (seed, step, place): a step can be repeated bit for bit.  An r above zero is
// never rounded to zero, or the next step would divide an m that is not by eps.  A block that holds an infinity or a NaN is non-finite from then on.
//
// What bounds it: HBM for tables with 32-bit states (28 bytes an element; 157 M fp32 702 us, 6.3 TB/s, and their norm 110 us, 5.7 TB/s; bf16 22 bytes, 578 us,
// 6.0 TB/s), with bf16 and 8 bits (10 bytes and 55 instructions an element; 627 M 1,323 us, 4.8 TB/s) neither HBM nor the issue slots, 70 % busy: the latency that 24 warps
// an SM leave uncovered; the launch for small models (8.9 k elements 4.8 us).
#include <algorithm>
#include <cmath>
#include <type_traits>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include "dg_internal.h"
#include "dg_pair.h"

namespace {

using namespace dg;

// A lane takes 8 neighbouring elements, a warp one block of 256; a thread works on two such pieces of a chunk at once.
constexpr int kThreads = 256, kEach = 8, kHalf = kThreads * kEach, kChunk = 2 * kHalf;
constexpr int kBlock = 256;
constexpr int kNormCtas = 148 * 8;
template <bool SMALL> constexpr int kStepCtas = SMALL ? 3 : 2;      // of a step, that an SM holds
constexpr float kLargest = 448.f;

// Tensors of one launch.  Their table travels with the launch, so that a captured graph holds it and nothing has to be copied ahead; a launch takes 32 KB of
// arguments at most, and the more of them the longer: three sizes.
struct Gradient {
    const void* g;
    int64_t n;
};
template <class Entry, int CAP> struct Table {
    Entry t[CAP];
    int32_t first[CAP + 1];               // running count of chunks
    int32_t count;
    uint32_t wide[(CAP + 31) / 32];       // bit: every address on the boundary that whole loads want
};
constexpr int kFew = 40, kSome = 136, kMany = 376;

struct Factors {
    double log_beta1, log_beta2;
    float lr, b1, a1, b2, a2, eps, keep;  // a = 1 - b; keep = 1 - lr wd
    float one;
    uint32_t seed;
};

template <class T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }

// Eight neighbouring elements, as whole 16-byte pieces (8 bytes for codes) or one by one; elements from n on are zero and not stored.
template <class T> struct Eight {
    uint4 raw[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T* p)
    {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) raw[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
    }
    __device__ __forceinline__ void load(const T* p, int n, bool wide)
    {
        if (wide && n >= 8) {
            load(p);
        } else {
            T* e = reinterpret_cast<T*>(raw);
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = i < n ? p[i] : from_float<T>(0.f);
        }
    }
    __device__ __forceinline__ float_pair pair(int i) const
    {
        const uint32_t w[4] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w};
        if constexpr (sizeof(T) == 4) {
            const float* f = reinterpret_cast<const float*>(raw);
            return pair_of(f[2 * i], f[2 * i + 1]);
        } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
            return pair_of(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
        } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            return pair_of(f.x, f.y);
        }
    }
};
template <class T> __device__ __forceinline__ void store8(T* p, int n, bool wide, const float_pair* pairs)
{
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = halves(pairs[i]);
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
    }
    if (wide && n >= 8) {
        if constexpr (sizeof(T) == 4) {
            __stcs(reinterpret_cast<float4*>(p), make_float4(v[0], v[1], v[2], v[3]));
            __stcs(reinterpret_cast<float4*>(p) + 1, make_float4(v[4], v[5], v[6], v[7]));
        } else {
            uint4 a;
            T* e = reinterpret_cast<T*>(&a);
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = from_float<T>(v[i]);
            __stcs(reinterpret_cast<uint4*>(p), a);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = from_float<T>(v[i]);
    }
}
__device__ __forceinline__ uint2 load_codes(const uint8_t* p, int n, bool wide)
{
    if (wide && n >= 8) return __ldcs(reinterpret_cast<const uint2*>(p));
    uint2 c = make_uint2(0u, 0u);
    for (int i = 0; i < 8 && i < n; ++i) (i < 4 ? c.x : c.y) |= (uint32_t)p[i] << (i % 4 * 8);
    return c;
}
__device__ __forceinline__ void store_codes(uint8_t* p, int n, bool wide, uint2 c)
{
    if (wide && n >= 8) {
        __stcs(reinterpret_cast<uint2*>(p), c);
        return;
    }
    for (int i = 0; i < 8 && i < n; ++i) p[i] = (uint8_t)((i < 4 ? c.x : c.y) >> (i % 4 * 8));
}
__device__ __forceinline__ void decode(uint2 c, float scale, float_pair* v)
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t w = i < 2 ? c.x : c.y;
        const float2 f = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> (i % 2 * 16)), __NV_E4M3)));
        v[i] = mul2(pair_of(f.x, f.y), both(scale));
    }
}

// The square root, by Newton's step with the remainder from a fused product (Markstein, IBM Journal of Research and Development, 1990): the correctly
// rounded one but for a few arguments in a million, where it is the neighbour, and below fp32's smallest normal number that of the approximation, within 2^-22.
// Zero is taken for the smallest number above it, whose reciprocal root is finite.
__device__ __forceinline__ float_pair square_root(float_pair v)
{
    const float2 f = halves(v);
    float a, b;
    asm("rsqrt.approx.f32 %0, %1;" : "=f"(a) : "f"(fmaxf(f.x, 0x1p-149f)));
    asm("rsqrt.approx.f32 %0, %1;" : "=f"(b) : "f"(fmaxf(f.y, 0x1p-149f)));
    const float_pair y = pair_of(a, b), s = mul2(v, y);
    return fma2(fma2(mul2(s, both(-1.f)), s, v), mul2(y, both(0.5f)), s);
}

// Random numbers: xor-shift and product, twice, for a pair of neighbours, 16 bits for each.  The odd factors are the leading bits of the golden
// ratio's and of square roots' fractions.
__device__ __forceinline__ uint32_t mix(uint32_t h)
{
    h = (h ^ h >> 16) * 0x6A09E667u;
    h = (h ^ h >> 15) * 0xBB67AE85u;
    return h ^ h >> 16;
}
__device__ __forceinline__ uint32_t key_of(uint32_t seed, int64_t step) { return mix(seed + (uint32_t)step * 0x3C6EF373u); }

// A block's values, eight a lane, as codes and a scale.  q = |x| 448 / largest; times 2^-120 the smallest normal number of e4m3 is the smallest one of fp32, so
// that an fp32 number's leading bits are the code, below 2^-6 too where both step evenly.  The noise is added below the code's last bit.
// (q times 2^-120 in one factor would leave fp32's range where the block's largest is beyond 28,672.)
__device__ __forceinline__ float largest(const float_pair* x)
{
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = halves(x[i]);
        asm("max.NaN.f32 %0, %0, %1;" : "+f"(most) : "f"(fabsf(f.x)));
        asm("max.NaN.f32 %0, %0, %1;" : "+f"(most) : "f"(fabsf(f.y)));
    }
    return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most) & 0x7FFFFFFFu));      // magnitudes are ordered as their bits, NaN above all
}
template <bool ROOT> __device__ __forceinline__ uint2 codes(const float_pair* x, const uint32_t* noise, float factor)
{
    uint32_t c[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        uint32_t t[4];                                            // the code in the leading byte; the sign is shifted out
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float2 f = halves(x[2 * i + j]), l = halves(mul2(mul2(x[2 * i + j], both(factor)), both(0x1p-120f)));
            const uint32_t n = noise[2 * i + j];
            t[2 * j] = (__float_as_uint(l.x) << 4) + __byte_perm(n, 0, 0x4104);
            t[2 * j + 1] = (__float_as_uint(l.y) << 4) + __byte_perm(n, 0, 0x4324);
            if (ROOT) {                                           // code 1 for what is above zero: the bits of 2^-125 and more reach that far
                t[2 * j] = max(t[2 * j], min(__float_as_uint(f.x), 0x01000000u));
                t[2 * j + 1] = max(t[2 * j + 1], min(__float_as_uint(f.y), 0x01000000u));
            } else {
                t[2 * j] |= __float_as_uint(f.x) & 0x80000000u;
                t[2 * j + 1] |= __float_as_uint(f.y) & 0x80000000u;
            }
        }
        c[i] = __byte_perm(__byte_perm(t[0], t[1], 0x0073), __byte_perm(t[2], t[3], 0x0073), 0x5410);
    }
    return make_uint2(c[0], c[1]);
}
// 448 / largest as the product of 448 and the reciprocal, which Newton's step with fused products rounds correctly (Markstein, as above).  Blocks whose largest
// is beyond 2^125, where the reciprocal leaves fp32's normal range, or below 1e-30, are zero.
__device__ __forceinline__ void encode(const float_pair* m, const float_pair* r, const uint32_t* noise, uint2* to_m, uint2* to_r, float* scale_m, float* scale_r)
{
    const float top_m = largest(m), top_r = largest(r);
    const float_pair top = pair_of(top_m, top_r), y = pair_of(reciprocal(top_m), reciprocal(top_r));
    const float2 f = halves(mul2(fma2(fma2(mul2(top, both(-1.f)), y, both(1.f)), y, y), both(kLargest))), s = halves(mul2(top, both(1.f / kLargest)));
    const bool none_m = top_m < 1e-30f, none_r = top_r < 1e-30f;
    *scale_m = none_m ? 0.f : s.x, *scale_r = none_r ? 0.f : s.y;
    *to_m = codes<false>(m, noise, none_m ? 0.f : f.x);
    *to_r = codes<true>(r, noise, none_r ? 0.f : f.y);
}

// The tensor that a chunk belongs to, by all threads of the CTA.
template <class Tab> __device__ __forceinline__ int find(const Tab& tab, int chunk)
{
    int before = 0;
    for (int k = 0; k < tab.count; k += kThreads) before += __syncthreads_count(k + (int)threadIdx.x < tab.count && tab.first[k + threadIdx.x] <= chunk);
    return before - 1;
}

template <class T, bool SMALL, int CAP>
__global__ void __launch_bounds__(kThreads, kStepCtas<SMALL>) k_adamw(const __grid_constant__ Table<dg_adamw_tensor, CAP> tab, const Factors f, const float* __restrict__ clip,
                                                                  int* __restrict__ arrived)
{
    __shared__ int warps_done;
    if (threadIdx.x == 0) warps_done = 0;                         // find() below is a barrier
    const int chunks = tab.first[tab.count];
    int at = -1;
    float rate = 0.f, correction = 0.f;
    uint32_t key = 0;
    const float coef = clip ? __ldg(clip) : 1.f;
    int before = -1;
    int64_t step = 0;
    for (int chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
        int i = at;
        if (at < 0) i = find(tab, chunk);
        else
            while (tab.first[i + 1] <= chunk) ++i;
        const dg_adamw_tensor& t = tab.t[i];
        const bool wide = tab.wide[i / 32] >> (i % 32) & 1;
        const int64_t e0 = (int64_t)(chunk - tab.first[i]) * kChunk + threadIdx.x * kEach, left = t.n - e0;
        using State = std::conditional_t<SMALL, uint8_t, float>;
        T* const p_at = reinterpret_cast<T*>(t.p) + e0;
        const T* const g_at = reinterpret_cast<const T*>(t.g) + e0;
        State *const m_at = reinterpret_cast<State*>(t.m) + e0, *const v_at = reinterpret_cast<State*>(t.v) + e0;
        float *const sm_at = SMALL ? t.m_scale + e0 / kBlock : nullptr, *const sv_at = SMALL ? t.v_scale + e0 / kBlock : nullptr;
        const bool full = wide && left >= kHalf + kEach;          // nothing of this thread's lies beyond the tensor
        Eight<T> p_in[2], g_in[2];
        [[maybe_unused]] Eight<float> m_in[2], v_in[2];
        [[maybe_unused]] uint2 cm[2], cv[2];
        float sm[2] = {0.f, 0.f}, sv[2] = {0.f, 0.f};
        auto count = [&](int u) { return (int)max((int64_t)0, min((int64_t)kEach, left - u * kHalf)); };
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            if (full) {
                g_in[u].load(g_at + u * kHalf);
                if constexpr (SMALL) {
                    cm[u] = __ldcs(reinterpret_cast<const uint2*>(m_at + u * kHalf));
                    cv[u] = __ldcs(reinterpret_cast<const uint2*>(v_at + u * kHalf));
                    sm[u] = sm_at[u * (kHalf / kBlock)], sv[u] = sv_at[u * (kHalf / kBlock)];
                } else {
                    m_in[u].load(m_at + u * kHalf);
                    v_in[u].load(v_at + u * kHalf);
                }
                p_in[u].load(p_at + u * kHalf);
            } else {
                const int n = count(u);
                g_in[u].load(g_at + u * kHalf, n, wide);
                if constexpr (SMALL) {
                    cm[u] = load_codes(m_at + u * kHalf, n, wide);
                    cv[u] = load_codes(v_at + u * kHalf, n, wide);
                    if (n > 0) sm[u] = sm_at[u * (kHalf / kBlock)], sv[u] = sv_at[u * (kHalf / kBlock)];
                } else {
                    m_in[u].load(m_at + u * kHalf, n, wide);
                    v_in[u].load(v_at + u * kHalf, n, wide);
                }
                p_in[u].load(p_at + u * kHalf, n, wide);
            }
        }
        if (i != at) {                                            // 1 - b^t = -expm1(t log b)
            step = *t.step + 1;
            rate = __fdividef(f.lr, -expm1f((float)((double)step * f.log_beta1)));
            correction = rsqrtf(-expm1f((float)((double)step * f.log_beta2)));
            key = key_of(f.seed, step);
            at = i;
        }
        if (chunk + (int)gridDim.x >= chunks) {                   // no more steps to read here: the warp that is last to say so here says it for the CTA
            if (threadIdx.x % 32 == 0 && atomicAdd(&warps_done, step < 0 ? 0 : 1) == kThreads / 32 - 1) {      // (its step has arrived)
                __threadfence();
                before = atomicAdd(arrived, 1);
            }
        }
        const uint32_t place = (uint32_t)((t.place + e0) >> 1);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            float_pair p[4], m[4], v[4], r[4];
            if constexpr (SMALL) {
                decode(cm[u], sm[u], m);
                decode(cv[u], sv[u], r);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = mul2(r[j], r[j]);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) m[j] = m_in[u].pair(j), v[j] = v_in[u].pair(j);
            }
            // What the means are made of is rounded operation by operation, so that the codes are those of the definition (the assembler would join a
            // packed product and sum, but not a product by a number that it does not know to be one); the update takes what is fastest.
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float_pair h = g_in[u].pair(j);
                if (clip) h = mul2(h, both(coef));
                m[j] = fma2(mul2(m[j], both(f.b1)), both(f.one), mul2(h, both(f.a1)));
                v[j] = fma2(mul2(v[j], both(f.b2)), both(f.one), mul2(mul2(h, h), both(f.a2)));
                r[j] = square_root(v[j]);
                const float2 d = halves(fma2(r[j], both(correction), both(f.eps)));
                const float_pair x = mul2(m[j], pair_of(reciprocal(d.x), reciprocal(d.y)));
                p[j] = fma2(x, both(-rate), mul2(p_in[u].pair(j), both(f.keep)));
            }
            const int n = full ? kEach : count(u);
            store8(p_at + u * kHalf, n, wide, p);
            if constexpr (SMALL) {
                uint32_t noise[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) noise[j] = mix((place + u * (kHalf / 2) + j) * 0x9E3779B1u + key);
                if (n < kEach)                                    // what lies beyond the tensor is no part of its block
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float2 a = halves(m[j]), b = halves(r[j]);
                        m[j] = pair_of(2 * j < n ? a.x : 0.f, 2 * j + 1 < n ? a.y : 0.f);
                        r[j] = pair_of(2 * j < n ? b.x : 0.f, 2 * j + 1 < n ? b.y : 0.f);
                    }
                float scale_m, scale_v;
                uint2 to_m, to_v;
                encode(m, r, noise, &to_m, &to_v, &scale_m, &scale_v);
                store_codes(m_at + u * kHalf, n, wide, to_m);
                store_codes(v_at + u * kHalf, n, wide, to_v);
                if (threadIdx.x % 32 == 0 && n > 0) sm_at[u * (kHalf / kBlock)] = scale_m, sv_at[u * (kHalf / kBlock)] = scale_v;
            } else {
                store8(m_at + u * kHalf, n, wide, m);
                store8(v_at + u * kHalf, n, wide, v);
            }
        }
    }
    // The warp that was last of all to have read its steps counts them all up.
    if (__shfl_sync(0xffffffffu, before, 0) != (int)gridDim.x - 1) return;
    for (int k = threadIdx.x % 32; k < tab.count; k += 32) ++*tab.t[k].step;
    if (threadIdx.x % 32 == 0) *arrived = 0;
}

// Sum of squares in 64 bits, every CTA's in its own place; the CTA that comes last of the last launch adds them in order.
template <class T, int CAP>
__global__ void __launch_bounds__(kThreads) k_grad_norm(const __grid_constant__ Table<Gradient, CAP> tab, double* __restrict__ partial, int total, double max_norm,
                                                        float* __restrict__ result, int* __restrict__ arrived)
{
    __shared__ double warp_sum[kThreads / 32];
    __shared__ int last;
    auto sum_of_cta = [&](double s) {
        for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
        __syncthreads();
        if (threadIdx.x % 32 == 0) warp_sum[threadIdx.x / 32] = s;
        __syncthreads();
        s = 0.0;
        for (int w = 0; w < kThreads / 32; ++w) s += warp_sum[w];
        return s;
    };
    const int chunks = tab.first[tab.count];
    double sum = 0.0;
    int i = -1;
    for (int chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
        if (i < 0) i = find(tab, chunk);
        else
            while (tab.first[i + 1] <= chunk) ++i;
        const Gradient& t = tab.t[i];
        const int64_t e0 = (int64_t)(chunk - tab.first[i]) * kChunk + threadIdx.x * kEach;
        const bool wide = tab.wide[i / 32] >> (i % 32) & 1;
        Eight<T> g[2];
#pragma unroll
        for (int u = 0; u < 2; ++u)
            g[u].load(reinterpret_cast<const T*>(t.g) + e0 + u * kHalf, (int)max((int64_t)0, min((int64_t)kEach, t.n - e0 - u * kHalf)), wide);
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 f = halves(g[u].pair(j));
                sum += (double)f.x * (double)f.x;
                sum += (double)f.y * (double)f.y;
            }
    }
    sum = sum_of_cta(sum);
    if (threadIdx.x == 0) partial[blockIdx.x] = sum;
    if (!result) return;
    if (threadIdx.x == 0) {
        __threadfence();
        last = atomicAdd(arrived, 1) == (int)gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    const double* all = partial + gridDim.x - total;              // this launch's places are the last ones
    double s = 0.0;
    for (int j = threadIdx.x; j < total; j += kThreads) s += __ldcg(all + j);
    s = sum_of_cta(s);
    if (threadIdx.x == 0) {
        const double norm = sqrt(s), coef = max_norm / (norm + 1e-6);
        result[0] = (float)norm;
        result[1] = (float)(coef > 1.0 ? 1.0 : coef);             // a NaN stays
        *arrived = 0;
    }
}

bool aligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }
int64_t chunks_of(int64_t n) { return (n + kChunk - 1) / kChunk; }

// Fills a table with as many of the tensors [at, count) of `type` as it holds; returns where the next one starts.
void entry(dg_adamw_tensor* to, const dg_adamw_tensor& t) { *to = t; }
void entry(Gradient* to, const dg_adamw_tensor& t) { *to = {t.g, t.n}; }
bool whole(const dg_adamw_tensor*, const dg_adamw_tensor& t, int32_t bits)
{
    return aligned(t.g, 16) && aligned(t.p, 16) && aligned(t.m, bits == 8 ? 8 : 16) && aligned(t.v, bits == 8 ? 8 : 16);
}
bool whole(const Gradient*, const dg_adamw_tensor& t, int32_t) { return aligned(t.g, 16); }
template <class Entry, int CAP> int fill(Table<Entry, CAP>* tab, const dg_adamw_tensor* t, int at, int count, int32_t type, int32_t bits)
{
    int64_t chunks = 0;
    tab->count = 0;
    for (uint32_t& w : tab->wide) w = 0;
    for (; at < count && tab->count < CAP; ++at) {
        if (t[at].type != type || t[at].n == 0) continue;
        const int64_t more = chunks_of(t[at].n);
        if (chunks + more >= (int64_t)1 << 30) break;             // chunk numbers, with a stride added, stay within 31 bits
        const int k = tab->count++;
        entry(&tab->t[k], t[at]);
        tab->first[k] = (int32_t)chunks;
        chunks += more;
        if (whole(tab->t, t[at], bits)) tab->wide[k / 32] |= 1u << (k % 32);
    }
    tab->first[tab->count] = (int32_t)chunks;
    return at;
}

int check(const dg_adamw_tensor* t, int32_t count, int32_t bits, bool norm)
{
    if (count < 0 || (bits != 8 && bits != 32)) return DG_ERR_DIMS;
    if (count > 0 && !t) return DG_ERR_NULL;
    for (int32_t i = 0; i < count; ++i) {
        if (t[i].n < 0 || t[i].n >= (int64_t)1 << 40 || t[i].type < 0 || t[i].type > 2) return DG_ERR_DIMS;
        if (t[i].n == 0) continue;
        const size_t item = t[i].type == DG_FLOAT32 ? 4 : 2, state = bits == 8 ? 1 : 4;
        if (!t[i].g) return DG_ERR_NULL;
        if (!aligned(t[i].g, item)) return DG_ERR_DIMS;
        if (norm) continue;
        if (!t[i].p || !t[i].m || !t[i].v || !t[i].step || (bits == 8 && (!t[i].m_scale || !t[i].v_scale))) return DG_ERR_NULL;
        if (!aligned(t[i].p, item) || !aligned(t[i].m, state) || !aligned(t[i].v, state) || !aligned(t[i].step, 8) || !aligned(t[i].m_scale, 4) ||
            !aligned(t[i].v_scale, 4))
            return DG_ERR_DIMS;
    }
    return DG_OK;
}

// `use(table, type constant, last)` for as many tables as the tensors need, in the smallest size that holds them, or the largest.
template <class Entry, class Use> int each_table(const dg_adamw_tensor* t, int32_t count, int32_t bits, Use use)
{
    int have[3] = {0, 0, 0};
    for (int32_t i = 0; i < count; ++i) have[t[i].type] += t[i].n > 0;
    for (int32_t type = 0; type < 3; ++type) {
        if (have[type] == 0) continue;
        const bool more_types = (type < 1 && have[1]) || (type < 2 && have[2]);
        auto with = [&](auto cap, auto value) {
            Table<Entry, decltype(cap)::value> tab;
            int left = have[type];
            for (int at = 0; left > 0;) {
                at = fill(&tab, t, at, count, type, bits);
                left -= tab.count;
                const int rc = use(tab, value, left == 0 && !more_types);
                if (rc) return rc;
            }
            return (int)DG_OK;
        };
        auto sized = [&](auto value) {
            if (have[type] <= kFew) return with(std::integral_constant<int, kFew>{}, value);
            if (have[type] <= kSome) return with(std::integral_constant<int, kSome>{}, value);
            return with(std::integral_constant<int, kMany>{}, value);
        };
        const int rc = type == DG_FLOAT32 ? sized(float{}) : type == DG_BFLOAT16 ? sized(__nv_bfloat16{}) : sized(__half{});
        if (rc) return rc;
    }
    return DG_OK;
}

}  // namespace

extern "C" int64_t dg_adamw_workspace(const dg_adamw_tensor* host_tensors, int32_t count)
{
    int64_t tables = 0;
    if (count < 0 || (count > 0 && !host_tensors)) return DG_ERR_NULL;
    for (int32_t type = 0; type < 3; ++type) {
        int64_t have = 0, chunks = 0;
        for (int32_t i = 0; i < count; ++i)
            if (host_tensors[i].type == type) ++have, chunks += chunks_of(std::max<int64_t>(host_tensors[i].n, 0));
        tables += have / kFew + 1 + chunks / ((int64_t)1 << 29);
    }
    return 16 + 8 * tables * kNormCtas;
}

extern "C" int dg_grad_norm(const dg_adamw_tensor* host_tensors, int32_t count, double max_norm, float* result, void* workspace, int64_t workspace_bytes,
                            void* stream)
{
    int rc = check(host_tensors, count, 32, true);
    if (rc) return rc;
    if (!result || !workspace) return DG_ERR_NULL;
    if (!(max_norm > 0.0) || !aligned(workspace, 16)) return DG_ERR_DIMS;
    if (workspace_bytes < dg_adamw_workspace(host_tensors, count)) return DG_ERR_SCRATCH;
    int* arrived = reinterpret_cast<int*>(workspace);
    double* partial = reinterpret_cast<double*>(reinterpret_cast<char*>(workspace) + 16);
    int total = 0;
    rc = each_table<Gradient>(host_tensors, count, 32, [&](auto& tab, auto value, bool last) {
        const int grid = std::min(kNormCtas, (int)tab.first[tab.count]);
        total += grid;
        k_grad_norm<decltype(value)><<<grid, kThreads, 0, (cudaStream_t)stream>>>(tab, partial + total - grid, total, max_norm, last ? result : nullptr, arrived);
        return (int)cudaGetLastError();
    });
    if (rc || total > 0) return rc;
    Table<Gradient, kFew> none{};                                 // no gradients: a sum of nothing
    k_grad_norm<float><<<1, kThreads, 0, (cudaStream_t)stream>>>(none, partial, 1, max_norm, result, arrived);
    return (int)cudaGetLastError();
}

extern "C" int dg_adamw_step(const dg_adamw_tensor* host_tensors, int32_t count, const dg_adamw_options* options, const float* clip, void* workspace,
                             int64_t workspace_bytes, void* stream)
{
    if (!options || !workspace) return DG_ERR_NULL;
    const int rc = check(host_tensors, count, options->bits, false);
    if (rc) return rc;
    if (!(options->beta1 >= 0.0 && options->beta1 < 1.0 && options->beta2 >= 0.0 && options->beta2 < 1.0 && options->eps >= 0.0 && options->lr >= 0.0 &&
          options->weight_decay >= 0.0) || !aligned(workspace, 16))
        return DG_ERR_DIMS;
    if (workspace_bytes < 16) return DG_ERR_SCRATCH;
    Factors f{};
    f.lr = (float)options->lr, f.log_beta1 = log(options->beta1), f.log_beta2 = log(options->beta2);
    f.b1 = (float)options->beta1, f.a1 = (float)(1.0 - options->beta1), f.b2 = (float)options->beta2, f.a2 = (float)(1.0 - options->beta2);
    f.one = 1.f, f.eps = (float)options->eps, f.keep = (float)(1.0 - options->lr * options->weight_decay), f.seed = options->seed;
    int* arrived = reinterpret_cast<int*>(workspace) + 1;
    const bool small = options->bits == 8;
    return each_table<dg_adamw_tensor>(host_tensors, count, options->bits, [&](auto& tab, auto value, bool) {
        using T = decltype(value);
        // Whole waves, each CTA with as many chunks: with 3 CTAs an SM 8 of them an SM leave a third of the last wave idle.
        const int grid = std::min(148 * (small ? 3 * kStepCtas<true> : 4 * kStepCtas<false>), (int)tab.first[tab.count]);
        if (small) k_adamw<T, true><<<grid, kThreads, 0, (cudaStream_t)stream>>>(tab, f, clip, arrived);
        else k_adamw<T, false><<<grid, kThreads, 0, (cudaStream_t)stream>>>(tab, f, clip, arrived);
        return (int)cudaGetLastError();
    });
}
