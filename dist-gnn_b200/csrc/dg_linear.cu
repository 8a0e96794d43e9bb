// Linear layer with bias, activation and residual in the product's epilogue, y = act(x w + b) + r, for 16-bit operands, and what its gradients need.
//
// k_linear_pair: x w on the tensor cores (tcgen05 kind::f16, fp32 accumulators in tensor memory) by CTA pairs that walk over tiles of 256 rows x up to 256
// columns.  w is read as it lies: [N x K] rows are K-major operands, [K x N] rows MN-major ones, both in 128B-swizzled boxes.
// k_linear_dw: the weight gradient x^T dz, both operands MN-major, rows cut into ranges whose partial results are added in order.
// k_linear_back: the same with dz = dy act'(z), its column sums and, where asked, dz itself made on the way.
// k_linear_dz: dz and its column sums alone.
// k_few_*: products of few rows, bound by latency.  k_thin, k_thin_grad: narrow layers.
// The fp32 product is dg_dense.cu's.
#include <algorithm>
#include <type_traits>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "dg_act.h"
#include "dg_internal.h"
#include "dg_tma.h"

namespace {

using namespace dg;

template <class T> struct Pair;
template <> struct Pair<__nv_bfloat16> {
    using Two = __nv_bfloat162;
    static __device__ __forceinline__ float2 wide(uint32_t v) { return __bfloat1622float2(*reinterpret_cast<const Two*>(&v)); }
    static __device__ __forceinline__ uint32_t narrow(float a, float b)
    {
        const Two t = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&t);
    }
    static __device__ __forceinline__ float_pair two(uint32_t v) { return pair_of(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u)); }
    static __device__ __forceinline__ uint32_t narrow(float_pair v)
    {
        const float2 f = halves(v);
        return narrow(f.x, f.y);
    }
    static __device__ __forceinline__ float one(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 round(float v) { return __float2bfloat16_rn(v); }
    static constexpr uint32_t kFormat = 1;
};
template <> struct Pair<__half> {
    using Two = __half2;
    static __device__ __forceinline__ float2 wide(uint32_t v) { return __half22float2(*reinterpret_cast<const Two*>(&v)); }
    static __device__ __forceinline__ uint32_t narrow(float a, float b)
    {
        const Two t = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&t);
    }
    static __device__ __forceinline__ float_pair two(uint32_t v)
    {
        const float2 f = wide(v);
        return pair_of(f.x, f.y);
    }
    static __device__ __forceinline__ uint32_t narrow(float_pair v)
    {
        const float2 f = halves(v);
        return narrow(f.x, f.y);
    }
    static __device__ __forceinline__ float one(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half round(float v) { return __float2half_rn(v); }
    static constexpr uint32_t kFormat = 0;
};
template <> struct Pair<float> {
    static __device__ __forceinline__ float one(float v) { return v; }
    static __device__ __forceinline__ float round(float v) { return v; }
};

// The tensor cores truncate when they add into an accumulator: where all terms are of one sign a chain of n accumulations, 16 terms each, is some n 2^-23 too small.  So
// long sums are taken in chains, whose results are added rounded to nearest: fp16, which rounds by 2^-11, after 512 accumulations (6e-5), bf16, by 2^-8, after 2,048.
constexpr int chain_terms(bool bf16) { return bf16 ? 32768 : 8192; }
template <class T> constexpr int kChainTerms = chain_terms(std::is_same<T, __nv_bfloat16>::value);

// ---- the product on the tensor cores ------------------------------------------------------------------------------------
constexpr int BM = 128, BK = 64;                  // rows of a CTA, K-columns of a stage: 128 bytes
constexpr int kEpilogueWarps = 16, kThreadsPair = 32 * (2 + kEpilogueWarps);
constexpr int kMaxStages = 8;
constexpr int kABytes = BM * BK * 2;
constexpr int kPiece = 32, kPieceBytes = 32 * kPiece * 2;      // an epilogue warp's 32 rows x 32 columns
constexpr int kBarBytes = 8 * (2 * kMaxStages + 5 + 2 * kEpilogueWarps) + 8;

struct LinearPairArgs {
    const void* bias;
    uint32_t* bits;
    int64_t ldbits;
    int64_t M;
    int32_t N, K;
    int32_t n_tile, n_panels, tiles;
    int32_t stages;
    int32_t b_boxes;                              // w MN-major: boxes of 64 columns a CTA loads; 0: K-major
    int32_t residual, save_z, whole_bias;
    int* status;
};

__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, int c0, int c1, uint32_t src)
{
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map), "r"(src), "r"(c0), "r"(c1) : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// MN-major 16-bit tile: boxes of 64 columns x `rows` K-rows of 128 bytes, 128B swizzle; 8-row groups are 1024 bytes apart (stride byte offset), boxes
// `box_bytes` (leading byte offset).
__device__ __forceinline__ uint64_t umma_desc_mn16(uint32_t smem_addr, uint32_t box_bytes)
{
    return (uint64_t)((smem_addr & 0x3FFFF) >> 4) | (uint64_t)(box_bytes >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// kind::f16: fp32 accumulator, A and B of `format` (0: fp16, 1: bf16)
__device__ __forceinline__ uint32_t umma_idesc_f16(uint32_t format, int m, int n, bool a_mn, bool b_mn)
{
    return 1u << 4 | format << 7 | format << 10 | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) | (uint32_t)(n >> 3) << 17 | (uint32_t)(m >> 4) << 24;
}
__device__ __forceinline__ void umma_f16_pair(uint32_t tmem_d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void umma_f16(uint32_t tmem_d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}

// Warps: 0 TMA, 1 MMA issue (even CTA) + tensor-memory allocation, 2-17 epilogue (lane quarter w % 4; four warps a quarter take its 32-column pieces
// in turn).  A stage is 64 K-columns of the CTA's 128 rows of x and of its half of the panel's columns of w.  Two accumulators (columns 0 / 256).
// Barriers: full (even CTA, the loads of both), empty and acc_full (both CTAs, by commit), acc_empty (even CTA: the epilogue warps of both), and one an
// epilogue warp and buffer for its residual's pieces.
// What bounds it: HBM up to some 500 columns (400,000 x 256 -> 256 bf16 with GELU, bias, residual and z 143 us, 5.7 TB/s; without them 67 us, 6.1 TB/s), the tensor
// cores beyond (65,536 x 1024 -> 1024 100 us, 1,379 TFLOP/s; with SiLU, residual and z 137).
// DEEP: K beyond a chain; tiles of up to 128 columns, so that a warp has one piece, which it holds in registers while the tile's other chains run.
template <class T, int ACT, bool DEEP>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreadsPair, 1)
k_linear_pair(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmY,
              const __grid_constant__ CUtensorMap tmR, const __grid_constant__ CUtensorMap tmZ, const LinearPairArgs a)
{
    extern __shared__ unsigned char smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    unsigned char* gbase = smem_raw + (base - raw);
    const int half_n = a.n_tile / 2, b_bytes = a.b_boxes ? a.b_boxes * BK * 128 : half_n * 128;
    const int stage_bytes = kABytes + b_bytes;
    const int staging = a.stages * stage_bytes, per_warp = (a.save_z ? 3 : 2) * kPieceBytes;
    const uint32_t bars = base + staging + kEpilogueWarps * per_warp;
    const uint32_t full0 = bars, empty0 = bars + 8 * kMaxStages, acc_full0 = bars + 16 * kMaxStages, acc_empty0 = acc_full0 + 16, done = acc_empty0 + 16;
    const uint32_t res0 = done + 8;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(gbase + staging + kEpilogueWarps * per_warp + 8 * (2 * kMaxStages + 5 + 2 * kEpilogueWarps));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = blockIdx.x & 1, pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const int slabs = (a.K + BK - 1) / BK;
    [[maybe_unused]] const int chains = DEEP ? (a.K + kChainTerms<T> - 1) / kChainTerms<T> : 1, in_chain = DEEP ? (slabs + chains - 1) / chains : slabs;
    constexpr int kTmemCols = 512;

    if (threadIdx.x == 0) {
        for (int s = 0; s < a.stages; ++s) {
            mbar_init(full0 + 8 * s, 1);
            mbar_init(empty0 + 8 * s, 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(acc_full0 + 8 * b, 1);
            mbar_init(acc_empty0 + 8 * b, 2 * kEpilogueWarps);
        }
        mbar_init(done, 1);
        for (int w = 0; w < 2 * kEpilogueWarps; ++w) mbar_init(res0 + 8 * w, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    cluster_sync();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tmem_slot;
    bool ok = true;

    if (warp == 0) {
        if (lane == 0) {                                          // TMA producer: one ring of stages across all tiles
            const uint32_t leader_full0 = in_leader(full0);
            int it = 0, s = 0, phase = 1;
            for (int tile = pair; tile < a.tiles && ok; tile += pairs) {
                const int row0 = (int)((int64_t)(tile / a.n_panels) * (2 * BM) + rank * BM);      // rows beyond the matrix arrive as zeros
                const int n0 = tile % a.n_panels * a.n_tile + rank * half_n;
                for (int i = 0; i < slabs; ++i, ++it) {
                    if (it >= a.stages) ok = mbar_wait(empty0 + 8 * s, phase);
                    if (!ok) break;
                    const uint32_t st = base + s * stage_bytes, bar = leader_full0 + 8 * s;
                    if (rank == 0) mbar_expect_tx(full0 + 8 * s, 2 * stage_bytes);
                    tma_load_2d_pair(st, &tmA, i * BK, row0, bar);
                    if (a.b_boxes)
                        for (int j = 0; j < a.b_boxes; ++j) tma_load_2d_pair(st + kABytes + j * BK * 128, &tmB, n0 + 64 * j, i * BK, bar);
                    else
                        tma_load_2d_pair(st + kABytes, &tmB, i * BK, n0, bar);
                    if (++s == a.stages) s = 0, phase ^= 1;
                }
            }
            if (rank == 0) await_loads(full0, it, a.stages);      // of both CTAs; the odd one leaves after this
        }
    } else if (warp == 1) {
        if (rank == 0) {                                          // MMA issuer: the warp waits and counts together, one lane issues
            const bool issuer = elect_one();
            auto wait = [&](uint32_t bar, int parity) { return __any_sync(0xffffffffu, issuer && mbar_wait(bar, parity)) != 0; };
            const uint32_t idesc = umma_idesc_f16(Pair<T>::kFormat, 2 * BM, a.n_tile, false, a.b_boxes != 0);
            const uint64_t a0 = umma_desc_sw128(base);
            const uint64_t b0 = a.b_boxes ? umma_desc_mn16(base + kABytes, BK * 128) : umma_desc_sw128(base + kABytes);
            const uint32_t next_stage = (uint32_t)stage_bytes >> 4, b_step = a.b_boxes ? 16 * 128 >> 4 : 2;      // 16 K-columns
            int s = 0, phase = 0, lt = 0;
            bool early = false;
            [[maybe_unused]] int chain = 0;
            for (int tile = pair; tile < a.tiles && ok; ++lt) {
                const int b = lt & 1, v = lt >> 1;
                const int count = DEEP ? min(in_chain, slabs - chain * in_chain) : slabs;
                if (!DEEP || ++chain == chains) tile += pairs, chain = 0;
                if (lt >= 2) ok = wait(acc_empty0 + 8 * b, (v - 1) & 1);     // both epilogues have drained this accumulator
                const uint32_t acc = tmem + (uint32_t)(b * 256);
                for (int i = 0; i < count && ok; ++i) {
                    if (!early) ok = wait(full0 + 8 * s, phase);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const int next = s + 1 == a.stages ? 0 : s + 1, next_phase = phase ^ (next == 0);
                    bool there = false;
                    if (issuer) {
                        // The next stage is asked for first: its answer, 200 clocks of the 500 that a turn of this warp took beside the MMAs (720 of a slab of 256
                        // columns), is on its way while these are issued (65,536 rows 1024 -> 1024 126 us -> 100, with SiLU, residual and z 147 -> 137).
                        there = mbar_test(full0 + 8 * next, next_phase);
                        const uint32_t at = (uint32_t)s * next_stage;
#pragma unroll
                        for (int k = 0; k < BK / 16; ++k) umma_f16_pair(acc, a0 + at + 2 * k, b0 + at + b_step * k, idesc, i > 0 || k > 0 ? 1u : 0u);
                        umma_commit_pair(empty0 + 8 * s);
                    }
                    early = __any_sync(0xffffffffu, there) != 0;
                    s = next, phase = next_phase;
                }
                if (ok && issuer) umma_commit_pair(acc_full0 + 8 * b);
                __syncwarp();
            }
            if (issuer) await_mmas_pair(done);
            __syncwarp();
        } else if (lane == 0) {
            mbar_wait(done, 0);
        }
    } else {
        // A lane holds a row's 32 columns of the accumulator.  Pieces of 32 rows x 64 bytes lie in shared memory with the 64B swizzle (conflict-free by
        // rows) and are moved by TMA, which leaves out what lies beyond the matrix: the residual arrives where y is then put together.
        const int w = warp - 2, q = warp & 3, first = w / 4 * kPiece;      // a warp may only read its own quarter of the TMEM lanes
        constexpr int step = kEpilogueWarps / 4 * kPiece;
        const uint32_t leader_acc_empty0 = in_leader(acc_empty0);
        const int own = staging + w * per_warp;
        const uint32_t swizzle = lane >> 1 & 3, my_res0 = res0 + 16 * w;
        const T* bias = static_cast<const T*>(a.bias);
        auto row_of = [&](int tile) { return (int64_t)(tile / a.n_panels) * (2 * BM) + rank * BM + q * 32; };
        auto fetch = [&](int tile, int c0, int s) {               // the residual's piece into buffer s, whose last store has been read
            const int64_t row = row_of(tile);
            const int col = tile % a.n_panels * a.n_tile + c0;
            if (row >= a.M || col >= a.N) return;
            mbar_expect_tx(my_res0 + 8 * s, kPieceBytes);
            tma_load_2d(base + own + s * kPieceBytes, &tmR, col, (int)row, my_res0 + 8 * s);
        };
        uint32_t res_phase = 0;                                   // a bit a buffer
        int lt = 0, s = 0;
        if (a.residual && lane == 0 && pair < a.tiles && first < a.n_tile) fetch(pair, first, 0);
        for (int tile = pair; tile < a.tiles && ok; tile += pairs, ++lt) {
            [[maybe_unused]] float held[kPiece];
            if constexpr (DEEP) {
#pragma unroll
                for (int j = 0; j < kPiece; ++j) held[j] = 0.f;
                for (int chain = 1; chain < chains; ++chain, ++lt) {
                    ok = __all_sync(0xffffffffu, mbar_wait(acc_full0 + 8 * (lt & 1), lt >> 1 & 1));
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    if (first < a.n_tile) {
                        const uint32_t at = tmem + (uint32_t)((lt & 1) * 256 + first) + ((uint32_t)(q * 32) << 16);
                        uint32_t r[kPiece];
                        __syncwarp();
                        tmem_ld16(at, r);
                        tmem_ld16(at + 16, r + 16);
                        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                        for (int j = 0; j < kPiece; ++j) held[j] += __uint_as_float(r[j]);
                    }
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster(leader_acc_empty0 + 8 * (lt & 1));
                }
                if (!ok) break;
            }
            const int b = lt & 1, v = lt >> 1;
            const int n0 = tile % a.n_panels * a.n_tile;
            const int64_t row0 = row_of(tile);
            const uint32_t acc = tmem + (uint32_t)(b * 256) + ((uint32_t)(q * 32) << 16);
            ok = __all_sync(0xffffffffu, mbar_wait(acc_full0 + 8 * b, v & 1));     // tcgen05.ld is warp-collective
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (first >= a.n_tile) {                              // nothing here for this warp
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(leader_acc_empty0 + 8 * b);
                continue;
            }
            for (int c0 = first; c0 < a.n_tile; c0 += step, s ^= 1) {
                uint32_t r[kPiece];
                __syncwarp();                                     // one lane has stored the last piece
                tmem_ld16(acc + (uint32_t)c0, r);
                tmem_ld16(acc + (uint32_t)c0 + 16, r + 16);
                const int col0 = n0 + c0;
                const bool live = row0 < a.M && col0 < a.N;       // the same for the warp
                if (lane == 0) {
                    bulk_wait_read();                             // what the last piece stored has left the buffers
                    if (a.residual) {
                        const bool more = c0 + step < a.n_tile;
                        if (more || tile + pairs < a.tiles) fetch(more ? tile : tile + pairs, more ? c0 + step : first, s ^ 1);
                    }
                }
                __syncwarp();
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                if constexpr (DEEP) {
#pragma unroll
                    for (int j = 0; j < kPiece; ++j) r[j] = __float_as_uint(held[j] + __uint_as_float(r[j]));
                }
                if (c0 + step >= a.n_tile) {                      // the accumulator has been read: its next tile may start
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster(leader_acc_empty0 + 8 * b);
                }
                if (!live) continue;
                if (a.residual) {
                    ok = __all_sync(0xffffffffu, mbar_wait(my_res0 + 8 * s, res_phase >> s & 1));
                    if (!ok) break;
                    res_phase ^= 1u << s;
                }
                unsigned char* y_row = gbase + own + s * kPieceBytes + lane * 64;
                unsigned char* z_row = gbase + own + 2 * kPieceBytes + lane * 64;
                uint32_t positive = 0u;
#pragma unroll
                for (int j = 0; j < kPiece / 8; ++j) {            // eight columns: 16 bytes
                    float_pair z[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) z[e] = pair_of(__uint_as_float(r[8 * j + 2 * e]), __uint_as_float(r[8 * j + 2 * e + 1]));
                    if (bias) {
                        const int c = col0 + 8 * j;
                        if (a.whole_bias && c + 8 <= a.N) {
                            const uint4 t = __ldg(reinterpret_cast<const uint4*>(bias + c));
                            const uint32_t u[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
                            for (int e = 0; e < 4; ++e) z[e] = add2(z[e], Pair<T>::two(u[e]));
                        } else {
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                z[e] = add2(z[e], pair_of(c + 2 * e < a.N ? Pair<T>::one(bias[c + 2 * e]) : 0.f, c + 2 * e + 1 < a.N ? Pair<T>::one(bias[c + 2 * e + 1]) : 0.f));
                        }
                    }
                    const uint32_t at = ((uint32_t)j ^ swizzle) * 16;
                    if (ACT != DG_ACT_NONE && a.save_z)
                        *reinterpret_cast<uint4*>(z_row + at) = make_uint4(Pair<T>::narrow(z[0]), Pair<T>::narrow(z[1]), Pair<T>::narrow(z[2]), Pair<T>::narrow(z[3]));
                    if (ACT == DG_ACT_RELU && a.bits) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float2 f = halves(z[e]);
                            positive |= ((f.x <= 0.f ? 0u : 1u) | (f.y <= 0.f ? 0u : 2u)) << (8 * j + 2 * e);
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) z[e] = act_value2<ACT>(z[e]);
                    uint4* to = reinterpret_cast<uint4*>(y_row + at);
                    if (a.residual) {
                        const uint4 t = *to;
                        const uint32_t u[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) z[e] = add2(z[e], Pair<T>::two(u[e]));
                    }
                    *to = make_uint4(Pair<T>::narrow(z[0]), Pair<T>::narrow(z[1]), Pair<T>::narrow(z[2]), Pair<T>::narrow(z[3]));
                }
                if (ACT == DG_ACT_RELU && a.bits && row0 + lane < a.M) a.bits[(row0 + lane) * a.ldbits + col0 / 32] = positive;
                fence_async();
                __syncwarp();
                if (lane == 0) {
                    tma_store_2d(&tmY, col0, (int)row0, base + own + s * kPieceBytes);
                    if (ACT != DG_ACT_NONE && a.save_z) tma_store_2d(&tmZ, col0, (int)row0, base + own + 2 * kPieceBytes);
                    bulk_commit();
                }
            }
        }
        if (lane == 0) bulk_wait();
        __syncwarp();
    }
    if (!ok) atomicExch(a.status, 1);
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    cluster_sync();                                               // no CTA leaves while the other's MMAs read its operands or arrive at its barriers
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
}

// ---- the weight gradient --------------------------------------------------------------------------------------------------
// A CTA owns a panel of up to 256 x 256 of dw and a range of rows.  Both operands come in boxes of 64 columns x 64 rows (MN-major); x's columns lie along
// the MMA's 128 rows, so a panel wider than 128 takes two accumulators.  The range's partial goes to scratch, four columns of dz and all of x's side by
// side; a second kernel adds the ranges in order.
// One range (fewer than 512 rows, or more than 74 panels) of one chain is written as it is.
// What bounds it: the tensor cores for wide layers (65,536 rows 1024 x 1024 91 us, 1,502 TFLOP/s), HBM for the others (232,965 rows 602 x 41 63 us, 4.8 TB/s).
// A chain of accumulations ends after kChainTerms rows, and the CTA adds the accumulators to its partial result: with ranges of one chain each, 300,000 x 264, 2304 fp16 were
// 2.3e-4 too small and 131,072 x 2304, 2304, whose 81 panels leave one range, 7.8e-4.
constexpr int kDwRows = 64, kDwBox = kDwRows * 128, kDwThreads = 32 * 6, kDwMaxStages = 8;
constexpr int kDwBarBytes = 8 * (2 * kDwMaxStages + 3) + 8;

struct LinearDwArgs {
    float4* partial;                              // [range][panel][q_store / 4][p_store]; null: the one range's sums are the result
    void* dw;
    int64_t row_stride, col_stride;
    int64_t M, rows_per_range;
    int32_t p_cols, q_cols;                       // K, N
    int32_t p_panels, q_panels, p_store, q_store;
    int32_t stages, p_boxes, q_boxes;             // of a full panel
    int* status;
    // k_linear_back
    const uint32_t* bits;
    int64_t ldbits;
    void* db;                                     // or null
    float* db_partial;                            // [range][N]; null: the one range's sums are the result
    int32_t store;                                // dz is kept
};

// What a CTA does: its panel and range.
struct DwPart {
    int panels, panel, range, p0, q0, p_boxes, q_boxes, halves, q_pad, slabs;
    int64_t r0;
    __device__ __forceinline__ DwPart(const LinearDwArgs& a, int rows)
    {
        panels = a.p_panels * a.q_panels, panel = blockIdx.x % panels, range = blockIdx.x / panels;
        p0 = panel / a.q_panels * 256, q0 = panel % a.q_panels * 256;
        const int p_here = min(256, a.p_cols - p0), q_here = min(256, a.q_cols - q0);
        p_boxes = (p_here + 63) / 64, q_boxes = (q_here + 63) / 64, halves = (p_here + 127) / 128, q_pad = (q_here + 15) / 16 * 16;
        r0 = range * a.rows_per_range;
        slabs = (int)((max((int64_t)0, min(a.M, r0 + a.rows_per_range) - r0) + rows - 1) / rows);
    }
};

// The accumulators of a CTA, by four warps: to its place among the partial results, added to what its earlier chains left there, or where it has the only chain
// rounded to dw.
template <class T> __device__ __forceinline__ void flush_dw(const LinearDwArgs& a, const DwPart& part, uint32_t tmem, int warp, int lane, bool add)
{
    const int q = warp & 3;                                       // a warp may only read its own quarter of the TMEM lanes
    const bool whole = a.col_stride == 1 && a.row_stride % 8 == 0 && (reinterpret_cast<uintptr_t>(a.dw) & 15) == 0;
    for (int h = 0; h < part.halves; ++h) {
        const int row = h * 128 + q * 32 + lane, p = part.p0 + row;
        float4* to_part = a.partial + ((int64_t)part.range * part.panels + part.panel) * (a.q_store / 4) * a.p_store + row;
        for (int c0 = 0; c0 < part.q_pad; c0 += 16) {
            uint32_t r[16];
            __syncwarp();                                         // tcgen05.ld is warp-collective, and lanes have stored as many columns as they have
            tmem_ld16(tmem + (uint32_t)(h * 256 + c0) + ((uint32_t)(q * 32) << 16), r);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
            if (a.partial) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (row < a.p_store) {
                        float4* const to = to_part + (int64_t)(c0 / 4 + j) * a.p_store;
                        float4 v = make_float4(__uint_as_float(r[4 * j]), __uint_as_float(r[4 * j + 1]), __uint_as_float(r[4 * j + 2]), __uint_as_float(r[4 * j + 3]));
                        if (add) {
                            const float4 u = __ldcg(to);
                            v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
                        }
                        __stcg(to, v);
                    }
                continue;
            }
            T* to = static_cast<T*>(a.dw) + p * a.row_stride + (part.q0 + c0) * a.col_stride;
            if (p < a.p_cols) {
                if (whole && part.q0 + c0 + 16 <= a.q_cols) {
                    uint32_t v[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] = Pair<T>::narrow(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1]));
                    reinterpret_cast<uint4*>(to)[0] = make_uint4(v[0], v[1], v[2], v[3]);
                    reinterpret_cast<uint4*>(to)[1] = make_uint4(v[4], v[5], v[6], v[7]);
                } else {
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if (part.q0 + c0 + j < a.q_cols) to[j * a.col_stride] = Pair<T>::round(__uint_as_float(r[j]));
                }
            }
        }
    }
}

template <class T>
__global__ void __launch_bounds__(kDwThreads, 1) k_linear_dw(const __grid_constant__ CUtensorMap tmP, const __grid_constant__ CUtensorMap tmQ, const LinearDwArgs a)
{
    extern __shared__ unsigned char smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    unsigned char* gbase = smem_raw + (base - raw);
    const int stage_bytes = (a.p_boxes + a.q_boxes) * kDwBox;
    const uint32_t bars = base + a.stages * stage_bytes;
    const uint32_t full0 = bars, empty0 = bars + 8 * kDwMaxStages, acc_full = bars + 16 * kDwMaxStages, acc_empty = acc_full + 8, done = acc_full + 16;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(gbase + a.stages * stage_bytes + 8 * (2 * kDwMaxStages + 3));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const DwPart part(a, kDwRows);
    constexpr int kTmemCols = 512, kChain = kChainTerms<T> / kDwRows;      // slabs of a chain

    if (threadIdx.x == 0) {
        for (int s = 0; s < a.stages; ++s) {
            mbar_init(full0 + 8 * s, 1);
            mbar_init(empty0 + 8 * s, 1);
        }
        mbar_init(acc_full, 1);
        mbar_init(acc_empty, 4);
        mbar_init(done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tmem_slot;
    bool ok = true;

    if (warp == 0) {
        if (lane == 0) {
            int s = 0, phase = 1, i = 0;
            for (; i < part.slabs && ok; ++i) {
                if (i >= a.stages) ok = mbar_wait(empty0 + 8 * s, phase);
                if (!ok) break;
                const uint32_t st = base + s * stage_bytes;
                const int row = (int)(part.r0 + (int64_t)i * kDwRows);
                mbar_expect_tx(full0 + 8 * s, (part.p_boxes + part.q_boxes) * kDwBox);
                for (int j = 0; j < part.p_boxes; ++j) tma_load_2d(st + j * kDwBox, &tmP, part.p0 + 64 * j, row, full0 + 8 * s);
                for (int j = 0; j < part.q_boxes; ++j) tma_load_2d(st + (a.p_boxes + j) * kDwBox, &tmQ, part.q0 + 64 * j, row, full0 + 8 * s);
                if (++s == a.stages) s = 0, phase ^= 1;
            }
            await_loads(full0, i, a.stages);
        }
    } else if (warp == 1) {
        const bool issuer = elect_one();
        auto wait = [&](uint32_t bar, int parity) { return __any_sync(0xffffffffu, issuer && mbar_wait(bar, parity)) != 0; };
        const uint32_t idesc = umma_idesc_f16(Pair<T>::kFormat, 128, part.q_pad, true, true);
        int s = 0, phase = 0;
        for (int chain = 0, left = part.slabs; left > 0 && ok; ++chain, left -= kChain) {
            // The chain before has left the accumulators.  All lanes ask: with one asking, as below, every stage's turn took 300 clocks more (65,536 rows 1024 x 1024 90 us -> 113).
            if (chain > 0) ok = __all_sync(0xffffffffu, mbar_wait(acc_empty, (chain - 1) & 1)) != 0;
            const int slabs = ok ? min(left, kChain) : 0;
            for (int i = 0; i < slabs && ok; ++i) {
                ok = wait(full0 + 8 * s, phase);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (issuer) {
                    const uint32_t st = base + s * stage_bytes;
                    const uint64_t p = umma_desc_mn16(st, kDwBox), q = umma_desc_mn16(st + a.p_boxes * kDwBox, kDwBox);
                    for (int h = 0; h < part.halves; ++h)
#pragma unroll
                        for (int k = 0; k < kDwRows / 16; ++k)    // 16 rows: 2048 bytes
                            umma_f16(tmem + (uint32_t)(h * 256), p + (uint32_t)((h * 2 * kDwBox + k * 2048) >> 4), q + (uint32_t)(k * 2048 >> 4), idesc,
                                     i > 0 || k > 0 ? 1u : 0u);
                    umma_commit(empty0 + 8 * s);
                }
                __syncwarp();
                if (++s == a.stages) s = 0, phase ^= 1;
            }
            if (ok && issuer) umma_commit(acc_full);
            __syncwarp();
        }
        if (issuer) await_mmas(done);
        __syncwarp();
    } else {
        const int chains = (part.slabs + kChain - 1) / kChain;
        for (int chain = 0; chain < chains; ++chain) {
            ok = __all_sync(0xffffffffu, mbar_wait(acc_full, chain & 1));      // tcgen05.ld is warp-collective
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            flush_dw<T>(a, part, tmem, warp, lane, chain > 0);
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(acc_empty);
        }
    }
    if (!ok) atomicExch(a.status, 1);
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
}

// The same product with dz made on the way, for x of up to 256 columns: dy arrives where dz is put together, z beside it; the operand that the tensor cores
// then read is also what TMA stores, and its column sums are taken by the threads that make it.  So the gradients of w and b and dz itself, which x's
// gradient needs, take one pass over x, dy and z; dz by a pass of its own reads and writes as much again (2,449,029 x 256, 256 bf16: 656 + 388 us, 732 this way).
// Warps: 0 TMA, 1 MMA issue + tensor-memory allocation, 2-9 dz (a row's 16-byte piece a thread and box of 32 rows x 64 columns), of which 2-5 flush, 10 stores dz.
constexpr int kBackRows = 32, kBackBox = kBackRows * 128, kBackMakers = 8, kBackThreads = 32 * (3 + kBackMakers), kBackMaxStages = 8;
constexpr int kBackBarBytes = 8 * (4 * kBackMaxStages + 3) + 8, kBackSumPitch = 9, kBackSumBytes = 32 * kBackMakers * kBackSumPitch * 4;

template <class T, int ACT>
__global__ void __launch_bounds__(kBackThreads, 1)
k_linear_back(const __grid_constant__ CUtensorMap tmP, const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmZ,
              const __grid_constant__ CUtensorMap tmS, const LinearDwArgs a)
{
    constexpr bool kSmooth = ACT == DG_ACT_GELU || ACT == DG_ACT_SILU;
    extern __shared__ unsigned char smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    unsigned char* gbase = smem_raw + (base - raw);
    const int q_at = a.p_boxes * kBackBox, z_at = q_at + a.q_boxes * kBackBox, stage_bytes = z_at + (kSmooth ? a.q_boxes * kBackBox : 0);
    float* sums = reinterpret_cast<float*>(gbase + a.stages * stage_bytes);
    const uint32_t bars = base + a.stages * stage_bytes + kBackSumBytes;
    const uint32_t full0 = bars, ready0 = bars + 8 * kBackMaxStages, empty0 = bars + 16 * kBackMaxStages, stored0 = bars + 24 * kBackMaxStages;
    const uint32_t acc_full = bars + 32 * kBackMaxStages, acc_empty = acc_full + 8, done = acc_full + 16;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(gbase + a.stages * stage_bytes + kBackSumBytes + 8 * (4 * kBackMaxStages + 3));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const DwPart part(a, kBackRows);
    constexpr int kTmemCols = 512, kChain = kChainTerms<T> / kBackRows;

    if (threadIdx.x == 0) {
        for (int s = 0; s < a.stages; ++s) {
            mbar_init(full0 + 8 * s, 1);
            mbar_init(ready0 + 8 * s, kBackMakers);
            mbar_init(empty0 + 8 * s, 1);
            mbar_init(stored0 + 8 * s, 1);
        }
        mbar_init(acc_full, 1);
        mbar_init(acc_empty, 4);
        mbar_init(done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tmem_slot;
    bool ok = true;

    if (warp == 0) {
        if (lane == 0) {
            int s = 0, phase = 1, i = 0;
            for (; i < part.slabs && ok; ++i) {
                if (i >= a.stages) ok = mbar_wait(empty0 + 8 * s, phase) && (!a.store || mbar_wait(stored0 + 8 * s, phase));
                if (!ok) break;
                const uint32_t st = base + s * stage_bytes;
                const int row = (int)(part.r0 + (int64_t)i * kBackRows);
                mbar_expect_tx(full0 + 8 * s, (part.p_boxes + (kSmooth ? 2 : 1) * part.q_boxes) * kBackBox);
                for (int j = 0; j < part.q_boxes; ++j) {
                    tma_load_2d(st + q_at + j * kBackBox, &tmQ, part.q0 + 64 * j, row, full0 + 8 * s);
                    if (kSmooth) tma_load_2d(st + z_at + j * kBackBox, &tmZ, part.q0 + 64 * j, row, full0 + 8 * s);
                }
                for (int j = 0; j < part.p_boxes; ++j) tma_load_2d(st + j * kBackBox, &tmP, part.p0 + 64 * j, row, full0 + 8 * s);
                if (++s == a.stages) s = 0, phase ^= 1;
            }
            await_loads(full0, i, a.stages);
        }
    } else if (warp == 1) {
        const bool issuer = elect_one();
        auto wait = [&](uint32_t bar, int parity) { return __any_sync(0xffffffffu, issuer && mbar_wait(bar, parity)) != 0; };
        const uint32_t idesc = umma_idesc_f16(Pair<T>::kFormat, 128, part.q_pad, true, true);
        int s = 0, phase = 0;
        for (int chain = 0, left = part.slabs; left > 0 && ok; ++chain, left -= kChain) {
            if (chain > 0) ok = __all_sync(0xffffffffu, mbar_wait(acc_empty, (chain - 1) & 1)) != 0;
            const int slabs = ok ? min(left, kChain) : 0;
            for (int i = 0; i < slabs && ok; ++i) {
                ok = wait(ready0 + 8 * s, phase);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (issuer) {
                    const uint32_t st = base + s * stage_bytes;
                    const uint64_t p = umma_desc_mn16(st, kBackBox), q = umma_desc_mn16(st + q_at, kBackBox);
                    for (int h = 0; h < part.halves; ++h)
#pragma unroll
                        for (int k = 0; k < kBackRows / 16; ++k)  // 16 rows: 2048 bytes
                            umma_f16(tmem + (uint32_t)(h * 256), p + (uint32_t)((h * 2 * kBackBox + k * 2048) >> 4), q + (uint32_t)(k * 2048 >> 4), idesc,
                                     i > 0 || k > 0 ? 1u : 0u);
                    umma_commit(empty0 + 8 * s);
                }
                __syncwarp();
                if (++s == a.stages) s = 0, phase ^= 1;
            }
            if (ok && issuer) umma_commit(acc_full);
            __syncwarp();
        }
        if (issuer) await_mmas(done);
        __syncwarp();
    } else if (warp < 2 + kBackMakers) {
        const int t = threadIdx.x - 64, row = t >> 3, piece = (t & 7) ^ (row & 7);      // the swizzle: which eight columns of a box lie here
        float_pair sum[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[j][e] = both(0.f);
        // The accumulators at a chain's end, by the first four of these warps; the others are held up by the barriers of the stages that follow.
        auto flush = [&](int chain) {
            ok = __all_sync(0xffffffffu, mbar_wait(acc_full, chain & 1));      // tcgen05.ld is warp-collective
            if (!ok) return;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            flush_dw<T>(a, part, tmem, warp, lane, chain > 0);
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(acc_empty);
        };
        int s = 0, phase = 0;
        for (int i = 0; i < part.slabs; ++i) {
            uint32_t above[4] = {0u, 0u, 0u, 0u};
            if constexpr (ACT == DG_ACT_RELU) {                   // on their way while the stage is waited for
                const int64_t at = part.r0 + (int64_t)i * kBackRows + row;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int c = part.q0 + 64 * j + 8 * piece;
                    if (at < a.M && c < a.q_cols) above[j] = __ldg(reinterpret_cast<const unsigned char*>(a.bits + at * a.ldbits) + c / 8);
                }
            }
            ok = __all_sync(0xffffffffu, mbar_wait(full0 + 8 * s, phase));
            if (!ok) break;
            unsigned char* st = gbase + (size_t)s * stage_bytes + t * 16;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (j >= part.q_boxes) break;
                uint4* at = reinterpret_cast<uint4*>(st + q_at + j * kBackBox);
                uint4 v = *at;
                float_pair g[4] = {Pair<T>::two(v.x), Pair<T>::two(v.y), Pair<T>::two(v.z), Pair<T>::two(v.w)};
                if constexpr (ACT == DG_ACT_RELU) {
                    const uint32_t m = above[j];
                    auto keep = [](uint32_t two) { return (two & 1 ? 0xFFFFu : 0u) | (two & 2 ? 0xFFFF0000u : 0u); };
                    v = make_uint4(v.x & keep(m), v.y & keep(m >> 2), v.z & keep(m >> 4), v.w & keep(m >> 6));
                    g[0] = Pair<T>::two(v.x), g[1] = Pair<T>::two(v.y), g[2] = Pair<T>::two(v.z), g[3] = Pair<T>::two(v.w);
                    *at = v;
                } else if constexpr (kSmooth) {
                    const uint4 u = *reinterpret_cast<const uint4*>(st + z_at + j * kBackBox);
                    g[0] = mul2(g[0], act_slope2<ACT>(Pair<T>::two(u.x))), g[1] = mul2(g[1], act_slope2<ACT>(Pair<T>::two(u.y)));
                    g[2] = mul2(g[2], act_slope2<ACT>(Pair<T>::two(u.z))), g[3] = mul2(g[3], act_slope2<ACT>(Pair<T>::two(u.w)));
                    *at = make_uint4(Pair<T>::narrow(g[0]), Pair<T>::narrow(g[1]), Pair<T>::narrow(g[2]), Pair<T>::narrow(g[3]));
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[j][e] = add2(sum[j][e], g[e]);
            }
            if (ACT != DG_ACT_NONE) fence_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(ready0 + 8 * s);
            if (++s == a.stages) s = 0, phase ^= 1;
            if (warp < 6 && i % kChain == kChain - 1 && i + 1 < part.slabs) {
                flush(i / kChain);
                if (!ok) break;
            }
        }
        if (a.db) {                                               // box by box: the 32 rows of a column, in order
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (j >= part.q_boxes) break;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 f = halves(sum[j][e]);
                    sums[t * kBackSumPitch + 2 * e] = f.x, sums[t * kBackSumPitch + 2 * e + 1] = f.y;
                }
                __syncwarp();
                asm volatile("bar.sync 1, %0;" ::"n"(32 * kBackMakers) : "memory");
                const int c = part.q0 + 64 * j + t;
                if (t < 64 && c < a.q_cols) {
                    float total = 0.f;
#pragma unroll 8
                    for (int r = 0; r < 32; ++r) total += sums[(r * 8 + (t >> 3 ^ (r & 7))) * kBackSumPitch + (t & 7)];
                    if (a.db_partial) a.db_partial[(int64_t)part.range * a.q_cols + c] = total;
                    else static_cast<T*>(a.db)[c] = Pair<T>::round(total);
                }
                __syncwarp();
                asm volatile("bar.sync 1, %0;" ::"n"(32 * kBackMakers) : "memory");
            }
        }
        if (warp < 6 && ok && part.slabs > 0) flush((part.slabs - 1) / kChain);
    } else if (lane == 0 && a.store) {
        int s = 0, phase = 0;
        for (int i = 0; i < part.slabs; ++i) {
            ok = mbar_wait(ready0 + 8 * s, phase);
            if (!ok) break;
            const int row = (int)(part.r0 + (int64_t)i * kBackRows);
            for (int j = 0; j < part.q_boxes; ++j) tma_store_2d(&tmS, part.q0 + 64 * j, row, base + s * stage_bytes + q_at + j * kBackBox);
            bulk_commit();
            bulk_wait_read();
            mbar_arrive(stored0 + 8 * s);
            if (++s == a.stages) s = 0, phase ^= 1;
        }
        bulk_wait();
    }
    if (!ok) atomicExch(a.status, 1);
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
}

// dw[p, q] = sum of the ranges' partials: a thread takes four columns of a row and an eighth of the ranges, in their order; the eighths are added in theirs.
template <class T>
__global__ void __launch_bounds__(256) k_linear_dw_reduce(const float4* __restrict__ partial, int ranges, int32_t p_panels, int32_t q_panels, int32_t p_store,
                                                          int32_t q_store, int32_t p_cols, int32_t q_cols, T* __restrict__ dw, int64_t row_stride, int64_t col_stride)
{
    __shared__ float4 part[8][32];
    const int panels = p_panels * q_panels, per_panel = q_store / 4 * p_store, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t i = (int64_t)blockIdx.x * 32 + lane, stride = (int64_t)panels * per_panel;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    if (i < stride) {
        const int each = (ranges + 7) / 8, end = min(ranges, (warp + 1) * each);
        const float4* from = partial + i;
#pragma unroll 8
        for (int r = warp * each; r < end; ++r) {
            const float4 v = __ldcg(from + r * stride);
            sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
        }
    }
    part[warp][lane] = sum;
    __syncthreads();
    if (warp || i >= stride) return;
    for (int w = 1; w < 8; ++w) {
        const float4 v = part[w][lane];
        sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
    }
    const int panel = (int)(i / per_panel), in = (int)(i % per_panel);
    const int p = panel / q_panels * 256 + in % p_store, q = panel % q_panels * 256 + in / p_store * 4;
    if (p >= p_cols) return;
    const float s[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (q + j < q_cols) dw[p * row_stride + (q + j) * col_stride] = Pair<T>::round(s[j]);
}

// ---- dz = dy act'(z) and its column sums ------------------------------------------------------------------------------------
// A thread owns eight neighbouring columns and walks over rows; the lanes of a row read neighbouring pieces.  `lanes` threads a row (a power of two), a
// CTA takes 8 * lanes columns and every (256 / lanes * gridDim.x)-th row.
constexpr int kDzThreads = 256;
// Eight neighbouring elements as they lie in memory.
template <class T> struct Raw {
    uint4 v[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T* p)
    {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
    }
    __device__ __forceinline__ void load(const T* p, int n)
    {
        T* e = reinterpret_cast<T*>(v);
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = i < n ? p[i] : Pair<T>::round(0.f);
    }
    __device__ __forceinline__ void wide(float* to) const
    {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 8; ++i) to[i] = reinterpret_cast<const float*>(v)[i];
        } else {
            const uint32_t u[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 f = Pair<T>::wide(u[e]);
                to[2 * e] = f.x, to[2 * e + 1] = f.y;
            }
        }
    }
};
template <class T> __device__ __forceinline__ void store8(T* p, int n, bool whole, const float* v)
{
    if (whole && n >= 8) {
        if constexpr (sizeof(T) == 4) {
            reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
            reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            *reinterpret_cast<uint4*>(p) = make_uint4(Pair<T>::narrow(v[0], v[1]), Pair<T>::narrow(v[2], v[3]), Pair<T>::narrow(v[4], v[5]), Pair<T>::narrow(v[6], v[7]));
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < n) p[e] = Pair<T>::round(v[e]);
    }
}

struct LinearDzArgs {
    int64_t lddy, ldz, ldbits, lddz, M;
    const uint32_t* bits;
    float* partial;                               // [gridDim.x][N], or null
    void* db;                                     // one CTA over the rows: its sums are the result
    int32_t N, lanes, whole_dy, whole_z, whole_dz;
};

template <class T, int ACT>
__global__ void __launch_bounds__(kDzThreads, 3) k_linear_dz(const T* __restrict__ dy, const T* __restrict__ z, T* __restrict__ dz, const LinearDzArgs a)
{
    __shared__ float sums[kDzThreads][9];
    const int lane = threadIdx.x & (a.lanes - 1), group = threadIdx.x / a.lanes, groups = kDzThreads / a.lanes;
    const int c = (blockIdx.y * a.lanes + lane) * 8, n = min(8, a.N - c);
    float sum[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[e] = 0.f;
    const int64_t step = (int64_t)gridDim.x * groups;
    auto work = [&](int64_t row, const Raw<T>& from, const Raw<T>& pre, uint32_t word) {
        float g[8];
        from.wide(g);
        if constexpr (ACT == DG_ACT_RELU) {
#pragma unroll
            for (int e = 0; e < 8; ++e) g[e] = word >> e & 1 ? g[e] : 0.f;
        } else if constexpr (ACT != DG_ACT_NONE) {
            float v[8];
            pre.wide(v);
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                if constexpr (sizeof(T) == 4) {
                    g[e] *= act_slope<ACT>(v[e]), g[e + 1] *= act_slope<ACT>(v[e + 1]);
                } else {
                    const float2 f = halves(mul2(pair_of(g[e], g[e + 1]), act_slope2<ACT>(pair_of(v[e], v[e + 1]))));
                    g[e] = f.x, g[e + 1] = f.y;
                }
            }
        }
        if (dz) store8(dz + row * a.lddz + c, n, a.whole_dz, g);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] += g[e];
    };
    auto bits_of = [&](int64_t row) { return ACT == DG_ACT_RELU ? __ldg(a.bits + row * a.ldbits + c / 32) >> (c % 32) : 0u; };
    int64_t row = (int64_t)blockIdx.x * groups + group;
    constexpr bool smooth = ACT == DG_ACT_GELU || ACT == DG_ACT_SILU;
    if (n == 8 && a.whole_dy && (!smooth || a.whole_z)) {
        constexpr int U = sizeof(T) == 4 ? 2 : 4;                 // rows in flight
        for (; row + (U - 1) * step < a.M; row += U * step) {
            Raw<T> from[U], pre[U];
            uint32_t word[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                from[u].load(dy + (row + u * step) * a.lddy + c);
                if constexpr (smooth) pre[u].load(z + (row + u * step) * a.ldz + c);
                word[u] = bits_of(row + u * step);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) work(row + u * step, from[u], pre[u], word[u]);
        }
    }
    if (n > 0)
        for (; row < a.M; row += step) {
            Raw<T> from, pre;
            from.load(dy + row * a.lddy + c, n);
            if constexpr (smooth) pre.load(z + row * a.ldz + c, n);
            work(row, from, pre, bits_of(row));
        }
    if (!a.partial && !a.db) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) sums[threadIdx.x][e] = sum[e];
    __syncthreads();
    for (int i = threadIdx.x; i < a.lanes * 8; i += kDzThreads) {
        const int l = i / 8, col = blockIdx.y * a.lanes * 8 + i;
        if (col >= a.N) continue;
        float s = 0.f;
        for (int k = 0; k < groups; ++k) s += sums[k * a.lanes + l][i % 8];
        if (a.db) static_cast<T*>(a.db)[col] = Pair<T>::round(s);
        else a.partial[(int64_t)blockIdx.x * a.N + col] = s;
    }
}

// db: 32 columns a CTA, 32 warps share the parts.
template <class T> __global__ void __launch_bounds__(1024) k_linear_db(const float* __restrict__ partial, int parts, int32_t N, T* __restrict__ db)
{
    __shared__ double sums[32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
    double s = 0.0;
    if (col < N)
#pragma unroll 8
        for (int i = warp; i < parts; i += 32) s += __ldg(partial + (int64_t)i * N + col);
    sums[warp][lane] = s;
    __syncthreads();
    if (warp || col >= N) return;
    for (int w = 1; w < 32; ++w) s += sums[w][lane];
    db[col] = Pair<T>::round((float)s);
}

// The CTAs over the rows: enough to fill the device twice over, and at least 32 rows a thread.
int dz_lanes(int32_t N)
{
    int lanes = 1;
    while (lanes < 32 && lanes * 8 < N) lanes *= 2;
    return lanes;
}
int dz_ctas(int64_t M, int32_t N)
{
    const int lanes = dz_lanes(N), columns = (N + lanes * 8 - 1) / (lanes * 8);
    const int64_t most = std::max(1, 148 * 6 / columns), rows = kDzThreads / lanes * 32;
    return (int)std::min<int64_t>(most, (M + rows - 1) / rows);
}

// ---- few rows -----------------------------------------------------------------------------------------------------------------
// 16 bits: y^T by mma.m16n8k16 with x along the 16 rows.  The order in which k goes through the sum is free as long as both operands agree on it, so a thread
// takes four neighbouring k's of both: 8 bytes of a row of x, and four rows (w [K x N], four neighbouring columns each, which are then columns of four
// MMAs) or 8 bytes of a row (w [N x K]) of w.  A CTA makes 32 columns, or 16; its warps share K, and their sums meet in shared memory.  Rows and columns
// beyond the matrix are read as the last ones, so that the loads of four steps go out together: with a question at each, 16 x 1024 -> 1024 took 10.3 us.
constexpr int kFewRows = 16, kFewWarps = 16;
template <bool OUT_IN> constexpr int kFewCols = OUT_IN ? 16 : 32;

template <class T> __device__ __forceinline__ uint2 load4(const T* p, int n, bool whole)
{
    if (whole && n >= 4) return __ldg(reinterpret_cast<const uint2*>(p));
    unsigned short v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = e < n ? __ldg(reinterpret_cast<const unsigned short*>(p) + e) : (unsigned short)0;
    return make_uint2(v[0] | (uint32_t)v[1] << 16, v[2] | (uint32_t)v[3] << 16);
}
template <class T> __device__ __forceinline__ void mma16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1)
{
    if constexpr (Pair<T>::kFormat == 1)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

struct FewArgs {
    const void *x, *w, *bias, *residual;
    void *y, *z;
    uint32_t* bits;
    int64_t ldx, ldw, ldr, ldy, ldz, ldbits, M;
    int32_t N, K, act, whole_x, whole_w;
};

// One element of the result, from its sum.  Lanes of a warp, or of half a warp, hold as many neighbouring columns of a row, the first a multiple of their number;
// elements beyond the matrix are not written.
template <class T> __device__ __forceinline__ void finish(const FewArgs& a, int64_t m, int col, float z)
{
    const bool live = col < a.N && m < a.M;
    if (live && a.bias) z += Pair<T>::one(static_cast<const T*>(a.bias)[col]);
    if (a.bits) {                                                 // 16 columns a half warp
        const uint32_t word = __ballot_sync(0xffffffffu, live && !(z <= 0.f)) >> (threadIdx.x & 16);
        if (threadIdx.x % 16 == 0 && m < a.M) reinterpret_cast<unsigned short*>(a.bits + m * a.ldbits)[col / 16] = (unsigned short)word;
    }
    if (!live) return;
    if (a.z) static_cast<T*>(a.z)[m * a.ldz + col] = Pair<T>::round(z);
    float y = a.act == DG_ACT_RELU ? act_value<DG_ACT_RELU>(z) : a.act == DG_ACT_GELU ? act_value<DG_ACT_GELU>(z) : a.act == DG_ACT_SILU ? act_value<DG_ACT_SILU>(z) : z;
    if (a.residual) y += Pair<T>::one(static_cast<const T*>(a.residual)[m * a.ldr + col]);
    static_cast<T*>(a.y)[m * a.ldy + col] = Pair<T>::round(y);
}

template <class T, bool OUT_IN>
__global__ void __launch_bounds__(32 * kFewWarps) k_few_rows16(const FewArgs a)
{
    constexpr int kCols = kFewCols<OUT_IN>, kMmas = kCols / 8;
    __shared__ float sums[kFewWarps][kFewRows][kCols + 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int64_t m0 = (int64_t)blockIdx.y * kFewRows;
    const int n0 = blockIdx.x * kCols;
    const T* x0 = static_cast<const T*>(a.x) + min(m0 + g, a.M - 1) * a.ldx;
    const T* x1 = static_cast<const T*>(a.x) + min(m0 + g + 8, a.M - 1) * a.ldx;
    const T* w = static_cast<const T*>(a.w);
    float acc[kMmas][4];
#pragma unroll
    for (int j = 0; j < kMmas; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[j][e] = 0.f;
    auto multiply = [&](const uint2& u0, const uint2& u1, const uint2* b) {
        const uint32_t xa[4] = {u0.x, u1.x, u0.y, u1.y};
        if constexpr (OUT_IN) {
#pragma unroll
            for (int j = 0; j < kMmas; ++j) mma16<T>(acc[j], xa, b[j].x, b[j].y);
        } else {
            mma16<T>(acc[0], xa, __byte_perm(b[0].x, b[1].x, 0x5410), __byte_perm(b[2].x, b[3].x, 0x5410));
            mma16<T>(acc[1], xa, __byte_perm(b[0].x, b[1].x, 0x7632), __byte_perm(b[2].x, b[3].x, 0x7632));
            mma16<T>(acc[2], xa, __byte_perm(b[0].y, b[1].y, 0x5410), __byte_perm(b[2].y, b[3].y, 0x5410));
            mma16<T>(acc[3], xa, __byte_perm(b[0].y, b[1].y, 0x7632), __byte_perm(b[2].y, b[3].y, 0x7632));
        }
    };
    constexpr int kLoads = OUT_IN ? kMmas : 4;
    const T* from[kLoads];                                        // of w, for k = 4 t
#pragma unroll
    for (int j = 0; j < kLoads; ++j)
        from[j] = OUT_IN ? w + (int64_t)min(n0 + 8 * j + g, a.N - 1) * a.ldw : w + (int64_t)j * a.ldw + min(n0 + 4 * g, (a.N - 1) / 4 * 4);
    // A chain's sums, to or on the warp's own.  Chains end as those of the tensor cores' kernels do: 16 x 1,048,576 -> 48 fp16 was 4e-4 too small in one.
    constexpr int kChain = kChainTerms<T> / 16;
    bool more = false;
    auto put = [&]() {
#pragma unroll
        for (int j = 0; j < kMmas; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int in_mma = 2 * t + (e & 1), col = OUT_IN ? 8 * j + in_mma : 4 * in_mma + j;
                float* const to = &sums[warp][g + (e & 2) * 4][col];
                *to = more ? *to + acc[j][e] : acc[j][e];
                acc[j][e] = 0.f;
            }
        more = true;
    };
    int step = warp;
    if (a.whole_x && a.whole_w) {
        const int whole_steps = a.K / 16;
        while (true) {
            const int stop = min(whole_steps, step + kChain * kFewWarps);
#pragma unroll 4
            for (; step < stop; step += kFewWarps) {
                const int k = step * 16 + 4 * t;
                const uint2 u0 = __ldg(reinterpret_cast<const uint2*>(x0 + k)), u1 = __ldg(reinterpret_cast<const uint2*>(x1 + k));
                uint2 b[kLoads];
#pragma unroll
                for (int j = 0; j < kLoads; ++j) b[j] = __ldg(reinterpret_cast<const uint2*>(from[j] + (OUT_IN ? (int64_t)k : k * a.ldw)));
                multiply(u0, u1, b);
            }
            if (step >= whole_steps) break;
            put();
        }
    }
    for (int n = 0; step * 16 < a.K; step += kFewWarps, ++n) {    // other alignments, and the last step of an odd K
        if (n > 0 && n % kChain == 0) put();
        const int k = step * 16 + 4 * t, nk = a.K - k, nn = a.N - min(n0 + 4 * g, (a.N - 1) / 4 * 4);
        uint2 b[kLoads];
#pragma unroll
        for (int j = 0; j < kLoads; ++j)
            b[j] = OUT_IN ? load4(from[j] + k, nk, a.whole_w) : j < nk ? load4(from[j] + k * a.ldw, nn, a.whole_w) : make_uint2(0u, 0u);
        multiply(load4(x0 + k, nk, a.whole_x), load4(x1 + k, nk, a.whole_x), b);
    }
    put();
    __syncthreads();
    const int m = threadIdx.x / kCols, col = threadIdx.x % kCols;      // a warp has 32 columns of a row, or 16 of two
    if (m >= kFewRows) return;
    float z = 0.f;
#pragma unroll
    for (int s = 0; s < kFewWarps; ++s) z += sums[s][m][col];
    finish<T>(a, m0 + m, n0 + col, z);
}

// fp32: a lane owns a column of w [K x N] (its warp's share of K), or a warp a row of w [N x K] with K along the lanes; x is read through the L1.
constexpr int kFewWarps32 = 16;
template <bool OUT_IN, int ROWS> __global__ void __launch_bounds__(32 * kFewWarps32) k_few_rows32(const FewArgs a)
{
    __shared__ float sums[kFewWarps32][ROWS][33];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t m0 = (int64_t)blockIdx.y * ROWS;
    const int n0 = blockIdx.x * 32;
    const float* x[ROWS];
#pragma unroll
    for (int m = 0; m < ROWS; ++m) x[m] = static_cast<const float*>(a.x) + min(m0 + m, a.M - 1) * a.ldx;
    const float* w = static_cast<const float*>(a.w);
    if constexpr (!OUT_IN) {
        float acc[ROWS] = {};
        const float* from = w + min(n0 + lane, a.N - 1);
#pragma unroll 16
        for (int k = warp; k < a.K; k += kFewWarps32) {
            const float v = __ldg(from + k * a.ldw);
#pragma unroll
            for (int m = 0; m < ROWS; ++m) acc[m] = fmaf(__ldg(x[m] + k), v, acc[m]);
        }
#pragma unroll
        for (int m = 0; m < ROWS; ++m) sums[warp][m][lane] = acc[m];
        __syncthreads();
        if (warp >= ROWS) return;
        float z = 0.f;
#pragma unroll
        for (int s = 0; s < kFewWarps32; ++s) z += sums[s][warp][lane];
        finish<float>(a, m0 + warp, n0 + lane, z);
    } else {
        float acc[2][ROWS] = {};                                  // columns n0 + 2 warp, n0 + 2 warp + 1
        const float *from0 = w + (int64_t)min(n0 + 2 * warp, a.N - 1) * a.ldw, *from1 = w + (int64_t)min(n0 + 2 * warp + 1, a.N - 1) * a.ldw;
#pragma unroll 8
        for (int k = lane; k < a.K; k += 32) {
            const float v0 = __ldg(from0 + k), v1 = __ldg(from1 + k);
#pragma unroll
            for (int m = 0; m < ROWS; ++m) {
                const float u = __ldg(x[m] + k);
                acc[0][m] = fmaf(u, v0, acc[0][m]);
                acc[1][m] = fmaf(u, v1, acc[1][m]);
            }
        }
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int m = 0; m < ROWS; ++m) {
                float v = acc[c][m];
                for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
                if (lane == 0) sums[0][m][2 * warp + c] = v;
            }
        __syncthreads();
        if (warp >= ROWS) return;
        finish<float>(a, m0 + warp, n0 + lane, sums[0][warp][lane]);
    }
}

// ---- narrow layers ------------------------------------------------------------------------------------------------------------------
// Up to 32 inputs and 32 outputs: a tile of the tensor cores' kernels costs some 2 us whatever its width, and rows that are no whole 16-byte pieces have to be
// copied for them (1,611,877 x 7 -> 11 fp32 SiLU took 321 us, a sixteenth of it for the bytes, and takes 63; its gradients 154), so these multiply on the CUDA cores, a row a thread, any strides, sums in fp32: K N products a row, for 32 x 32 about as long as the
// bytes take.  Rows travel through shared memory, so that both ways are whole lines whatever the width; the place of an element by a product and a
// shift instead of a division.
constexpr int kThinRows = 128, kThinMost = 32, kThinPitch = 36;      // pitch: rows on 16 bytes, eight of them on all banks

struct Divide {                                   // e / d for e < 4,096 and d <= 32
    uint32_t factor, d;
    __device__ __forceinline__ explicit Divide(int by) : factor(((1u << 20) + by - 1) / by), d(by) {}
    __device__ __forceinline__ int rows(int e) const { return (int)((uint32_t)e * factor >> 20); }
};
// rows x cols elements of a matrix to or from shared memory, by all threads; use(value as fp32, row, column, place in shared memory)
template <class T, class Use> __device__ __forceinline__ void thin_load(const T* p, int64_t ld, int rows, int cols, const Divide& by, Use use)
{
#pragma unroll 4
    for (int e = threadIdx.x; e < rows * cols; e += kThinRows) {
        const int r = by.rows(e), c = e - r * cols;
        use(Pair<T>::one(p[r * ld + c]), r, c, r * kThinPitch + c);
    }
}
template <class T> __device__ __forceinline__ void thin_store(T* p, int64_t ld, int rows, int cols, const Divide& by, const float* from)
{
#pragma unroll 4
    for (int e = threadIdx.x; e < rows * cols; e += kThinRows) {
        const int r = by.rows(e), c = e - r * cols;
        p[r * ld + c] = Pair<T>::round(from[r * kThinPitch + c]);
    }
}
// acc[n] = sum over k < K of row[k] w[k][n], w in rows of kThinMost.
template <int NMAX> __device__ __forceinline__ void thin_product(float* acc, const float* row, const float* w, int K)
{
#pragma unroll
    for (int n = 0; n < NMAX; ++n) acc[n] = 0.f;
    for (int k0 = 0; k0 < K; k0 += 4) {                           // rows are zero up to a multiple of four
        const float4 four = *reinterpret_cast<const float4*>(row + k0);
        const float u[4] = {four.x, four.y, four.z, four.w};
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int n = 0; n < NMAX; n += 4) {
                const float4 v = *reinterpret_cast<const float4*>(w + (k0 + k) * kThinMost + n);
                acc[n] = fmaf(u[k], v.x, acc[n]), acc[n + 1] = fmaf(u[k], v.y, acc[n + 1]);
                acc[n + 2] = fmaf(u[k], v.z, acc[n + 2]), acc[n + 3] = fmaf(u[k], v.w, acc[n + 3]);
            }
    }
}
// w [K x N] as fp32, [k][n] or transposed, zero beyond the matrix.
template <class T> __device__ __forceinline__ void thin_weight(float* to, const T* w, int64_t ldw, bool out_in, int K, int N, bool transposed)
{
    for (int e = threadIdx.x; e < kThinMost * kThinMost; e += kThinRows) {
        const int a = e / kThinMost, b = e % kThinMost, k = transposed ? b : a, n = transposed ? a : b;
        to[e] = k < K && n < N ? Pair<T>::one(out_in ? w[n * ldw + k] : w[k * ldw + n]) : 0.f;
    }
}

template <class T, int ACT, int NMAX>
__global__ void __launch_bounds__(kThinRows) k_thin(const FewArgs a, const int out_in)
{
    __shared__ __align__(16) float w[kThinMost * kThinMost], rows_in[kThinRows * kThinPitch], rows_out[kThinRows * kThinPitch], shift[kThinMost];
    const T *x = static_cast<const T*>(a.x), *r = static_cast<const T*>(a.residual);
    T *y = static_cast<T*>(a.y), *z = static_cast<T*>(a.z);
    const Divide by_k(a.K), by_n(a.N);
    thin_weight(w, static_cast<const T*>(a.w), a.ldw, out_in != 0, a.K, a.N, false);
    if (threadIdx.x < kThinMost) shift[threadIdx.x] = a.bias && threadIdx.x < a.N ? Pair<T>::one(static_cast<const T*>(a.bias)[threadIdx.x]) : 0.f;
    for (int i = threadIdx.x; i < kThinRows * kThinPitch; i += kThinRows) rows_in[i] = 0.f;
    float* const mine = rows_out + threadIdx.x * kThinPitch;
    for (int64_t m0 = (int64_t)blockIdx.x * kThinRows; m0 < a.M; m0 += (int64_t)gridDim.x * kThinRows) {
        const int rows = (int)min((int64_t)kThinRows, a.M - m0);
        __syncthreads();
        thin_load(x + m0 * a.ldx, a.ldx, rows, a.K, by_k, [&](float v, int, int, int at) { rows_in[at] = v; });
        if (r && !z) thin_load(r + m0 * a.ldr, a.ldr, rows, a.N, by_n, [&](float v, int, int, int at) { rows_out[at] = v; });
        __syncthreads();
        float acc[NMAX];
        thin_product<NMAX>(acc, rows_in + threadIdx.x * kThinPitch, w, a.K);
#pragma unroll
        for (int n = 0; n < NMAX; ++n) acc[n] += shift[n];
        if (ACT == DG_ACT_RELU && a.bits && (int)threadIdx.x < rows) {
            uint32_t word = 0;
#pragma unroll
            for (int n = 0; n < NMAX; ++n) word |= (acc[n] <= 0.f ? 0u : 1u) << n;
            a.bits[(m0 + threadIdx.x) * a.ldbits] = word;
        }
        if (z) {                                                  // z and y go out one after the other through the same rows
#pragma unroll
            for (int n = 0; n < NMAX; ++n) mine[n] = acc[n];
            __syncthreads();
            thin_store(z + m0 * a.ldz, a.ldz, rows, a.N, by_n, rows_out);
            __syncthreads();
            if (r) {
                thin_load(r + m0 * a.ldr, a.ldr, rows, a.N, by_n, [&](float v, int, int, int at) { rows_out[at] = v; });
                __syncthreads();
            }
        }
#pragma unroll
        for (int n = 0; n < NMAX; ++n) mine[n] = act_value<ACT>(acc[n]) + (r ? mine[n] : 0.f);
        __syncthreads();
        thin_store(y + m0 * a.ldy, a.ldy, rows, a.N, by_n, rows_out);
    }
}

// All gradients in one pass over x, dy and z: dz goes to shared memory and stays in fp32, a thread makes a row of dx, and every thread of the dw part four by
// four of its elements (a row of ones below x makes db the last row of dw) over a share of the tile's rows, tile after tile; the CTAs' sums are added in order.
struct ThinGradArgs {
    const void *x, *w, *dy, *z;
    const uint32_t* bits;
    void *dx, *dw, *db;
    float* partial;                               // [CTA][(K + 1) N], or null: the one CTA's sums are the result
    int64_t ldx, ldw, lddy, ldz, ldbits, lddx, row_stride, col_stride, M;
    int32_t N, K, out_in;
};

template <class T, int ACT>
__global__ void __launch_bounds__(kThinRows) k_thin_grad(const ThinGradArgs a)
{
    __shared__ __align__(16) float w[kThinMost * kThinMost], xs[kThinRows * kThinPitch], ds[kThinRows * kThinPitch];
    const T *x = static_cast<const T*>(a.x), *dy = static_cast<const T*>(a.dy), *z = static_cast<const T*>(a.z);
    const Divide by_k(a.K), by_n(a.N);
    const bool sums = a.dw || a.db;
    if (a.dx) thin_weight(w, static_cast<const T*>(a.w), a.ldw, a.out_in != 0, a.K, a.N, true);      // [n][k]
    for (int i = threadIdx.x; i < kThinRows * kThinPitch; i += kThinRows) xs[i] = ds[i] = 0.f;
    __syncthreads();
    // x's row of ones (column K); rows beyond the matrix have dz = 0
    xs[threadIdx.x * kThinPitch + a.K] = 1.f;
    const int k_blocks = a.K / 4 + 1, blocks = k_blocks * ((a.N + 3) / 4), groups = kThinRows / blocks;      // 9 x 8 blocks at most
    const int block = threadIdx.x % blocks, group = threadIdx.x / blocks, k0 = block % k_blocks * 4, n0 = block / k_blocks * 4;
    float acc[4][4] = {};
    for (int64_t m0 = (int64_t)blockIdx.x * kThinRows; m0 < a.M; m0 += (int64_t)gridDim.x * kThinRows) {
        const int rows = (int)min((int64_t)kThinRows, a.M - m0);
        __syncthreads();
        if (a.dw) thin_load(x + m0 * a.ldx, a.ldx, rows, a.K, by_k, [&](float v, int, int, int at) { xs[at] = v; });
        thin_load(dy + m0 * a.lddy, a.lddy, rows, a.N, by_n, [&](float v, int row, int c, int at) {
            if constexpr (ACT == DG_ACT_RELU) v = a.bits[(m0 + row) * a.ldbits] >> c & 1 ? v : 0.f;
            else if constexpr (ACT != DG_ACT_NONE) v *= act_slope<ACT>(Pair<T>::one(z[(m0 + row) * a.ldz + c]));
            ds[at] = v;
        });
        if (rows < kThinRows)                                     // a last tile: what the one before left
            for (int e = threadIdx.x + rows * kThinPitch; e < kThinRows * kThinPitch; e += kThinRows) ds[e] = 0.f;
        __syncthreads();
        if (sums && group < groups)
            for (int row = group; row < rows; row += groups) {
                const float4 u = *reinterpret_cast<const float4*>(xs + row * kThinPitch + k0), v = *reinterpret_cast<const float4*>(ds + row * kThinPitch + n0);
                const float p[4] = {u.x, u.y, u.z, u.w}, q[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(p[i], q[j], acc[i][j]);
            }
        if (a.dx) {
            float out[kThinMost];
            if (a.K <= 8) thin_product<8>(out, ds + threadIdx.x * kThinPitch, w, a.N);
            else if (a.K <= 16) thin_product<16>(out, ds + threadIdx.x * kThinPitch, w, a.N);
            else thin_product<32>(out, ds + threadIdx.x * kThinPitch, w, a.N);
            __syncthreads();                                      // dz has been read
#pragma unroll
            for (int k = 0; k < kThinMost; ++k)
                if (k < a.K) ds[threadIdx.x * kThinPitch + k] = out[k];
            __syncthreads();
            thin_store(static_cast<T*>(a.dx) + m0 * a.lddx, a.lddx, rows, a.K, by_k, ds);
            __syncthreads();
            for (int c = a.N; c < a.K; ++c) ds[threadIdx.x * kThinPitch + c] = 0.f;      // dz's padding, which products read as zero
        }
    }
    if (!sums) return;
    __syncthreads();
    float* total = xs;                                            // [group][4 x 4 blocks]: 128 threads x 16 numbers
    if (group < groups)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) total[threadIdx.x * 16 + i * 4 + j] = acc[i][j];
    __syncthreads();
    for (int e = threadIdx.x; e < (a.K + 1) * a.N; e += kThinRows) {
        const int k = by_n.rows(e), n = e - k * a.N, b = n / 4 * k_blocks + k / 4, in = k % 4 * 4 + n % 4;
        float s = 0.f;
        for (int g = 0; g < groups; ++g) s += total[(g * blocks + b) * 16 + in];
        if (a.partial) a.partial[(int64_t)blockIdx.x * (a.K + 1) * a.N + e] = s;
        else if (k == a.K) {
            if (a.db) static_cast<T*>(a.db)[n] = Pair<T>::round(s);
        } else if (a.dw) static_cast<T*>(a.dw)[k * a.row_stride + n * a.col_stride] = Pair<T>::round(s);
    }
}

// 32 elements of dw and db a CTA, 32 warps share the parts.
template <class T> __global__ void __launch_bounds__(1024) k_thin_sums(const ThinGradArgs a, const int parts)
{
    __shared__ double sums[32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e = blockIdx.x * 32 + lane, count = (a.K + 1) * a.N;
    double s = 0.0;
    if (e < count)
#pragma unroll 8
        for (int i = warp; i < parts; i += 32) s += __ldg(a.partial + (int64_t)i * count + e);
    sums[warp][lane] = s;
    __syncthreads();
    if (warp || e >= count) return;
    for (int v = 1; v < 32; ++v) s += sums[v][lane];
    const int k = e / a.N, n = e % a.N;
    if (k == a.K) {
        if (a.db) static_cast<T*>(a.db)[n] = Pair<T>::round((float)s);
    } else if (a.dw) {
        static_cast<T*>(a.dw)[k * a.row_stride + n * a.col_stride] = Pair<T>::round((float)s);
    }
}

// ---- rows of whole 16-byte pieces ------------------------------------------------------------------------------------------------
// A 16-byte piece of the copy a thread, out of the five 32-bit words that its elements lie in (rows start on any even address; the first and last word may
// hold a neighbour's element, which is not used), shifted by half a word where the row starts on one.
__global__ void __launch_bounds__(256) k_pad_rows16(const unsigned short* __restrict__ src, int64_t ld_src, int64_t n, int32_t cols, uint4* __restrict__ dst, int32_t pieces)
{
    const int64_t total = n * pieces, stride = (int64_t)gridDim.x * blockDim.x;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += stride) {
        const int64_t row = i / pieces;
        const int c = (int)(i - row * pieces) * 8, left = cols - c;      // elements of the row from here on
        const unsigned short* s = src + row * ld_src + c;
        const bool odd = reinterpret_cast<uintptr_t>(s) & 2;
        const uint32_t* words = reinterpret_cast<const uint32_t*>(s - odd);
        uint32_t w[5];
#pragma unroll
        for (int e = 0; e < 5; ++e) w[e] = 2 * e - odd < left && (e < 4 || odd) ? __ldcs(words + e) : 0u;
        uint32_t v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[e] = odd ? __funnelshift_r(w[e], w[e + 1], 16) : w[e];
            if (2 * e + 1 >= left) v[e] = 2 * e < left ? v[e] & 0xFFFFu : 0u;
        }
        dst[i] = make_uint4(v[0], v[1], v[2], v[3]);
    }
}

// ---- host side ---------------------------------------------------------------------------------------------------------------------
bool on_rows(const void* p, int64_t ld, int item) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld * item % 16 == 0; }

// [rows x cols] of 16-bit elements, row-major, boxes of 64 columns (128B swizzle; 32: 64B swizzle) x box_rows rows, out-of-range elements read as zero.
int make_map16(CUtensorMap* map, const void* ptr, int32_t type, int64_t rows, int64_t cols, int64_t ld, int box_rows, int box_cols = 64)
{
    EncodeTiledFn fn = encode_tiled();
    if (!fn) return DG_ERR_UNSUPPORTED;
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
    const cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows};
    const cuuint32_t elem[2] = {1, 1};
    const CUresult r = fn(map, type == DG_BFLOAT16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(ptr), dims, strides, box,
                          elem, CU_TENSOR_MAP_INTERLEAVE_NONE, box_cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? DG_OK : DG_ERR_UNSUPPORTED;
}

template <class T, int ACT> int launch_pair(const CUtensorMap* maps, const LinearPairArgs& a, unsigned ctas, size_t smem, cudaStream_t stream)
{
    auto run = [&](auto* kernel, std::atomic<bool>* granted) {
        const int rc = allow_smem((const void*)kernel, granted);
        if (rc) return rc;
        kernel<<<ctas, kThreadsPair, smem, stream>>>(maps[0], maps[1], maps[2], maps[3], maps[4], a);
        return (int)cudaGetLastError();
    };
    static std::atomic<bool> granted[2][64];
    return a.K > kChainTerms<T> ? run(k_linear_pair<T, ACT, true>, granted[0]) : run(k_linear_pair<T, ACT, false>, granted[1]);
}
template <class T> int launch_pair(int act, const CUtensorMap* maps, const LinearPairArgs& a, unsigned ctas, size_t smem, cudaStream_t stream)
{
    switch (act) {
        case DG_ACT_RELU: return launch_pair<T, DG_ACT_RELU>(maps, a, ctas, smem, stream);
        case DG_ACT_GELU: return launch_pair<T, DG_ACT_GELU>(maps, a, ctas, smem, stream);
        case DG_ACT_SILU: return launch_pair<T, DG_ACT_SILU>(maps, a, ctas, smem, stream);
        default: return launch_pair<T, DG_ACT_NONE>(maps, a, ctas, smem, stream);
    }
}

// The columns of a tile: as many as the result has, up to 256, in fewer while that leaves pairs without a tile.
int tile_columns(int64_t m_tiles, int32_t N, int pairs)
{
    if (N <= 64) return (N + 31) / 32 * 32;
    int cols = std::min(256, (N + 63) / 64 * 64);
    while (cols > 64 && m_tiles * ((N + cols - 1) / cols) < pairs) cols -= 64;
    return cols;
}

int linear16(const dg_linear_args* g, cudaStream_t stream)
{
    if (!on_rows(g->x, g->ldx, 2) || !on_rows(g->w, g->ldw, 2) || !on_rows(g->y, g->ldy, 2) || (g->residual && !on_rows(g->residual, g->ldr, 2)) ||
        (g->z && !on_rows(g->z, g->ldz, 2)))
        return DG_ERR_UNSUPPORTED;
    LinearPairArgs a{};
    const int sms = sm_count();
    if (sms < 2) return DG_ERR_STATE;
    a.bias = g->bias, a.bits = g->bits, a.ldbits = g->ldbits, a.M = g->M, a.N = g->N, a.K = g->K;
    const int64_t m_tiles = (g->M + 2 * BM - 1) / (2 * BM);
    a.n_tile = tile_columns(m_tiles, g->N, sms / 2);
    if (g->K > chain_terms(g->type == DG_BFLOAT16)) a.n_tile = std::min(a.n_tile, kEpilogueWarps / 4 * kPiece);
    a.n_panels = (g->N + a.n_tile - 1) / a.n_tile;
    if (m_tiles * a.n_panels >= (int64_t)1 << 30) return DG_ERR_UNSUPPORTED;
    a.tiles = (int)(m_tiles * a.n_panels);
    a.b_boxes = g->out_in ? 0 : (a.n_tile / 2 + 63) / 64;
    a.residual = g->residual != nullptr, a.save_z = g->z != nullptr, a.whole_bias = (reinterpret_cast<uintptr_t>(g->bias) & 15) == 0;
    a.status = dg_status_word();
    if (!a.status) return DG_ERR_STATE;
    CUtensorMap maps[5];
    int rc;
    if ((rc = make_map16(&maps[0], g->x, g->type, g->M, g->K, g->ldx, BM)) ||
        (rc = g->out_in ? make_map16(&maps[1], g->w, g->type, g->N, g->K, g->ldw, a.n_tile / 2) : make_map16(&maps[1], g->w, g->type, g->K, g->N, g->ldw, BK)) ||
        (rc = make_map16(&maps[2], g->y, g->type, g->M, g->N, g->ldy, 32, kPiece)))
        return rc;
    maps[3] = maps[4] = maps[2];
    if (g->residual && (rc = make_map16(&maps[3], g->residual, g->type, g->M, g->N, g->ldr, 32, kPiece))) return rc;
    if (g->z && (rc = make_map16(&maps[4], g->z, g->type, g->M, g->N, g->ldz, 32, kPiece))) return rc;
    const size_t stage = kABytes + (a.b_boxes ? a.b_boxes * BK * 128 : a.n_tile / 2 * 128);
    const size_t rest = (size_t)kEpilogueWarps * (a.save_z ? 3 : 2) * kPieceBytes + kBarBytes + 1024;
    a.stages = (int)std::min<size_t>(kMaxStages, (227 * 1024 - rest) / stage);
    const unsigned ctas = 2u * (unsigned)std::min(a.tiles, sms / 2);
    const size_t smem = a.stages * stage + rest;
    return g->type == DG_BFLOAT16 ? launch_pair<__nv_bfloat16>(g->act, maps, a, ctas, smem, stream) : launch_pair<__half>(g->act, maps, a, ctas, smem, stream);
}

int linear_few(const dg_linear_args* g, cudaStream_t stream)
{
    FewArgs a{g->x, g->w, g->bias, g->residual, g->y, g->z, g->bits, g->ldx, g->ldw, g->ldr, g->ldy, g->ldz, g->ldbits, g->M, g->N, g->K, g->act, 0, 0};
    if (g->type == DG_FLOAT32) {
        auto run = [&](auto out_in, auto rows) {
            constexpr int ROWS = decltype(rows)::value;
            const dim3 grid((unsigned)((g->N + 31) / 32), (unsigned)((g->M + ROWS - 1) / ROWS));
            k_few_rows32<decltype(out_in)::value, ROWS><<<grid, 32 * kFewWarps32, 0, stream>>>(a);
        };
        auto sized = [&](auto out_in) { g->M == 1 ? run(out_in, std::integral_constant<int, 1>{}) : run(out_in, std::integral_constant<int, 4>{}); };
        if (g->out_in) sized(std::true_type{});
        else sized(std::false_type{});
        return (int)cudaGetLastError();
    }
    auto on_8 = [](const void* p, int64_t ld) { return (reinterpret_cast<uintptr_t>(p) & 7) == 0 && ld % 4 == 0; };
    a.whole_x = on_8(g->x, g->ldx), a.whole_w = on_8(g->w, g->ldw);
    const int cols = g->out_in ? kFewCols<true> : kFewCols<false>;
    const dim3 grid((unsigned)((g->N + cols - 1) / cols), (unsigned)((g->M + kFewRows - 1) / kFewRows));
    auto run = [&](auto value) {
        using T = decltype(value);
        if (g->out_in) k_few_rows16<T, true><<<grid, 32 * kFewWarps, 0, stream>>>(a);
        else k_few_rows16<T, false><<<grid, 32 * kFewWarps, 0, stream>>>(a);
    };
    if (g->type == DG_BFLOAT16) run(__nv_bfloat16{});
    else run(__half{});
    return (int)cudaGetLastError();
}

bool aligned(const void* p, int item) { return reinterpret_cast<uintptr_t>(p) % item == 0; }

// Ranges of rows: a CTA for every range and panel, as many as the device has, at least four stages each.
struct DwShape {
    int32_t p_panels, q_panels, p_store, q_store, ranges;
    int64_t rows_per_range, floats;
};
DwShape dw_shape(int64_t M, int32_t N, int32_t K, int32_t type)
{
    DwShape s{};
    s.p_panels = (K + 255) / 256, s.q_panels = (N + 255) / 256;
    s.p_store = (std::min(K, 256) + 15) / 16 * 16, s.q_store = (std::min(N, 256) + 15) / 16 * 16;
    const int64_t panels = (int64_t)s.p_panels * s.q_panels, slabs = (M + kDwRows - 1) / kDwRows;
    const int64_t ranges = std::max<int64_t>(1, std::min<int64_t>(148 / panels, slabs / 4));
    s.rows_per_range = (slabs + ranges - 1) / ranges * kDwRows;
    s.ranges = (int)((M + s.rows_per_range - 1) / s.rows_per_range);
    s.floats = s.ranges > 1 || M > chain_terms(type == DG_BFLOAT16) ? s.ranges * panels * s.p_store * s.q_store : 0;
    return s;
}

}  // namespace

namespace {

bool thin(int32_t N, int32_t K) { return N <= kThinMost && K <= kThinMost; }
unsigned thin_ctas(int64_t M, int each_sm) { return (unsigned)std::min<int64_t>((M + kThinRows - 1) / kThinRows, 148 * each_sm); }

template <class T, class Use> int with_act(int act, Use use)
{
    switch (act) {
        case DG_ACT_RELU: return use(T{}, std::integral_constant<int, DG_ACT_RELU>{});
        case DG_ACT_GELU: return use(T{}, std::integral_constant<int, DG_ACT_GELU>{});
        case DG_ACT_SILU: return use(T{}, std::integral_constant<int, DG_ACT_SILU>{});
        default: return use(T{}, std::integral_constant<int, DG_ACT_NONE>{});
    }
}
template <class Use> int with_type(int type, int act, Use use)
{
    return type == DG_FLOAT32 ? with_act<float>(act, use) : type == DG_BFLOAT16 ? with_act<__nv_bfloat16>(act, use) : with_act<__half>(act, use);
}

int linear_thin(const dg_linear_args* g, cudaStream_t stream)
{
    const FewArgs a{g->x, g->w, g->bias, g->residual, g->y, g->z, g->bits, g->ldx, g->ldw, g->ldr, g->ldy, g->ldz, g->ldbits, g->M, g->N, g->K, g->act, 0, 0};
    const unsigned ctas = thin_ctas(g->M, 5);
    return with_type(g->type, g->act, [&](auto value, auto act) {
        using T = decltype(value);
        constexpr int ACT = decltype(act)::value;
        if (g->N <= 8) k_thin<T, ACT, 8><<<ctas, kThinRows, 0, stream>>>(a, g->out_in);
        else if (g->N <= 16) k_thin<T, ACT, 16><<<ctas, kThinRows, 0, stream>>>(a, g->out_in);
        else k_thin<T, ACT, 32><<<ctas, kThinRows, 0, stream>>>(a, g->out_in);
        return (int)cudaGetLastError();
    });
}

}  // namespace

extern "C" int64_t dg_linear_few(int32_t N, int32_t K, int32_t type) { return thin(N, K) ? ((int64_t)1 << 31) - 1 : type == DG_FLOAT32 ? 16 : 32; }

extern "C" int64_t dg_linear_grad_scratch(int64_t M, int32_t N, int32_t K)
{
    if (M < 1 || N < 1 || K < 1 || !thin(N, K)) return 0;
    const int64_t ctas = thin_ctas(M, 4);
    return ctas > 1 ? ctas * (K + 1) * N : 0;
}

extern "C" int dg_linear_grad(const dg_linear_grad_args* g, void* stream)
{
    if (!g || !g->dy || (!g->dx && !g->dw && !g->db)) return DG_ERR_NULL;
    const int64_t M = g->M;
    const int32_t N = g->N, K = g->K, act = g->act;
    if (M < 1 || M >= (int64_t)1 << 31 || N < 1 || K < 1 || g->type < 0 || g->type > 2 || act < 0 || act > 3) return DG_ERR_DIMS;
    if (!thin(N, K)) return DG_ERR_UNSUPPORTED;
    const bool smooth = act == DG_ACT_GELU || act == DG_ACT_SILU;
    if ((g->dx && !g->w) || (g->dw && !g->x) || (smooth && !g->z) || (act == DG_ACT_RELU && !g->bits)) return DG_ERR_NULL;
    if (g->lddy < N || (g->dx && (g->lddx < K || g->ldw < (g->out_in ? K : N))) || (g->dw && g->ldx < K) || (smooth && g->ldz < N) ||
        (act == DG_ACT_RELU && g->ldbits < 1))
        return DG_ERR_DIMS;
    const int item = g->type == DG_FLOAT32 ? 4 : 2;
    for (const void* p : {g->x, g->w, g->dy, g->z, (const void*)g->dx, (const void*)g->dw, (const void*)g->db})
        if (!aligned(p, item)) return DG_ERR_DIMS;
    const int64_t floats = g->dw || g->db ? dg_linear_grad_scratch(M, N, K) : 0;
    if (floats > 0 && !g->scratch) return DG_ERR_NULL;
    if (g->scratch_floats < floats) return DG_ERR_SCRATCH;
    ThinGradArgs a{g->x, g->w, g->dy, g->z, g->bits, g->dx, g->dw, g->db, floats > 0 ? g->scratch : nullptr, g->ldx, g->ldw, g->lddy, g->ldz, g->ldbits, g->lddx,
                   g->row_stride, g->col_stride, M, N, K, g->out_in};
    cudaStream_t s = (cudaStream_t)stream;
    const unsigned ctas = thin_ctas(M, 4);
    return with_type(g->type, act, [&](auto value, auto activation) {
        using T = decltype(value);
        k_thin_grad<T, decltype(activation)::value><<<ctas, kThinRows, 0, s>>>(a);
        if (a.partial) k_thin_sums<T><<<(unsigned)(((K + 1) * N + 31) / 32), 1024, 0, s>>>(a, (int)ctas);
        return (int)cudaGetLastError();
    });
}

extern "C" int dg_linear(const dg_linear_args* g, void* stream)
{
    if (!g || !g->x || !g->w || !g->y) return DG_ERR_NULL;
    if (g->M < 0 || g->M >= (int64_t)1 << 31 || g->N < 1 || g->K < 1 || g->type < 0 || g->type > 2 || g->act < 0 || g->act > 3) return DG_ERR_DIMS;
    if (g->ldx < g->K || g->ldw < (g->out_in ? g->K : g->N) || g->ldy < g->N || (g->residual && g->ldr < g->N) || (g->z && g->ldz < g->N)) return DG_ERR_DIMS;
    if (g->bits && (g->act != DG_ACT_RELU || g->ldbits % 2 || g->ldbits * 32 < g->N || !aligned(g->bits, 8))) return DG_ERR_DIMS;
    const int item = g->type == DG_FLOAT32 ? 4 : 2;
    if (!aligned(g->x, item) || !aligned(g->w, item) || !aligned(g->y, item) || !aligned(g->bias, item) || !aligned(g->residual, item) || !aligned(g->z, item)) return DG_ERR_DIMS;
    if (g->M == 0) return DG_OK;
    if (thin(g->N, g->K)) return linear_thin(g, (cudaStream_t)stream);
    if (g->M <= dg_linear_few(g->N, g->K, g->type)) return linear_few(g, (cudaStream_t)stream);
    return g->type == DG_FLOAT32 ? dg_dense_linear(g, (cudaStream_t)stream) : linear16(g, (cudaStream_t)stream);
}

extern "C" int64_t dg_linear_dz_scratch(int64_t M, int32_t N) { return M < 1 || N < 1 || dz_ctas(M, N) == 1 ? 0 : (int64_t)dz_ctas(M, N) * N; }

extern "C" int dg_linear_dz(const void* dy, int64_t lddy, const void* z, int64_t ldz, const uint32_t* bits, int64_t ldbits, int32_t act, void* dz, int64_t lddz,
                            void* db, int64_t M, int32_t N, int32_t type, float* scratch, void* stream)
{
    if (!dy || (!dz && !db)) return DG_ERR_NULL;
    if (M < 1 || N < 1 || type < 0 || type > 2 || act < 0 || act > 3 || lddy < N || (dz && lddz < N)) return DG_ERR_DIMS;
    if (act == DG_ACT_RELU ? !bits || ldbits * 32 < N : act != DG_ACT_NONE && (!z || ldz < N)) return DG_ERR_NULL;
    const int item = type == DG_FLOAT32 ? 4 : 2;
    if (!aligned(dy, item) || !aligned(z, item) || !aligned(dz, item) || !aligned(db, item)) return DG_ERR_DIMS;
    LinearDzArgs a{};
    a.lddy = lddy, a.ldz = ldz, a.ldbits = ldbits, a.lddz = lddz, a.M = M, a.N = N, a.bits = bits;
    const bool direct = dg_linear_dz_scratch(M, N) == 0;
    if (db && !direct && !scratch) return DG_ERR_NULL;
    a.partial = db && !direct ? scratch : nullptr, a.db = direct ? db : nullptr;
    a.lanes = dz_lanes(N);
    a.whole_dy = on_rows(dy, lddy, item), a.whole_z = on_rows(z, ldz, item), a.whole_dz = on_rows(dz, lddz, item);
    const dim3 grid((unsigned)dz_ctas(M, N), (unsigned)((N + a.lanes * 8 - 1) / (a.lanes * 8)));
    cudaStream_t s = (cudaStream_t)stream;
    auto run = [&](auto value) {
        using T = decltype(value);
        const T *from = static_cast<const T*>(dy), *pre = static_cast<const T*>(z);
        T* to = static_cast<T*>(dz);
        switch (act) {
            case DG_ACT_RELU: k_linear_dz<T, DG_ACT_RELU><<<grid, kDzThreads, 0, s>>>(from, pre, to, a); break;
            case DG_ACT_GELU: k_linear_dz<T, DG_ACT_GELU><<<grid, kDzThreads, 0, s>>>(from, pre, to, a); break;
            case DG_ACT_SILU: k_linear_dz<T, DG_ACT_SILU><<<grid, kDzThreads, 0, s>>>(from, pre, to, a); break;
            default: k_linear_dz<T, DG_ACT_NONE><<<grid, kDzThreads, 0, s>>>(from, pre, to, a);
        }
        if (a.partial) k_linear_db<T><<<(unsigned)((N + 31) / 32), 1024, 0, s>>>(scratch, (int)grid.x, N, static_cast<T*>(db));
    };
    if (type == DG_FLOAT32) run(float{});
    else if (type == DG_BFLOAT16) run(__nv_bfloat16{});
    else run(__half{});
    return (int)cudaGetLastError();
}

extern "C" int64_t dg_linear_dw_scratch(int64_t M, int32_t N, int32_t K, int32_t type)
{
    if (M < 1 || N < 1 || K < 1) return 0;
    if (type == DG_FLOAT32) return dg_dense_linear_dw_scratch(N, K);
    const DwShape shape = dw_shape(M, N, K, type);
    return shape.floats ? shape.floats + (int64_t)shape.ranges * N : 0;
}

extern "C" int dg_linear_dw(const dg_linear_dw_args* g, void* stream)
{
    if (!g || !g->x || !g->dy || !g->dw) return DG_ERR_NULL;
    const int64_t M = g->M;
    const int32_t N = g->N, K = g->K, type = g->type, act = g->act;
    if (M < 1 || M >= (int64_t)1 << 31 || N < 1 || K < 1 || g->ldx < K || g->lddy < N || type < 0 || type > 2 || act < 0 || act > 3) return DG_ERR_DIMS;
    const bool smooth = act == DG_ACT_GELU || act == DG_ACT_SILU, fused = act != DG_ACT_NONE || g->db;
    if ((smooth && !g->z) || (act == DG_ACT_RELU && !g->bits)) return DG_ERR_NULL;
    if ((smooth && g->ldz < N) || (act == DG_ACT_RELU && g->ldbits * 32 < N) || (g->dz && (act == DG_ACT_NONE || g->lddz < N))) return DG_ERR_DIMS;
    const int item = type == DG_FLOAT32 ? 4 : 2;
    if (!aligned(g->dw, item) || !aligned(g->db, item) || !aligned(g->scratch, 16)) return DG_ERR_DIMS;
    if (type == DG_FLOAT32) return fused ? DG_ERR_UNSUPPORTED : dg_dense_linear_dw(g, (cudaStream_t)stream);
    if (!on_rows(g->x, g->ldx, 2) || !on_rows(g->dy, g->lddy, 2) || (smooth && !on_rows(g->z, g->ldz, 2)) || (g->dz && !on_rows(g->dz, g->lddz, 2)) || (fused && K > 256))
        return DG_ERR_UNSUPPORTED;
    const DwShape shape = dw_shape(M, N, K, type);
    const int64_t floats = dg_linear_dw_scratch(M, N, K, type);
    if (floats > 0 && !g->scratch) return DG_ERR_NULL;
    if (g->scratch_floats < floats) return DG_ERR_SCRATCH;
    LinearDwArgs a{};
    a.partial = floats > 0 ? reinterpret_cast<float4*>(g->scratch) : nullptr;
    a.dw = g->dw, a.row_stride = g->row_stride, a.col_stride = g->col_stride;
    a.M = M, a.rows_per_range = shape.rows_per_range, a.p_cols = K, a.q_cols = N;
    a.p_panels = shape.p_panels, a.q_panels = shape.q_panels, a.p_store = shape.p_store, a.q_store = shape.q_store;
    a.p_boxes = (std::min(K, 256) + 63) / 64, a.q_boxes = (std::min(N, 256) + 63) / 64;
    if (K > 64) a.p_boxes = (a.p_boxes + 1) / 2 * 2;              // an MMA reads 128 columns; what lies beyond x's reaches rows that are not stored
    a.bits = g->bits, a.ldbits = g->ldbits, a.db = g->db, a.db_partial = floats > 0 ? g->scratch + shape.floats : nullptr, a.store = g->dz != nullptr;
    a.status = dg_status_word();
    if (!a.status) return DG_ERR_STATE;
    CUtensorMap maps[4];
    int rc;
    const int rows = fused ? kBackRows : kDwRows;
    if ((rc = make_map16(&maps[0], g->x, type, M, K, g->ldx, rows)) || (rc = make_map16(&maps[1], g->dy, type, M, N, g->lddy, rows))) return rc;
    maps[2] = maps[3] = maps[1];
    if (smooth && (rc = make_map16(&maps[2], g->z, type, M, N, g->ldz, rows))) return rc;
    if (g->dz && (rc = make_map16(&maps[3], g->dz, type, M, N, g->lddz, rows))) return rc;
    const unsigned ctas = (unsigned)(shape.ranges * shape.p_panels * shape.q_panels);
    const int64_t slots = (int64_t)shape.p_panels * shape.q_panels * (shape.p_store * shape.q_store / 4);
    cudaStream_t s = (cudaStream_t)stream;
    auto product = [&](auto value) {
        using T = decltype(value);
        const size_t stage = (size_t)(a.p_boxes + a.q_boxes) * kDwBox;
        a.stages = (int)std::min<size_t>(kDwMaxStages, (227 * 1024 - kDwBarBytes - 1024) / stage);
        static std::atomic<bool> granted[64];
        const int code = allow_smem((const void*)k_linear_dw<T>, granted);
        if (code) return code;
        k_linear_dw<T><<<ctas, kDwThreads, a.stages * stage + kDwBarBytes + 1024, s>>>(maps[0], maps[1], a);
        return (int)cudaGetLastError();
    };
    auto product_with = [&](auto value, auto activation) {
        using T = decltype(value);
        constexpr int ACT = decltype(activation)::value;
        const size_t stage = (size_t)(a.p_boxes + (smooth ? 2 : 1) * a.q_boxes) * kBackBox, rest = kBackSumBytes + kBackBarBytes + 1024;
        a.stages = (int)std::min<size_t>(kBackMaxStages, (227 * 1024 - rest) / stage);
        static std::atomic<bool> granted[64];
        const int code = allow_smem((const void*)k_linear_back<T, ACT>, granted);
        if (code) return code;
        k_linear_back<T, ACT><<<ctas, kBackThreads, a.stages * stage + rest, s>>>(maps[0], maps[1], maps[2], maps[3], a);
        return (int)cudaGetLastError();
    };
    auto run = [&](auto value) {
        using T = decltype(value);
        const int code = !fused                  ? product(value)
                         : act == DG_ACT_RELU    ? product_with(value, std::integral_constant<int, DG_ACT_RELU>{})
                         : act == DG_ACT_GELU    ? product_with(value, std::integral_constant<int, DG_ACT_GELU>{})
                         : act == DG_ACT_SILU    ? product_with(value, std::integral_constant<int, DG_ACT_SILU>{})
                                                 : product_with(value, std::integral_constant<int, DG_ACT_NONE>{});
        if (code || !a.partial) return code;
        k_linear_dw_reduce<T><<<(unsigned)((slots + 31) / 32), 256, 0, s>>>(a.partial, shape.ranges, a.p_panels, a.q_panels, a.p_store, a.q_store, K, N, static_cast<T*>(g->dw),
                                                                        g->row_stride, g->col_stride);
        if (g->db) k_linear_db<T><<<(unsigned)((N + 31) / 32), 1024, 0, s>>>(a.db_partial, shape.ranges, N, static_cast<T*>(g->db));
        return (int)cudaGetLastError();
    };
    return type == DG_BFLOAT16 ? run(__nv_bfloat16{}) : run(__half{});
}

extern "C" int dg_pad_rows16(const void* src, int64_t ld_src, int64_t n, int32_t cols, void* dst, int64_t ld_dst, void* stream)
{
    if (n < 0 || cols < 0 || ld_src < cols || ld_dst < cols || ld_dst % 8 || ld_dst >= ((int64_t)1 << 31)) return DG_ERR_DIMS;
    if (n == 0 || ld_dst == 0) return DG_OK;
    if (!src || !dst) return DG_ERR_NULL;
    if (!aligned(src, 2) || !aligned(dst, 16)) return DG_ERR_DIMS;
    const int64_t blocks = (n * (ld_dst / 8) + 255) / 256;
    k_pad_rows16<<<(unsigned)std::min<int64_t>(blocks, 148 * 32), 256, 0, (cudaStream_t)stream>>>(static_cast<const unsigned short*>(src), ld_src, n, cols,
                                                                                                static_cast<uint4*>(dst), (int32_t)(ld_dst / 8));
    return (int)cudaGetLastError();
}
