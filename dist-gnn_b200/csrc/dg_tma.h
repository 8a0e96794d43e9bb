// What the kernels that are fed by TMA share on both sides: loads, operand descriptors, tensor maps and launch limits.
#pragma once
#include <cuda.h>
#include <atomic>
#include <cstdint>
#include "dg_internal.h"
#include "dg_umma.h"

namespace dg {

__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t bar)
{
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                 ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1) : "memory");
}
// A load into this CTA whose arrival is counted at a barrier of the pair's even CTA (cta_group::2).
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t cluster_bar)
{
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                 ::"r"(dst), "l"(map), "r"(cluster_bar), "r"(c0), "r"(c1) : "memory");
}
// Shared-memory matrix descriptor of a K-major tile stored as 128-byte rows with the 128B swizzle: 8-row groups are
// 1024 bytes apart (stride byte offset), the leading byte offset is unused for this layout, descriptor version 1.
__device__ __forceinline__ uint64_t umma_desc_sw128(uint32_t smem_addr)
{
    uint64_t d = 0;
    d |= (uint64_t)((smem_addr & 0x3FFFF) >> 4);            // start address, 16-byte units
    d |= (uint64_t)1 << 16;                                   // leading byte offset (ignored with swizzle), 16-byte units
    d |= (uint64_t)(1024 >> 4) << 32;                         // stride byte offset between 8-row groups
    d |= (uint64_t)1 << 46;                                   // descriptor version for sm_100
    d |= (uint64_t)2 << 61;                                   // layout type: SWIZZLE_128B
    return d;
}

// Raises a kernel's dynamic shared-memory limit to the most a CTA can have, once per device instead of before every launch.
inline int allow_smem(const void* kernel, std::atomic<bool>* done)
{
    int dev = 0;
    DG_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64) return DG_ERR_STATE;
    if (done[dev].load(std::memory_order_relaxed)) return DG_OK;
    DG_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
    done[dev].store(true, std::memory_order_relaxed);
    return DG_OK;
}

inline int sm_count()
{
    static std::atomic<int> count[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
    int n = count[dev].load(std::memory_order_relaxed);
    if (n == 0) {
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
        count[dev].store(n, std::memory_order_relaxed);
    }
    return n;
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The driver's call wants a current context, which a thread that has not used the runtime yet - autograd's, whose first call may be one of these - has not.
inline EncodeTiledFn encode_tiled()
{
    static thread_local bool bound = false;
    int dev = 0;
    if (!bound) bound = cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess;
    static EncodeTiledFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeTiledFn>(p);
    }();
    return fn;
}

}  // namespace dg
