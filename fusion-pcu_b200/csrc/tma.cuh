// tma.cuh -- mbarriers, TMA tile loads and the tensor-map encoder, shared by the matrix products.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>

#include <mutex>

#include "common.cuh"
#include "pcu_b200.h"

namespace pcu {

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void mbar_init(uint64_t *bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(bar)), "r"(count) : "memory");
}

__device__ __forceinline__ void mbar_expect_tx(uint64_t *bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(bar)), "r"(bytes)
                 : "memory");
}

__device__ __forceinline__ void mbar_arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}

__device__ __forceinline__ bool mbar_try_wait(uint64_t *bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(smem_addr(bar)), "r"(parity)
        : "memory");
    return done != 0;
}

// The same for barriers at which other CTAs of the cluster arrive without handing memory over:
// relaxed, since an acquire at cluster scope drops the SM's cached lines.
__device__ __forceinline__ bool mbar_try_wait_cluster(uint64_t *bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.relaxed.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(smem_addr(bar)), "r"(parity)
        : "memory");
    return done != 0;
}

// Bounded wait: false after kWaitLimitNs (the caller reports kWatchdog).
template <typename Try> __device__ __forceinline__ bool bounded_wait(Try attempt) {
    if (attempt()) return true;
    const unsigned long long t0 = global_ns();
    for (;;) {
#pragma unroll 1
        for (int i = 0; i < 64; ++i)
            if (attempt()) return true;
        if (global_ns() - t0 > kWaitLimitNs) return false;
    }
}

__device__ __forceinline__ bool mbar_wait(uint64_t *bar, uint32_t parity) {
    return bounded_wait([&] { return mbar_try_wait(bar, parity); });
}

// For memory that another CTA of the cluster hands over with a release at cluster scope.
__device__ __forceinline__ bool mbar_acquire_cluster(uint64_t *bar, uint32_t parity) {
    const bool ok = bounded_wait([&] { return mbar_try_wait_cluster(bar, parity); });
    asm volatile("fence.acq_rel.cluster;" ::: "memory");
    return ok;
}

__device__ __forceinline__ bool mbar_wait_cluster(uint64_t *bar, uint32_t parity) {
    return bounded_wait([&] { return mbar_try_wait_cluster(bar, parity); });
}

__device__ __forceinline__ void tma_load_2d(void *dst, const CUtensorMap *map, uint64_t *bar, int x, int y) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::
            "r"(smem_addr(dst)),
        "l"(map), "r"(smem_addr(bar)), "r"(x), "r"(y)
        : "memory");
}

// ---- thread block clusters
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

__device__ __forceinline__ uint32_t cluster_address(uint32_t address, uint32_t rank) {
    uint32_t remote;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(address), "r"(rank));
    return remote;
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}

// A value of another CTA of the cluster at this CTA's shared address `address`.
__device__ __forceinline__ void cluster_read(float &v, uint32_t address, uint32_t rank) {
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_address(address, rank)) : "memory");
}
__device__ __forceinline__ void cluster_read(double &v, uint32_t address, uint32_t rank) {
    asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(cluster_address(address, rank)) : "memory");
}

}  // namespace pcu

namespace pcu_host {

// Once per device: the dynamic shared memory that a kernel may ask for, and whether it is launched
// with the registers a thread that its warps share out.
template <auto kernel> int allow_shared(int bytes, int registers = 0) {
    static std::mutex lock;
    static bool configured[64] = {false};
    int device = 0;
    if (cudaError_t e = cudaGetDevice(&device); e != cudaSuccess) return set_cuda_error(e);
    std::lock_guard<std::mutex> guard(lock);
    if (device < 64 && configured[device]) return PCU_B200_OK;
    cudaFuncAttributes attributes;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) e = cudaFuncGetAttributes(&attributes, kernel);
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        return set_cuda_error(e);
    }
    if (attributes.numRegs < registers) return PCU_B200_ERROR_UNSUPPORTED;
    if (device < 64) configured[device] = true;
    return PCU_B200_OK;
}

// A launch of a kernel that begins with in_stream_order(), in clusters of `ranks` CTAs along x (0: as the
// kernel says).
template <typename... Params, typename... Args>
int launch_cluster(void (*kernel)(Params...), unsigned grid, unsigned block, size_t shared, unsigned ranks,
                   cudaStream_t stream, const Args &...args) {
    cudaLaunchConfig_t config{};
    config.gridDim = grid;
    config.blockDim = block;
    config.dynamicSmemBytes = shared;
    config.stream = stream;
    cudaLaunchAttribute attributes[2]{};
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = 1;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim.x = ranks;
    attributes[1].val.clusterDim.y = attributes[1].val.clusterDim.z = 1;
    config.attrs = attributes;
    config.numAttrs = ranks ? 2 : 1;
    if (cudaError_t e = cudaLaunchKernelEx(&config, kernel, args...); e != cudaSuccess) {
        (void)cudaGetLastError();
        return set_cuda_error(e);
    }
    return PCU_B200_OK;
}

template <typename... Params, typename... Args>
int launch_grid(void (*kernel)(Params...), unsigned grid, unsigned block, cudaStream_t stream, const Args &...args) {
    return launch_cluster(kernel, grid, block, 0, 0, stream, args...);
}

inline PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
    static std::once_flag once;
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    std::call_once(once, [] {
        void *ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
    });
    return fn;
}

}  // namespace pcu_host
