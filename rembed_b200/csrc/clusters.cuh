// clusters.cuh - how many thread-block clusters of a kernel run at once.
#pragma once

#include <cuda_runtime.h>

namespace rg {

// Clusters of `size` (a power of two up to 8) CTAs of a kernel that can run at
// once on the current device; GPCs differ in their SMs, so it is asked for.
// Allows the kernel its shared memory first.  `known` is this kernel's own.
struct ClusterCounts {
    int of[32][4];
};
template <class Kernel>
cudaError_t clusters_at_once(Kernel kern, int threads, int smem, int size, ClusterCounts& known, int& count) {
    int dev = 0, log2 = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    while (1 << log2 < size) ++log2;
    count = dev < 32 ? __atomic_load_n(&known.of[dev][log2], __ATOMIC_ACQUIRE) : 0;
    if (count > 0) return cudaSuccess;
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(size);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = size;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    e = cudaOccupancyMaxActiveClusters(&count, kern, &cfg);
    if (e != cudaSuccess) return e;
    if (dev < 32) __atomic_store_n(&known.of[dev][log2], count, __ATOMIC_RELEASE);
    return cudaSuccess;
}

}  // namespace rg
