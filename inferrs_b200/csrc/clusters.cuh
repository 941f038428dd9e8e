// Clusters of CTAs: their barrier, a look into another CTA's shared memory, and how many of them run at once.
#pragma once
#include "common.cuh"

constexpr int IB_MAX_CLUSTER = 8;

__device__ __forceinline__ void ib_cluster_sync() {
    __syncwarp();      // (the threads of a warp arrive as one)
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// where the CTA of that rank has what this one has at `local`
__device__ __forceinline__ unsigned ib_cluster_address(const void* local, unsigned rank) {
    unsigned a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((unsigned)__cvta_generic_to_shared(local)), "r"(rank));
    return a;
}
__device__ __forceinline__ float ib_cluster_f32(const float* local, unsigned rank) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(ib_cluster_address(local, rank)));
    return v;
}

struct IbClusters { std::atomic<int> known[64][IB_MAX_CLUSTER + 1] = {}; };      // by device and size; 0: not asked yet

// A cluster lies in one of the machine's groups of SMs, so that more clusters than this take a second turn although SMs are free (groups of 16 and
// 18 SMs: of clusters of 1 to 8 CTAs that each fill an SM 148, 74, 45, 33, 26, 22, 15, 15).  Asked for once on every device; 0: it cannot be told.
template <typename Kernel>
static inline int ib_clusters_at_once(IbClusters& clusters, Kernel kernel, int size, int threads, size_t smem) {
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
    n = clusters.known[dev][size].load(std::memory_order_relaxed);
    if (n > 0) return n;
    cudaLaunchConfig_t cfg = {};
    cfg.dynamicSmemBytes = smem;
    cfg.gridDim = dim3((unsigned)size);
    cfg.blockDim = dim3((unsigned)threads);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = size;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
        cudaGetLastError();           // (not a fault of the call)
        return 0;
    }
    clusters.known[dev][size].store(n, std::memory_order_relaxed);
    return n;
}
