// prima.cpp_b200/csrc/cluster.cuh — a cluster's CTAs: their places, their barrier, reads of each other's shared memory.
#pragma once
#include <algorithm>

#include "common.cuh"

namespace pb {

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
// all threads of all CTAs: what was written in front of it is seen behind it
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t remote_addr(const void * at, uint32_t cta) {
    uint32_t ra;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"(smem_u32(at)), "r"(cta));
    return ra;
}
__device__ __forceinline__ double remote(const double * at, uint32_t cta) {
    double v;
    asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(remote_addr(at, cta)) : "memory");
    return v;
}
__device__ __forceinline__ float remote(const float * at, uint32_t cta) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote_addr(at, cta)) : "memory");
    return v;
}
__device__ __forceinline__ int remote(const int * at, uint32_t cta) {
    int v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(remote_addr(at, cta)) : "memory");
    return v;
}

// clusters of 1, 2, 4 or 8 CTAs that run at the same time where a CTA takes an SM: a cluster stays within a group of SMs.  What cudaOccupancyMaxActiveClusters says on a B200 with 148 SMs, 8 from
// below; persistent kernels launch no more, since the rest of a grid would start where these have ended
inline int clusters_at_once(int ctas, int sms) { return std::max(1, (ctas >= 8 ? 15 : ctas >= 4 ? 33 : ctas >= 2 ? 74 : 148) * sms / 148); }
// kernel of n clusters of so many CTAs; dependent: it may start while the kernel in front of it ends, and waits for that itself
template <typename K, typename... A>
cudaError_t launch_clusters(K * kernel, int64_t n, int ctas, int threads, size_t smem, bool dependent, cudaStream_t st, const A &... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned) (n * ctas)); cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = smem; cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned) ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = dependent ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace pb
