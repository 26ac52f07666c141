// Thread-block clusters: the other CTAs' shared memory.
#pragma once

#include "common.cuh"

namespace ts {

__device__ __forceinline__ uint32_t cluster_rank_of() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size_of() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
// All threads of all CTAs of the cluster; what they wrote to shared memory before is visible after.
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The value at `p` (in this CTA's shared memory) of the CTA of that rank.
template <class T>
__device__ __forceinline__ T cluster_read(const T* p, uint32_t rank) {
  static_assert(sizeof(T) == 4 || sizeof(T) == 8, "32 or 64 bits");
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
  T v;
  if constexpr (sizeof(T) == 4) {
    uint32_t r;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(r) : "r"(at) : "memory");
    memcpy(&v, &r, 4);
  } else {
    unsigned long long r;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(r) : "r"(at) : "memory");
    memcpy(&v, &r, 8);
  }
  return v;
}

// Launch with a cluster of `size` CTAs along x (grid.x a multiple of it).
template <class... Params, class... Args>
cudaError_t launch_cluster(void (*kernel)(Params...), dim3 grid, int threads, size_t smem, cudaStream_t s, int size,
                           const Args&... args) {
  cudaLaunchConfig_t config = {};
  config.gridDim = grid;
  config.blockDim = dim3(static_cast<unsigned>(threads));
  config.dynamicSmemBytes = smem;
  config.stream = s;
  cudaLaunchAttribute attr[1] = {};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(size);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  config.attrs = attr;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, kernel, args...);
}

}  // namespace ts
