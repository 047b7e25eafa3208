// Thread-block clusters on sm_100a: ranks, the hardware barrier over a cluster,
// reads of another CTA's shared memory, and a launch helper.
#pragma once

#include "common.cuh"

namespace strix {
namespace cluster {

__device__ __forceinline__ uint32_t rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

// All threads of all CTAs of the cluster meet here; shared-memory writes before it
// are visible to the whole cluster after it.
__device__ __forceinline__ void sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Address, in the cluster's shared window, of `smem_addr` of CTA `cta`.
__device__ __forceinline__ uint32_t map_shared(uint32_t smem_addr, uint32_t cta) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr), "r"(cta));
  return r;
}

__device__ __forceinline__ float ld_shared_f32(uint32_t cluster_addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_addr) : "memory");
  return v;
}

__device__ __forceinline__ float4 ld_shared_f32x4(uint32_t cluster_addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(cluster_addr)
               : "memory");
  return v;
}

// A launch of `grid` CTAs in clusters of `size` along x (1: none), chained to the
// kernel before it like launch_chain (common.cuh).
template <typename... P, typename... A>
inline cudaError_t launch(void (*kernel)(P...), unsigned grid, unsigned size, unsigned block, size_t smem,
                          cudaStream_t st, A&&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid), cfg.blockDim = dim3(block), cfg.dynamicSmemBytes = smem, cfg.stream = st;
  cudaLaunchAttribute attr[2] = {};
  int n = 0;
  if (size > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = size, attr[n].val.clusterDim.y = 1, attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr, cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kernel, P(static_cast<A&&>(args))...);
}

// How many clusters of `size` CTAs the current device runs at once, at one CTA per SM. Two
// threads may fill one table of answers at the same time: *out is written once, with the answer.
template <typename... P>
inline cudaError_t places(int* out, void (*kernel)(P...), unsigned size, unsigned block, size_t smem) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(size * 64), cfg.blockDim = dim3(block), cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = size, attr.val.clusterDim.y = 1, attr.val.clusterDim.z = 1;
  cfg.attrs = &attr, cfg.numAttrs = 1;
  int n = 0;
  const cudaError_t err = cudaOccupancyMaxActiveClusters(&n, kernel, &cfg);
  if (err == cudaSuccess) *out = n;
  return err;
}

}  // namespace cluster
}  // namespace strix
