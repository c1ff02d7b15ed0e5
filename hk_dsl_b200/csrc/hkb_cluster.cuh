// Thread-block clusters: rank, barrier, a peer's shared memory, and the launch.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <initializer_list>

#include "../../include/hkb.h"

extern thread_local int hkb_tls_cuda_error;

namespace hkb {

__device__ __forceinline__ int cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return (int)r;
}
__device__ __forceinline__ int cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return (int)r;
}
// Every thread of every CTA of the cluster; what was written before it (shared or global) is seen behind it.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
// The address, in CTA `rank` of the cluster, of what lies at `addr` in this CTA's shared memory.
__device__ __forceinline__ uint32_t peer_smem(uint32_t addr, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float4 peer_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ float peer_f1(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}

// Whether 64-bit arguments are all ints.
inline bool ints(std::initializer_list<int64_t> values) {
  for (int64_t v : values)
    if (v < -0x80000000LL || v > 0x7fffffffLL) return false;
  return true;
}

// One argument struct, `cluster` CTAs of grid.x a cluster (1: an ordinary launch; past 8, the portable size,
// the kernel has to be allowed to).
inline int launch_cluster(const void* kernel, dim3 grid, int threads, int cluster, int smem_bytes, const void* args, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem_bytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 1 : 0;
  void* params[1] = {const_cast<void*>(args)};
  cudaError_t e = cudaLaunchKernelExC(&cfg, kernel, params);
  if (e == cudaSuccess) e = cudaGetLastError();
  else (void)cudaGetLastError();
  if (e != cudaSuccess) { hkb_tls_cuda_error = (int)e; return HKB_ERR_CUDA; }
  return HKB_OK;
}

}  // namespace hkb
