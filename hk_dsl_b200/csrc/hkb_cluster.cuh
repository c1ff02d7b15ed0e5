// Thread-block clusters (rank, barrier, a peer's shared memory), launches that follow closely on one another.
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

// Whether a softmax scale is positive and, in fp32 and times log2 e, neither subnormal nor infinite: at 0 a masked logit,
// -inf, is no number, and at infinity a logit of 0.
inline bool positive_scale(double scale) { return scale >= 0x1p-126 && scale <= 0x1p126; }

// The calls of a decode step are short kernels that each read what the one before wrote. They are launched with
// programmatic stream serialisation: a kernel's CTAs may take their places while the kernel before still runs. Every
// kernel launched so begins with `after_the_last`, which waits until everything before it is complete and its writes are
// seen (nothing is read or written in front of it), and calls `let_the_next` where the next one's CTAs may come in.
__device__ __forceinline__ void after_the_last() { asm volatile("griddepcontrol.wait;\n" ::: "memory"); }
__device__ __forceinline__ void let_the_next() { asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory"); }

// The percentage of an SM's memory that is shared memory. One split for a step's kernels: an SM that changes it empties
// first, so a step that alternated kernels with and without rings lost the head start (2 requests x 131072 tokens, 256
// pages: 41.2 against 36.2 us a step).
constexpr int STEP_CARVEOUT = 100;

// More than 48 KB of dynamic shared memory, or a cluster past the portable size, is asked for once a device.
template <class K>
inline cudaError_t arm(K kernel, cudaFuncAttribute attribute, int value, bool (&armed)[64]) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && dev >= 0 && dev < 64 && !armed[dev]) {
    e = cudaFuncSetAttribute(kernel, attribute, value);
    if (e == cudaSuccess) armed[dev] = true;
  }
  if (e != cudaSuccess) { (void)cudaGetLastError(); hkb_tls_cuda_error = (int)e; }
  return e;
}

// One argument struct; `cluster` CTAs of grid.x a cluster (1: none; past 8, the portable size, the kernel has to be
// allowed to).
inline int launch(const void* kernel, dim3 grid, int threads, int cluster, int smem_bytes, const void* args, cudaStream_t st, int carveout = STEP_CARVEOUT) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem_bytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[3];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributePreferredSharedMemoryCarveout;
  attr[1].val.sharedMemCarveout = carveout;
  attr[2].id = cudaLaunchAttributeClusterDimension;
  attr[2].val.clusterDim.x = cluster;
  attr[2].val.clusterDim.y = attr[2].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 3 : 2;
  void* params[1] = {const_cast<void*>(args)};
  cudaError_t e = cudaLaunchKernelExC(&cfg, kernel, params);
  if (e == cudaSuccess) e = cudaGetLastError();
  else (void)cudaGetLastError();
  if (e != cudaSuccess) { hkb_tls_cuda_error = (int)e; return HKB_ERR_CUDA; }
  return HKB_OK;
}

}  // namespace hkb
