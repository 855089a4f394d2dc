// cluster.cuh -- blocks of a cluster exchanging through one another's shared memory.
#pragma once

#include "common.cuh"

namespace tp {

namespace {

typedef unsigned long long u64;

constexpr int MAX_CLUSTER = 8;

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// A block may touch another one's shared memory only once that one runs: a kernel arrives at its
// beginning and waits before its first access (all its threads, in this order).
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t remote(const void* p, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(tp_smem_addr(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void remote_store(uint32_t at, u64 v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(at), "l"(v) : "memory");
}
__device__ __forceinline__ void remote_store(uint32_t at, int v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(v) : "memory");
}
__device__ __forceinline__ uint32_t remote_load(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ int remote_add(uint32_t at, int v) {
  int old;
  asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(old) : "r"(at), "r"(v) : "memory");
  return old;
}

// Launches `kernel` with `cluster` blocks to a cluster (a block by itself is one).
template <typename... P, typename... A>
int launch_clusters(void (*kernel)(P...), int64_t blocks, int threads, int cluster, cudaStream_t stream,
                    A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.stream = stream;
  cudaLaunchAttribute together;
  together.id = cudaLaunchAttributeClusterDimension;
  together.val.clusterDim.x = (unsigned)cluster;
  together.val.clusterDim.y = 1;
  together.val.clusterDim.z = 1;
  cfg.attrs = &together;
  cfg.numAttrs = cluster > 1 ? 1 : 0;
  return cuda_status(cudaLaunchKernelEx(&cfg, kernel, args...));
}

}  // namespace

}  // namespace tp
