// Thread-block cluster helpers: rank, barrier and reads of a peer CTA's shared
// memory (distributed shared memory), plus the host side of a cluster launch.
#pragma once

#include <atomic>

#include "qia_common.cuh"

namespace qia {

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

// All threads of all CTAs of the cluster; orders shared-memory accesses.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}

// The two halves of cluster_sync: a CTA may store into a peer's shared memory
// once every CTA of the cluster has started, which a wait after an early arrive
// establishes cheaply.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }

// shared::cluster address of `p` (in this CTA's shared memory) in CTA `rank`.
__device__ __forceinline__ uint32_t cluster_map(const void* p, uint32_t rank) {
  uint32_t out;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
               : "=r"(out)
               : "r"(uint32_t(__cvta_generic_to_shared(p))), "r"(rank));
  return out;
}

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

__device__ __forceinline__ void st_cluster_f32x2(uint32_t addr, float a, float b) {
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(addr), "f"(a), "f"(b) : "memory");
}

// Clusters of `size` CTAs of a kernel that the device holds at once (a cluster
// stays within a GPU processing cluster, so this can be less than slots / size);
// 0 where that size cannot run. `cached`: seventeen zeros of static storage.
template <class... KArgs>
int resident_clusters(void (*kernel)(KArgs...), int threads, int smem, int size, std::atomic<int>* cached) {
  int n = cached[size].load(std::memory_order_relaxed);
  if (n == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(size));
    cfg.blockDim = dim3(unsigned(threads));
    cfg.dynamicSmemBytes = size_t(smem);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = unsigned(size);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n <= 0) {
      cudaGetLastError();
      n = -1;
    }
    cached[size].store(n, std::memory_order_relaxed);   // (every thread finds the same)
  }
  return n > 0 ? n : 0;
}

// Lets `kernel` use `smem` bytes of dynamic shared memory (and clusters of more
// than eight CTAs) on the current device, once per device: `done` is static
// storage, one bit per device.
template <class... KArgs>
int allow_launch(const char* what, void (*kernel)(KArgs...), int smem, std::atomic<uint64_t>* done, bool big_clusters = false) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return set_error(QIA_ERR_CUDA, "%s: no device", what);
  const uint64_t bit = uint64_t(1) << dev;
  if (done->load(std::memory_order_acquire) & bit) return QIA_OK;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess && big_clusters) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(QIA_ERR_CUDA, "%s: cudaFuncSetAttribute: %s", what, cudaGetErrorString(e));
  }
  done->fetch_or(bit, std::memory_order_release);
  return QIA_OK;
}

// Launches `kernel` with clusters of `cluster` CTAs along x (grid.x a multiple
// of it).
template <class... KArgs, class... Args>
int launch_cluster(const char* what, void (*kernel)(KArgs...), dim3 grid, int threads, size_t smem, int cluster,
                   cudaStream_t st, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(unsigned(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(cluster);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, KArgs(args)...);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(QIA_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
  }
  count_launch();
  return QIA_OK;
}

}  // namespace qia
