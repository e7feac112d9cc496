// dq_launch.h -- launches and launch set-up that the host sides share.
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "../../include/dq_linear.h"

namespace dq {

inline bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline size_t up256(size_t v) { return (v + 255) & ~static_cast<size_t>(255); }

// after: programmatic stream serialization -- the kernel may start while the
// one before it drains, and waits (griddepcontrol.wait) before it reads that
// one's results.  cluster: CTAs of a cluster along (x, y).
template <typename... Params, typename... Args>
int launch(void (*kern)(Params...), dim3 grid, int threads, size_t smem, cudaStream_t st, bool after, dim3 cluster,
           const Args&... args) {
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (after) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster.x * cluster.y > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = cluster.x;
    attr[n].val.clusterDim.y = cluster.y;
    attr[n++].val.clusterDim.z = 1;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kern, args...) == cudaSuccess ? DQ_OK : DQ_ERR_LAUNCH;
}

// Shared-memory opt-in of a kernel, once per device.
constexpr int kMaxDevices = 64;
template <typename K>
int allow_smem(K kern, int bytes, std::atomic<int>* set) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return DQ_ERR_CUDA;
  if (set[dev].load(std::memory_order_acquire)) return DQ_OK;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
    return DQ_ERR_LAUNCH;
  set[dev].store(1, std::memory_order_release);
  return DQ_OK;
}

}  // namespace dq
