// Launch helpers of the 4-bit KV cache kernels.
#pragma once

#include <atomic>
#include <cstdint>
#include <cuda_runtime.h>

namespace dialb200 {

// Kernel's dynamic shared memory limit, raised once a device.
template <auto Kernel>
cudaError_t kv4_allow_smem(size_t bytes) {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
  return e;
}

// A launch that may begin while the kernel before it in the stream ends; every
// kernel launched so waits (griddepcontrol.wait) before it touches memory that
// the stream's earlier work writes or reads.
template <typename K, typename... Args>
cudaError_t kv4_start(K kernel, dim3 grid, int threads, size_t smem, cudaStream_t s, const Args&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace dialb200
