// A kernel's limit of dynamic shared memory, raised once per device.
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

namespace mccl {
namespace ops {

// `done` is the kernel's own word (a static of its launcher), a bit per device.
template <typename K>
cudaError_t raise_smem_limit(K kernel, int bytes, std::atomic<uint64_t>& done) {
  int device = 0;
  cudaError_t rc = cudaGetDevice(&device);
  if (rc != cudaSuccess) return rc;
  const uint64_t bit = 1ull << (device & 63);
  if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
  rc = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (rc == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
  return rc;
}

}  // namespace ops
}  // namespace mccl
