// More than 48 KB of dynamic shared memory is allowed a kernel for one device at a time, the current one: a launcher keeps a bit for each device that it has
// asked for, not one for the process.
#pragma once
#include <cuda_runtime_api.h>
#include <atomic>
#include <cstdint>

namespace mb {

// `asked`: a static of the launcher, one for each kernel. A device beyond the 64th is asked for again with every call.
inline cudaError_t allow_smem(const void* kernel, int bytes, std::atomic<uint64_t>& asked) {
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  const uint64_t bit = device < 64 ? 1ull << device : 0;
  if (asked.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) asked.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

}  // namespace mb
