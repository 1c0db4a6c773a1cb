// A kernel's shared memory above 48 KB, asked for once on each device.
#pragma once

#include <atomic>

#include <cuda_runtime.h>
#include <stdint.h>

namespace axb {

struct OptIn {
  std::atomic<uint64_t> devices{0};

  template <typename Kernel>
  bool done(Kernel kernel, int bytes) {
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device > 63) return false;
    const uint64_t bit = uint64_t{1} << device;
    if (devices.load(std::memory_order_acquire) & bit) return true;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
    devices.fetch_or(bit, std::memory_order_release);
    return true;
  }
};

}  // namespace axb
