// Values held in 4 bits: a group of values shares two bf16 numbers (s, m) and every value is a code c of 0..15 that stands for
// m + s c.  Cache rows of a head of H dims: groups of 32 dims, G = H / 32 of them; H / 2 bytes of codes in 8 chunks, chunk r
// with dims 4r .. 4r + 3 of every group, group by group (the lower dim in the lower half of a byte), and G pairs (s, m).  A
// chunk is what a row of an MMA tile needs of V, two neighbouring chunks are what a lane needs of K.
#pragma once

#include <atomic>

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "mma_sync.cuh"

namespace axb {

constexpr int kInt4Group = 32;

// Codes as operands of a product: the bf16 number with the bits v < 256 is v 2^-133 (below 2^-126 a denormal, which MMAs take
// as it is, then the first binade of the same spacing).  So the low nibble of each half is a code times 2^-133 as it lies,
// the next one 16 times that: one logic operation for two codes, and no offset.  The other operand carries 2^kInt4Shift, so
// that products stay far above the denormal numbers of fp32: results are 2^(kInt4Shift - 133) of the sums of codes.
// 64 keeps both sides of fp32's range: x and p up to 2^63, and s and m times them up to 2^55, are no overflow.
constexpr int kInt4Shift = 64;
constexpr float kInt4Scale = 18446744073709551616.f;   // 2^kInt4Shift
constexpr float kInt4Back = 590295810358705651712.f;   // 2^(133 - kInt4Shift)

__device__ __forceinline__ uint32_t int4_low(uint32_t x) { return x & 0x000f000fu; }
__device__ __forceinline__ uint32_t int4_high(uint32_t x) { return x & 0x00f000f0u; }  // 16 codes

// The two bf16 of a pair (s, m) as they lie.
__device__ __forceinline__ float pair_s(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float pair_m(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }

// A bad index that the device found: code 5 of the status word.
__device__ __forceinline__ void int4_report(int* status) { *reinterpret_cast<volatile int*>(status) = 5; }

// A kernel's shared memory above 48 KB, asked for once on each device.
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
