// Values held in 4 bits: a group of values shares two bf16 numbers (s, m) and every value is a code c of 0..15 that stands for
// m + s c.  Cache rows of a head of H dims: groups of 32 dims, G = H / 32 of them; H / 2 bytes of codes in 8 chunks, chunk r
// with dims 4r .. 4r + 3 of every group, group by group (the lower dim in the lower half of a byte), and G pairs (s, m).  A
// chunk is what a row of an MMA tile needs of V, two neighbouring chunks are what a lane needs of K.
#pragma once

#include <cuda_bf16.h>
#include <stdint.h>

#include "mma_sync.cuh"

namespace axb {

constexpr int kInt4Group = 32;

// Bits [4i, 4i + 4) and [16 + 4i, 20 + 4i) of x as two bf16 numbers 128 + code: the codes are the last bits of a mantissa
// of 128 = 2^7, so a shift and one logic operation convert two of them.  The 128 is taken off the sums.
__device__ __forceinline__ uint32_t int4_pair(uint32_t x, int i) {
  uint32_t y;
  asm("lop3.b32 %0, %1, 0x000f000f, 0x43004300, 0xEA;" : "=r"(y) : "r"(x >> (4 * i)));
  return y;
}

// The two bf16 of a pair (s, m) as they lie.
__device__ __forceinline__ float pair_s(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float pair_m(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }

// A bad index that the device found: code 5 of the status word.
__device__ __forceinline__ void int4_report(int* status) { *reinterpret_cast<volatile int*>(status) = 5; }

}  // namespace axb
