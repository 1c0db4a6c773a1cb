// Rows of keys, values and queries on their way into a paged cache.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "mma_sync.cuh"

namespace axb {

// n / d for n below 2^31.
struct FastDiv {
  uint32_t d, mul, shift;
  FastDiv() = default;
  explicit FastDiv(int by) : d(static_cast<uint32_t>(by)), shift(31) {
    while ((uint64_t{1} << (shift - 31)) < d) ++shift;
    mul = static_cast<uint32_t>(((uint64_t{1} << shift) + d - 1) / d);
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const {
    return static_cast<uint32_t>((static_cast<uint64_t>(n) * mul) >> shift);
  }
};

// Rows of heads in: element strides of (sequence, token, head); dims are neighbours.
struct HeadRows {
  const __nv_bfloat16* x;
  int64_t b, t, h;
};

// Dims 8 l .. 8 l + 7 of a head, turned as interleaved pairs by (sin, cos) `at[0 .. 4)`.
__device__ __forceinline__ uint4 rotate8(uint4 x, const float2* at) {
  uint32_t* w = reinterpret_cast<uint32_t*>(&x);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack2(w[i]), a = at[i];
    w[i] = pack2(f.x * a.y - f.y * a.x, f.y * a.y + f.x * a.x);
  }
  return x;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace axb
