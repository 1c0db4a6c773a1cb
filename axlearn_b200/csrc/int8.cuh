// Values held in 8 bits: a block with the largest magnitude A holds whole numbers c = round(127 x / A), ties to even, and stands
// for c A / 127.  A block with a NaN or an infinity stands for NaN; one whose A is below 2^-119, where 127 / A would leave fp32,
// for zeros.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <stdint.h>

namespace axb {

constexpr float kInt8Least = 0x1p-119f;
constexpr float kInt8Whole = 12582912.f;  // 1.5 * 2^23: whole numbers are the last bits

// What turns values into codes: A, and kFactor / A (0 in blocks of zeros and of NaN).  kFactor is 127, or 1 where values are
// codes times another block's A.
template <int kFactor = 127>
struct Int8Scale {
  float top, inverse;
  __device__ __forceinline__ explicit Int8Scale(float a) : top(a), inverse(0.f) {
    if (!(a <= FLT_MAX)) top = __int_as_float(0x7fffffff);
    else if (a < kInt8Least) top = 0.f;
    else inverse = kFactor / a;
  }
  __device__ __forceinline__ bool empty() const { return inverse == 0.f; }
};

// Codes of eight values.  A product with the rounded kFactor / A is within 2^-15 of kFactor x / A, so its rounding is right
// unless it ends next to a half; there kFactor x - c A tells whether a neighbour is nearer.  With x and A of 8 bits (a cache) or
// of 16 (products of two bf16 numbers) that difference is exact.
template <int kFactor>
__device__ __forceinline__ void int8_levels(const float (&x)[8], const Int8Scale<kFactor>& s, float (&level)[8]) {
  if (s.empty()) {
#pragma unroll
    for (int i = 0; i < 8; ++i) level[i] = 0.f;
    return;
  }
  float off_by = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float t = x[i] * s.inverse;
    level[i] = (t + kInt8Whole) - kInt8Whole;
    off_by = fmaxf(off_by, fabsf(t - level[i]));
  }
  if (off_by > 0.5f - 0x1p-14f) {
    const float half = 0.5f * s.top;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float rest = fmaf(static_cast<float>(kFactor), x[i], -level[i] * s.top);
      const bool odd = static_cast<int>(level[i]) & 1;
      if (rest > half || (rest == half && odd)) level[i] += 1.f;
      if (rest < -half || (rest == -half && odd)) level[i] -= 1.f;
    }
  }
}

// Eight codes as bytes.
__device__ __forceinline__ uint2 int8_pack(const float (&level)[8]) {
  uint32_t u[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) u[i] = __float_as_uint(level[i] + kInt8Whole);
  return make_uint2(__byte_perm(__byte_perm(u[0], u[1], 0x0040), __byte_perm(u[2], u[3], 0x0040), 0x5410),
                    __byte_perm(__byte_perm(u[4], u[5], 0x0040), __byte_perm(u[6], u[7], 0x0040), 0x5410));
}

// A bad index that the device found: code 5 of the status word.
__device__ __forceinline__ void int8_report(int* status) { *reinterpret_cast<volatile int*>(status) = 5; }

}  // namespace axb
