// Values held in 8 bits: a block with the largest magnitude A holds whole numbers c = round(127 x / A), ties to even, and stands
// for c A / 127.  A block with a NaN or an infinity stands for NaN; one whose A is below 2^-119, where 127 / A would leave fp32,
// for zeros.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <stdint.h>

#include <initializer_list>

#include "f32x2.cuh"

namespace axb {

constexpr float kInt8Least = 0x1p-119f;
constexpr float kInt8Whole = 12582912.f;  // 1.5 * 2^23: whole numbers are the last bits

// What turns values into codes.  kFactor is 127, or 1 where values are codes times another block's A.
template <int kFactor = 127>
struct Int8Scale {
  float top;                          // A, as the block has it: NaN, or 0 of a block of zeros
  float factor, divisor, reciprocal;  // kFactor and A, both 2^-8 of it where kFactor x could leave fp32
  __device__ __forceinline__ explicit Int8Scale(float a) : top(a) {
    if (!(a <= FLT_MAX)) top = __int_as_float(0x7fffffff);
    else if (a < kInt8Least) top = 0.f;
    const float down = a > 0x1p100f ? 0x1p-8f : 1.f;
    factor = kFactor * down, divisor = a * down;
    reciprocal = top > 0.f ? __frcp_rn(divisor) : 0.f;
  }
  __device__ __forceinline__ bool empty() const { return reciprocal == 0.f; }
};

// Codes of eight values as bytes.  The quotient is a product with the reciprocal and one correction by the exact remainder of a fused
// product (Markstein, IBM J. Res. Dev. 34, 1990), which rounds it correctly in 32 bits; with x and A of 8 bits (a cache) or of 16 (products of two bf16 numbers) a quotient that is not
// k + 1/2 is off it by more than half a unit, so adding 1.5 2^23 rounds as in exact arithmetic.  Ties are no rare case to be left
// to a branch: x = A / 2 is 63.5 (every second vector of 256 values has one; 16384 x 4096 rows 49.1 us with such a branch, 39.6 without).
// A level is a float with its code in the last bits.  `kPairs`: two values an instruction, where it pays (us without / with them: rows of
// 16384 x 4096 39.6 / 33.5, silu(gate) * up of 16384 x 11008 183 / 202, an append of 8 x 2048 23.4 / 24.3).
template <bool kPairs, int kFactor>
__device__ __forceinline__ void int8_levels(uint32_t (&u)[8], const float (&x)[8], const Int8Scale<kFactor>& s) {
  if constexpr (kPairs) {
    const uint64_t factor = f32x2(s.factor, s.factor), by = f32x2(s.reciprocal, s.reciprocal), minus = f32x2(-s.divisor, -s.divisor);
    const uint64_t whole = f32x2(kInt8Whole, kInt8Whole);
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const uint64_t y = mul2(f32x2(x[i], x[i + 1]), factor), q = mul2(y, by);
      const uint64_t level = s.empty() ? whole : add2(fma2(fma2(q, minus, y), by, q), whole);
      u[i] = static_cast<uint32_t>(level), u[i + 1] = static_cast<uint32_t>(level >> 32);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float y = x[i] * s.factor, q = y * s.reciprocal;
      u[i] = s.empty() ? __float_as_uint(kInt8Whole) : __float_as_uint(fmaf(fmaf(-q, s.divisor, y), s.reciprocal, q) + kInt8Whole);
    }
  }
}

__device__ __forceinline__ uint2 int8_bytes(const uint32_t (&u)[8]) {
  return make_uint2(__byte_perm(__byte_perm(u[0], u[1], 0x0040), __byte_perm(u[2], u[3], 0x0040), 0x5410),
                    __byte_perm(__byte_perm(u[4], u[5], 0x0040), __byte_perm(u[6], u[7], 0x0040), 0x5410));
}

template <int kFactor>
__device__ __forceinline__ uint2 int8_codes(const float (&x)[8], const Int8Scale<kFactor>& s) {
  uint32_t u[8];
  int8_levels<false>(u, x, s);
  return int8_bytes(u);
}

// What levels stand for, rounded to bf16: their codes times A / 127.
__device__ __forceinline__ uint4 int8_values(const uint32_t (&u)[8], float scale) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 v = __floats2bfloat162_rn((__uint_as_float(u[2 * i]) - kInt8Whole) * scale,
                                                   (__uint_as_float(u[2 * i + 1]) - kInt8Whole) * scale);
    w[i] = reinterpret_cast<const uint32_t&>(v);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// The larger magnitude; NaN is the largest of all.
__device__ __forceinline__ float int8_larger(float top, float x) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(top), "f"(fabsf(x)));
  return y;
}

// Arguments of the entry points travel as one block of 64-bit words (pointers, whole numbers, and doubles), in the order of their
// structs: twenty of ctypes' conversions cost 3 us, packing them 1.
struct Int8RowsCall {
  const void* x;
  void* codes;
  float* scales;
  int64_t rows, dim, ldx, gated;
};
struct Int8NormCall {
  const void *x, *residual, *weight;
  void *total, *codes;
  float* scales;
  void* values;
  int64_t rows, dim;
  double eps;
};
struct Int8LinearCall {
  const void* x;
  const float* x_scales;
  const void* w;
  const float* w_scales;
  void* y;
  int64_t M, N, K, accumulate, plan, resident;  // plan: slices of K (0: free) of up to 128 rows, features of a tile of more
  int* status;
};
struct Int8DenseCall {
  const void* x;  // [M, K] in bf16
  int64_t ldx;
  void* held;     // room for its codes [M, K] and, behind them, scales [M]
  const void* w;
  const float* w_scales;
  void* y;
  int64_t M, N, K, accumulate, features, resident;  // features: 0: up to 128 rows
  int* status;
};
struct Int8AppendCall {
  const void *k, *v;
  int64_t k_b, k_t, k_h, v_b, v_t, v_h;
  void *k_out, *v_out, *k_codes, *k_tops, *v_codes, *v_tops;
  const int *page_table, *start, *live;
  int64_t B, T, num_kv_heads, head_dim, page_size, max_pages, num_pages;
  int* status;
};
struct Int8RopeAppendCall {
  void *qkv, *q_out, *k_codes, *k_tops, *v_codes, *v_tops;
  const int *page_table, *lengths, *live;
  const float* angle;
  int64_t angle_rows, B, T, num_q_heads, num_kv_heads, head_dim, page_size, max_pages, num_pages;
  int* status;
};
struct Int8AttnCall {
  const void *q, *k_codes, *k_tops, *v_codes, *v_tops;
  const int *page_table, *lengths;
  void* out;
  float* scratch;
  int64_t limit, B, num_q_heads, num_kv_heads, head_dim, page_size, max_pages, num_pages, splits;
  double softmax_scale;
  int* status;
};

}  // namespace axb

extern "C" int axb_int8_rows(const axb::Int8RowsCall* call, cudaStream_t stream);
extern "C" int axb_int8_gemm(const axb::Int8LinearCall* call, cudaStream_t stream);
extern "C" int axb_gemm_skinny_int8(const axb::Int8LinearCall* call, cudaStream_t stream);

namespace axb {

// Whether whole numbers of a call are those of an `int`.
inline bool int8_ints(std::initializer_list<int64_t> values) {
  for (int64_t v : values)
    if (v < -0x7fffffffll || v > 0x7fffffffll) return false;
  return true;
}

}  // namespace axb
