// Values held in 8 bits: a block with the largest magnitude A holds whole numbers c = round(127 x / A), ties to even, and stands
// for c A / 127.  A block with a NaN or an infinity stands for NaN; one whose A is below 2^-119, where 127 / A would leave fp32,
// for zeros.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <stdint.h>

#include <initializer_list>

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

// Codes of eight values as bytes, and as floats.  x times the rounded kFactor / A is within 2^-15 of kFactor x / A, so its
// rounding is right unless it ends next to a half; there kFactor x - c A tells whether a neighbour is nearer.  With x and A of 8
// bits (a cache) or of 16 (products of two bf16 numbers) that difference is exact.
template <int kFactor>
__device__ __forceinline__ uint2 int8_codes(const float (&x)[8], const Int8Scale<kFactor>& s, float (&level)[8]) {
  if (s.empty()) {
#pragma unroll
    for (int i = 0; i < 8; ++i) level[i] = 0.f;
    return make_uint2(0, 0);
  }
  float off_by = 0.f;
  uint32_t u[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float whole = fmaf(x[i], s.inverse, kInt8Whole);
    u[i] = __float_as_uint(whole);
    level[i] = whole - kInt8Whole;
    off_by = fmaxf(off_by, fabsf(fmaf(x[i], s.inverse, -level[i])));
  }
  if (off_by > 0.5f - 0x1p-14f) {
    const float half = 0.5f * s.top;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float rest = fmaf(static_cast<float>(kFactor), x[i], -level[i] * s.top);
      const bool odd = static_cast<int>(level[i]) & 1;
      if (rest > half || (rest == half && odd)) level[i] += 1.f;
      if (rest < -half || (rest == -half && odd)) level[i] -= 1.f;
      u[i] = __float_as_uint(level[i] + kInt8Whole);
    }
  }
  return make_uint2(__byte_perm(__byte_perm(u[0], u[1], 0x0040), __byte_perm(u[2], u[3], 0x0040), 0x5410),
                    __byte_perm(__byte_perm(u[4], u[5], 0x0040), __byte_perm(u[6], u[7], 0x0040), 0x5410));
}

// A bad index that the device found: code 5 of the status word.
__device__ __forceinline__ void int8_report(int* status) { *reinterpret_cast<volatile int*>(status) = 5; }

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
