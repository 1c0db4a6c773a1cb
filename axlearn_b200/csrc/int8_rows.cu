// Rows of activations in 8 bits (`int8.cuh`), a block a row: of a matrix as it is, of an RMS norm with the residual's addition
// ahead of it, of silu(gate) * up.  Scales are A / 127 in 32 bits.
//
// A CTA takes a row and keeps it in registers, so that memory is read once: the largest magnitude and, for the norm, the sum of
// squares meet in one barrier, since a norm's codes do not depend on its 1 / rms, which only the scale carries: with t the
// summed row and w the norm's weights, round(127 t w / max |t w|).  t w has 16 bits, so codes are those of exact arithmetic.
//
// Measured: the norm of 8192 x 4096 with residual, sum and values 46.3 us (46.1 at the copy rate); rows of 16384 x 4096 33.5 (30.7), of
// 16384 x 11008 97 (83), silu(gate) * up of it 185 (138), which its exponentials and quotients bound.  One row of 2048 takes 1.6 to 1.9,
// an empty launch's time.
#include <math.h>

#include "chain.cuh"
#include "int8.cuh"
#include "mma_sync.cuh"

namespace axb {

enum Int8RowsKind { kRowsPlain, kRowsNorm, kRowsSwiglu };

struct Int8RowsParams {
  const __nv_bfloat16 *x, *other;  // other: the residual (null: none)
  const __nv_bfloat16* weight;     // the norm's
  int64_t ldx;                     // kRowsPlain, kRowsSwiglu
  int8_t* codes;
  float* scales;
  __nv_bfloat16 *total, *values;   // null: not wanted
  int dim;
  float inverse_dim, eps;
};

// t / (1 + exp(-t)), for t < 0 as t exp(t) / (1 + exp(t)): divisors from 1 to 2, where one above 2^126 (t < -87.3) would make the
// approximate quotient zero.  exp(-|t|) carries 2^24, so that it is no denormal ahead of its product with t.  (A unit or two each of
// the exponential, the reciprocal and the products, and |t| 2^-24 of the exponent: nothing beside half a code.  16384 x 11008 185 us, as
// before with the quotient that fails there; with the exponential as it is and a quotient 191.)
__device__ __forceinline__ float int8_silu(float t) {
  const float e = ex2(fmaf(fabsf(t), -1.4426950408889634f, 24.f));
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(fmaf(e, 0x1p-24f, 1.f)));
  return (t < 0.f ? t * e * 0x1p-24f : t) * r;
}

template <int KIND, int VPT, int kThreads>
__global__ void __launch_bounds__(kThreads)
int8_rows_kernel(Int8RowsParams p) {
  chain_link();
  __shared__ float s_sum[32];
  __shared__ uint32_t s_top[32];
  const int64_t row = blockIdx.x;
  const int vectors = p.dim >> 3, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const uint4* x = reinterpret_cast<const uint4*>(p.x + (KIND == kRowsNorm ? row * p.dim : row * p.ldx));
  float f[VPT][8];
  float most[4] = {}, sum = 0.f;
  {
    uint4 a[VPT], b[VPT], w[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = threadIdx.x + i * blockDim.x;
      a[i] = b[i] = w[i] = make_uint4(0, 0, 0, 0);
      if (v >= vectors) continue;
      a[i] = x[v];
      if (KIND == kRowsNorm && p.other != nullptr) b[i] = reinterpret_cast<const uint4*>(p.other + row * p.dim)[v];
      if (KIND == kRowsNorm) w[i] = reinterpret_cast<const uint4*>(p.weight)[v];
      if (KIND == kRowsSwiglu) b[i] = x[vectors + v];
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = threadIdx.x + i * blockDim.x;
      uint32_t u[4] = {a[i].x, a[i].y, a[i].z, a[i].w};
      const uint32_t o[4] = {b[i].x, b[i].y, b[i].z, b[i].w}, g[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
      if (KIND == kRowsNorm && p.other != nullptr) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const __nv_bfloat162 s =
              __hadd2(reinterpret_cast<const __nv_bfloat162&>(u[j]), reinterpret_cast<const __nv_bfloat162&>(o[j]));
          u[j] = reinterpret_cast<const uint32_t&>(s);
        }
        if (v < vectors) reinterpret_cast<uint4*>(p.total + row * p.dim)[v] = make_uint4(u[0], u[1], u[2], u[3]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float2 t = unpack2(u[j]);
        if (KIND == kRowsNorm) {
          sum = fmaf(t.x, t.x, fmaf(t.y, t.y, sum));
          const float2 by = unpack2(g[j]);
          t.x *= by.x, t.y *= by.y;
        } else if (KIND == kRowsSwiglu) {
          const float2 up = unpack2(o[j]);
          t.x = int8_silu(t.x) * up.x;
          t.y = int8_silu(t.y) * up.y;
        }
        f[i][2 * j] = t.x, f[i][2 * j + 1] = t.y;
        most[j] = int8_larger(int8_larger(most[j], t.x), t.y);
      }
    }
  }
  // (Bits are in the same order, NaN at the end.)
  uint32_t top = __float_as_uint(int8_larger(int8_larger(most[0], most[1]), int8_larger(most[2], most[3])));
  top = __reduce_max_sync(0xffffffffu, top);
  if (KIND == kRowsNorm) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  }
  if (warps > 1) {
    if (lane == 0) s_sum[warp] = sum, s_top[warp] = top;
    __syncthreads();
    top = __reduce_max_sync(0xffffffffu, lane < warps ? s_top[lane] : 0u);
    if (KIND == kRowsNorm) {
      sum = lane < warps ? s_sum[lane] : 0.f;
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    }
  }
  const Int8Scale<> s(__uint_as_float(top));
  float scale = 0.f;  // (one thread's, unless all need it)
  if (threadIdx.x == 0 || p.values != nullptr) scale = s.top / 127.f;
  if (KIND == kRowsNorm) scale *= rsqrtf(fmaf(sum, p.inverse_dim, p.eps));
  if (threadIdx.x == 0) p.scales[row] = scale;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    if (v >= vectors) continue;
    uint32_t u[8];
    int8_levels<KIND == kRowsPlain>(u, f[i], s);
    reinterpret_cast<uint2*>(p.codes + row * p.dim)[v] = int8_bytes(u);
    if (p.values != nullptr) reinterpret_cast<uint4*>(p.values + row * p.dim)[v] = int8_values(u, scale);
  }
}

constexpr int kInt8RowsMost = 1024 * 8 * 8;  // values of a row

template <int KIND>
static int int8_rows(const Int8RowsParams& p, int64_t rows, cudaStream_t stream) {
  // Many rows: vectors of a thread so that CTAs are small; few: so that a row is spread wide.  Four vectors and more need the registers
  // that 512 threads leave (rows of 16384 x 11008 97 us, 103 with 1024 threads' registers).
  const int vectors = p.dim / 8, most = rows >= 296 ? 128 : 1024;
  int vpt = 1;
  while (vpt < 8 && (vectors + vpt - 1) / vpt > (vpt < 4 ? most : 512)) vpt *= 2;
  const int threads = ((vectors + vpt - 1) / vpt + 31) / 32 * 32;
  const dim3 grid(static_cast<unsigned>(rows));
  if (vpt == 1) launch_chained(int8_rows_kernel<KIND, 1, 1024>, grid, threads, 0, stream, p);
  else if (vpt == 2) launch_chained(int8_rows_kernel<KIND, 2, 1024>, grid, threads, 0, stream, p);
  else if (vpt == 4) launch_chained(int8_rows_kernel<KIND, 4, 512>, grid, threads, 0, stream, p);
  else if (threads <= 512) launch_chained(int8_rows_kernel<KIND, 8, 512>, grid, threads, 0, stream, p);
  else launch_chained(int8_rows_kernel<KIND, 8, 1024>, grid, threads, 0, stream, p);
  return cudaGetLastError() == cudaSuccess ? 0 : -4;
}

static bool int8_rows_fit(int64_t rows, int64_t dim, int64_t ldx) {
  return rows >= 0 && rows <= 0x7fffffff && dim >= 8 && dim % 8 == 0 && dim <= kInt8RowsMost && ldx % 8 == 0;
}

}  // namespace axb

// codes [rows, dim], scales [rows] of x [rows, dim] with a pitch of ldx; `gated`: of silu(x[:, :dim]) * x[:, dim:].  All pointers
// 16-byte aligned; -10: not supported.
extern "C" int axb_int8_rows(const axb::Int8RowsCall* call, cudaStream_t stream) {
  using namespace axb;
  const Int8RowsCall& a = *call;
  if (!int8_rows_fit(a.rows, a.dim, a.ldx)) return -10;
  for (const void* x : {a.x, static_cast<const void*>(a.codes)})
    if (reinterpret_cast<uintptr_t>(x) & 15) return -10;
  if (a.rows == 0) return 0;
  Int8RowsParams p = {};
  p.x = static_cast<const __nv_bfloat16*>(a.x);
  p.ldx = a.ldx, p.codes = static_cast<int8_t*>(a.codes), p.scales = a.scales, p.dim = static_cast<int>(a.dim);
  return a.gated ? int8_rows<kRowsSwiglu>(p, a.rows, stream) : int8_rows<kRowsPlain>(p, a.rows, stream);
}

// t = x + residual in bf16 (x without one), into `total`; codes and scales of t rsqrt(mean t^2 + eps) weight, and what they stand
// for into `values` (null: not wanted).  Rows of `dim` values one behind the other, 16-byte aligned.
extern "C" int axb_int8_add_rms_norm(const axb::Int8NormCall* call, cudaStream_t stream) {
  using namespace axb;
  const Int8NormCall& a = *call;
  if (!int8_rows_fit(a.rows, a.dim, a.dim) || (a.residual != nullptr && a.total == nullptr)) return -10;
  for (const void* x : {a.x, a.residual, a.weight, static_cast<const void*>(a.total), static_cast<const void*>(a.codes),
                        static_cast<const void*>(a.values)})
    if (reinterpret_cast<uintptr_t>(x) & 15) return -10;
  if (a.rows == 0) return 0;
  Int8RowsParams p = {};
  p.x = static_cast<const __nv_bfloat16*>(a.x), p.other = static_cast<const __nv_bfloat16*>(a.residual);
  p.weight = static_cast<const __nv_bfloat16*>(a.weight);
  p.codes = static_cast<int8_t*>(a.codes), p.scales = a.scales;
  p.total = static_cast<__nv_bfloat16*>(a.total), p.values = static_cast<__nv_bfloat16*>(a.values);
  p.dim = static_cast<int>(a.dim), p.inverse_dim = 1.f / p.dim, p.eps = static_cast<float>(a.eps);
  return int8_rows<kRowsNorm>(p, a.rows, stream);
}
