// Products with weights held in 4 bits: y[M, N] = x[M, K] W (+ y), W [K, N] in groups of 64 or 128 rows of a column, each
// with a step s and a smallest value m (bf16), W[k, n] = m + s c.
//
// Layout: blocks of 16 features (columns) x 64 rows, [N / 16, K / 64, 512] bytes, in the order in which a lane of an
// m16n8k16 MMA holds its A operand: lane (r, c) = (lane / 4, lane % 4) has the 16 bytes of features r, r + 8 and rows
// 16c .. 16c + 15, one 32-bit word for each of four MMAs; word j holds rows 16c + 4j .. + 3, byte (2 odd + pair) the row
// 4j + 2 pair + odd, feature r in the lower half and r + 8 in the upper.  K is padded to 128, N to 16.  Pairs:
// [N / 16, K / group, 8, 2, (s, m)] by feature mod 8, feature / 8.  The contraction order is permuted the same way on both
// sides: a lane reads 16 neighbouring values of a row of x.
//
//   int4_linear_kernel   up to 64 rows: features are the M side of the MMA, rows of x its N side; a CTA takes 32 features,
//                        its warps every eighth 128 rows of W; partial sums meet in shared memory.
//                        y = sum_g s_g (sum x c) + m_g sum x, sums of x by an MMA with ones.
//   int4_expand_kernel   W in bf16 for the tensor-core GEMM of more rows.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "chain.cuh"
#include "int4.cuh"
#include "mma_sync.cuh"

namespace axb {

__device__ __forceinline__ uint32_t int4_pair(uint32_t x, int i) {
  uint32_t y;
  asm("lop3.b32 %0, %1, 0x000f000f, 0x43004300, 0xEA;" : "=r"(y) : "r"(x >> (4 * i)));
  return y;
}

struct Int4LinearParams {
  const __nv_bfloat16* x;  // [M, ldx]
  const uint4* codes;
  const uint2* pairs;      // of features r and r + 8
  __nv_bfloat16* y;        // [M, ldy]
  int64_t ldx, ldy;
  int M, N, K;
  int accumulate;
};

constexpr int kLinWarps = 8, kLinThreads = 32 * kLinWarps;
constexpr int kLinTiles = 2;  // 16-feature tiles of a CTA

// kBlocks: 8 rows of x each; kGroup: 64 or 128.
template <int kBlocks, int kGroup>
__global__ void __launch_bounds__(kLinThreads)
int4_linear_kernel(Int4LinearParams p) {
  chain_link();
  extern __shared__ __align__(16) float s_sum[];  // [warp][row of x][32 features]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  const int n16 = (p.N + 15) / 16, k128 = (p.K + 127) / 128;
  const int tile0 = blockIdx.x * kLinTiles;
  float acc[kLinTiles][kBlocks][4] = {};
  for (int kb = warp; kb < k128; kb += kLinWarps) {
    uint4 w[kLinTiles][2];
#pragma unroll
    for (int i = 0; i < kLinTiles; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        w[i][h] = tile0 + i < n16 ? p.codes[(static_cast<int64_t>(tile0 + i) * (2 * k128) + 2 * kb + h) * 32 + lane]
                                  : make_uint4(0, 0, 0, 0);
    float part[kLinTiles][kBlocks][4], xs[kBlocks][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (h == 0 || kGroup == 64) {
#pragma unroll
        for (int j = 0; j < kBlocks; ++j) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            xs[j][e] = 0.f;
#pragma unroll
            for (int i = 0; i < kLinTiles; ++i) part[i][j][e] = 0.f;
          }
        }
      }
      uint32_t xb[kBlocks][8];
#pragma unroll
      for (int j = 0; j < kBlocks; ++j) {
        const int row = j * 8 + r, k = kb * 128 + h * 64 + c * 16;
        const uint4* src = reinterpret_cast<const uint4*>(p.x + row * p.ldx + k);
        uint4 a = make_uint4(0, 0, 0, 0), b = a;
        if (row < p.M && k < p.K) a = src[0];
        if (row < p.M && k + 8 < p.K) b = src[1];
        xb[j][0] = a.x, xb[j][1] = a.y, xb[j][2] = a.z, xb[j][3] = a.w;
        xb[j][4] = b.x, xb[j][5] = b.y, xb[j][6] = b.z, xb[j][7] = b.w;
      }
      const uint32_t ones[4] = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
#pragma unroll
      for (int q = 0; q < 4; ++q) {
#pragma unroll
        for (int j = 0; j < kBlocks; ++j) mma(xs[j], ones, xb[j][2 * q], xb[j][2 * q + 1]);
#pragma unroll
        for (int i = 0; i < kLinTiles; ++i) {
          const uint32_t word = q == 0 ? w[i][h].x : q == 1 ? w[i][h].y : q == 2 ? w[i][h].z : w[i][h].w;
          const uint32_t a[4] = {int4_pair(word, 0), int4_pair(word, 1), int4_pair(word, 2), int4_pair(word, 3)};
#pragma unroll
          for (int j = 0; j < kBlocks; ++j) mma(part[i][j], a, xb[j][2 * q], xb[j][2 * q + 1]);
        }
      }
      if (h == 1 || kGroup == 64) {
        const int g = kGroup == 64 ? 2 * kb + h : kb, groups = kGroup == 64 ? 2 * k128 : k128;
#pragma unroll
        for (int i = 0; i < kLinTiles; ++i) {
          if (tile0 + i >= n16) break;
          const uint2 u = p.pairs[(static_cast<int64_t>(tile0 + i) * groups + g) * 8 + r];
          const float s0 = pair_s(u.x), s1 = pair_s(u.y), m0 = pair_m(u.x) - 128.f * s0, m1 = pair_m(u.y) - 128.f * s1;
#pragma unroll
          for (int j = 0; j < kBlocks; ++j) {
            acc[i][j][0] += s0 * part[i][j][0] + m0 * xs[j][0];
            acc[i][j][1] += s0 * part[i][j][1] + m0 * xs[j][1];
            acc[i][j][2] += s1 * part[i][j][2] + m1 * xs[j][0];
            acc[i][j][3] += s1 * part[i][j][3] + m1 * xs[j][1];
          }
        }
      }
    }
  }
  constexpr int kRows = kBlocks * 8, kFeatures = kLinTiles * 16;
#pragma unroll
  for (int i = 0; i < kLinTiles; ++i)
#pragma unroll
    for (int j = 0; j < kBlocks; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        s_sum[(warp * kRows + j * 8 + 2 * c + (e & 1)) * kFeatures + i * 16 + (e >> 1) * 8 + r] = acc[i][j][e];
  __syncthreads();
  for (int at = threadIdx.x; at < kRows * kFeatures; at += kLinThreads) {
    const int row = at / kFeatures, n = tile0 * 16 + at % kFeatures;
    if (row >= p.M || n >= p.N) continue;
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kLinWarps; ++w) sum += s_sum[w * kRows * kFeatures + at];
    __nv_bfloat16* dst = p.y + row * p.ldy + n;
    if (p.accumulate) sum += __bfloat162float(*dst);
    *dst = __float2bfloat16(sum);
  }
}

// W^T [N16 * 16, K128 * 128] in bf16: a warp a block.
__global__ void __launch_bounds__(256)
int4_expand_kernel(const uint4* codes, const uint2* pairs, __nv_bfloat16* out, int n16, int k64, int group) {
  const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  const int64_t blocks = static_cast<int64_t>(n16) * k64;
  for (int64_t block = blockIdx.x * int64_t{8} + (threadIdx.x >> 5); block < blocks; block += gridDim.x * int64_t{8}) {
    const int64_t tile = block / k64;
    const int kb = static_cast<int>(block - tile * k64);
    const uint4 w = codes[block * 32 + lane];
    const uint2 u = pairs[(tile * (k64 * 64 / group) + kb * 64 / group) * 8 + r];
    const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const uint32_t pair = half ? u.y : u.x;
      const float s = pair_s(pair), m = pair_m(pair);
      uint32_t v[8];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e)  // rows 4j + 2e, + 1: bytes e and 2 + e
          v[2 * j + e] = pack2(fmaf(s, static_cast<float>((words[j] >> (8 * e + 4 * half)) & 15u), m),
                               fmaf(s, static_cast<float>((words[j] >> (16 + 8 * e + 4 * half)) & 15u), m));
      uint4* dst = reinterpret_cast<uint4*>(out + (tile * 16 + half * 8 + r) * (int64_t{64} * k64) + kb * 64 + c * 16);
      dst[0] = make_uint4(v[0], v[1], v[2], v[3]);
      dst[1] = make_uint4(v[4], v[5], v[6], v[7]);
    }
  }
}

template <int kBlocks, int kGroup>
static int launch_int4_linear(const Int4LinearParams& p, cudaStream_t stream) {
  constexpr int kBytes = kLinWarps * kBlocks * 8 * kLinTiles * 16 * 4;
  if constexpr (kBytes > 48 * 1024) {
    static const cudaError_t configured = cudaFuncSetAttribute(int4_linear_kernel<kBlocks, kGroup>,
                                                               cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
    if (configured != cudaSuccess) return -3;
  }
  launch_chained(int4_linear_kernel<kBlocks, kGroup>, (p.N + kLinTiles * 16 - 1) / (kLinTiles * 16), kLinThreads, kBytes, stream, p);
  return cudaGetLastError() == cudaSuccess ? 0 : -4;
}

template <int kGroup>
static int int4_linear(const Int4LinearParams& p, cudaStream_t stream) {
  if (p.M <= 8) return launch_int4_linear<1, kGroup>(p, stream);
  if (p.M <= 16) return launch_int4_linear<2, kGroup>(p, stream);
  if (p.M <= 32) return launch_int4_linear<4, kGroup>(p, stream);
  return launch_int4_linear<8, kGroup>(p, stream);
}

}  // namespace axb

// x [M, K] bf16 with rows of ldx (K, ldx multiples of 8, 16-byte aligned), y [M, N] with rows of ldy; M <= 64.
extern "C" int axb_int4_linear(const void* x, const void* codes, const void* pairs, void* y, int M, int N, int K, int group,
                               int64_t ldx, int64_t ldy, int accumulate, cudaStream_t stream) {
  using namespace axb;
  const uintptr_t align = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(pairs);
  if (M < 0 || M > 64 || N < 1 || K < 1 || K % 8 || ldx % 8 || (align & 15) || (group != 64 && group != 128)) return -10;
  if (M == 0) return 0;
  const Int4LinearParams p{static_cast<const __nv_bfloat16*>(x), static_cast<const uint4*>(codes),
                           static_cast<const uint2*>(pairs), static_cast<__nv_bfloat16*>(y), ldx, ldy, M, N, K, accumulate};
  return group == 64 ? int4_linear<64>(p, stream) : int4_linear<128>(p, stream);
}

// out [ceil(N / 16) * 16, ceil(K / 128) * 128] bf16, 16-byte aligned: W^T with its padding.
extern "C" int axb_int4_expand(const void* codes, const void* pairs, void* out, int N, int K, int group, cudaStream_t stream) {
  using namespace axb;
  const uintptr_t align = reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(pairs);
  if (N < 1 || K < 1 || (align & 15) || (group != 64 && group != 128)) return -10;
  const int n16 = (N + 15) / 16, k64 = (K + 127) / 128 * 2;
  int64_t ctas = (static_cast<int64_t>(n16) * k64 + 7) / 8;
  if (ctas > 148 * 16) ctas = 148 * 16;
  int4_expand_kernel<<<static_cast<unsigned>(ctas), 256, 0, stream>>>(static_cast<const uint4*>(codes),
                                                                      static_cast<const uint2*>(pairs),
                                                                      static_cast<__nv_bfloat16*>(out), n16, k64, group);
  return cudaGetLastError() == cudaSuccess ? 0 : -4;
}
