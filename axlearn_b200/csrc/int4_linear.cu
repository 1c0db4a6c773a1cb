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
//   int4_linear_kernel   up to 16 rows: features are the M side of the MMA, rows of x its N side.  A CTA takes 64 features and
//                        a slice of K, its four warps every fourth 128 rows of the slice; `cp.async` fills a warp's ring of
//                        three units ahead of the arithmetic.  Partial sums meet in shared memory, those of the slices in
//                        the cluster's.  y = sum_g s_g (sum x c) + m_g sum x, sums of x by an MMA with ones; codes enter as
//                        denormal bf16 numbers (`int4.cuh`), x is multiplied by 2^kInt4Shift: no code is ever converted.
//                        Measured (us; the codes at the copy rate): 1 x 2048 x 2048 3.6 (0.3), 1 x 4096 x 28672 16.9 (9.5: copies
//                        alone take 11.2, arithmetic alone 15.5), 16 x 14336 x 4096 15.0 (4.9), 1 x 16384 x 18944 33.2 (25.2).
//                        No pipe is full (one row: issue 42%, ALU 43%, MMAs 31%; 16 rows, at 182 registers two CTAs an SM: 37%,
//                        34%, 37%): what bounds it is latency at few warps an SM, and at 28672 columns 448 CTAs on 148 SMs.  More
//                        CTAs an SM with fewer features each, or with a shorter ring, were not faster: sums of x and loads of x
//                        grow as fast.
//   int4_expand_kernel   W in bf16 for the tensor-core GEMM of more rows.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "chain.cuh"
#include "cluster.cuh"
#include "int4.cuh"
#include "mma_sync.cuh"

namespace axb {

struct Int4LinearParams {
  const __nv_bfloat16* x;  // [M, ldx]
  const uint4* codes;
  const uint2* pairs;      // of features r and r + 8
  __nv_bfloat16* y;        // [M, ldy]
  int64_t ldx, ldy;
  int M, N, K;
  int accumulate;
  int splits;              // slices of K, the CTAs of a cluster
};

__device__ __forceinline__ void cp_async_zfill(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}

__device__ __forceinline__ uint32_t times_bf16x2(uint32_t x, __nv_bfloat162 f) {
  const __nv_bfloat162 y = __hmul2(reinterpret_cast<__nv_bfloat162&>(x), f);
  return reinterpret_cast<const uint32_t&>(y);
}

constexpr int kLinWarps = 4, kLinThreads = 32 * kLinWarps;
constexpr int kLinStages = 3;
constexpr int kLinMaxSplits = 8;

constexpr int kLinTiles = 4;  // of 16 features

// kBlocks: 8 rows of x each; kGroup: 64 or 128.
template <int kBlocks, int kGroup>
struct Int4Lin {
  static constexpr int kGroups = 128 / kGroup;                      // of a unit: kLinTiles x 16 features, 128 rows of W
  static constexpr int kCodes = kLinTiles * 1024, kPairs = kLinTiles * kGroups * 64;
  static constexpr int kUnit = kCodes + kPairs;
  static constexpr int kRows = kBlocks * 8, kFeatures = kLinTiles * 16;
  static constexpr int kPitch = kFeatures + 4;                      // floats of a row of partial sums
  static constexpr int kRing = kLinWarps * kLinStages * kUnit, kSums = (kLinWarps + 1) * kRows * kPitch * 4;
  static constexpr int kSmem = kRing > kSums ? kRing : kSums;
};

template <int kBlocks, int kGroup>
__global__ void __launch_bounds__(kLinThreads)
int4_linear_kernel(Int4LinearParams p) {
  chain_link();
  using L = Int4Lin<kBlocks, kGroup>;
  extern __shared__ __align__(128) uint8_t s_lin[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  const int n16 = (p.N + 15) / 16, k128 = (p.K + 127) / 128;
  const int split = blockIdx.x % p.splits;
  const int tile0 = blockIdx.x / p.splits * kLinTiles;
  const int per_split = (k128 + p.splits - 1) / p.splits;
  const int hi = min(k128, (split + 1) * per_split);
  uint8_t* ring = s_lin + warp * kLinStages * L::kUnit;
  // A unit: 16-byte pieces of the codes (lane by lane as the MMA takes them), then of the pairs.  Tiles behind the last one
  // are zeros.
  auto load = [&](int stage, int kb) {
    const uint32_t dst = sptr(ring) + stage * L::kUnit + lane * 16;
#pragma unroll
    for (int i = 0; i < kLinTiles; ++i) {
      const bool ok = tile0 + i < n16;
      const int64_t tile = ok ? tile0 + i : 0;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        cp_async_zfill(dst + (2 * i + h) * 512, p.codes + (tile * (2 * k128) + 2 * kb + h) * 32 + lane, ok);
    }
    constexpr int kPieces = L::kPairs / 16, kOfTile = L::kGroups * 4;
#pragma unroll
    for (int at = 0; at < kPieces; at += 32) {
      const int i = (at + lane) / kOfTile, piece = (at + lane) % kOfTile;
      if (at + lane < kPieces) {
        const bool ok = tile0 + i < n16;
        const int64_t tile = ok ? tile0 + i : 0;
        cp_async_zfill(dst + L::kCodes + at * 16,
                       reinterpret_cast<const uint4*>(p.pairs) + (tile * k128 + kb) * kOfTile + piece, ok);
      }
    }
  };
  int kb = split * per_split + warp;
#pragma unroll
  for (int i = 0; i < kLinStages; ++i) {
    if (kb + i * kLinWarps < hi) load(i, kb + i * kLinWarps);
    cp_commit();
  }
  float acc[kLinTiles][kBlocks][4] = {};
  const __nv_bfloat162 up = __float2bfloat162_rn(kInt4Scale);
  // 64 rows of W meet 16 neighbouring values of each row of x in a lane: asked for a unit ahead.
  uint4 xv[2][kBlocks][2];
  auto load_x = [&](int h, int unit) {
#pragma unroll
    for (int j = 0; j < kBlocks; ++j) {
      const int row = j * 8 + r, k = unit * 128 + h * 64 + c * 16;
      const uint4* src = reinterpret_cast<const uint4*>(p.x + row * p.ldx + k);
      const bool ok = row < p.M && unit < hi;
      xv[h][j][0] = ok && k < p.K ? src[0] : make_uint4(0, 0, 0, 0);
      xv[h][j][1] = ok && k + 8 < p.K ? src[1] : make_uint4(0, 0, 0, 0);
    }
  };
  load_x(0, kb), load_x(1, kb);
  int stage = 0;
  for (; kb < hi; kb += kLinWarps) {
    float part[kLinTiles][kBlocks][4], xs[kBlocks][4];
    cp_wait_group<kLinStages - 1>();
    __syncwarp();
    const uint8_t* unit = ring + stage * L::kUnit;
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
      uint4 w[kLinTiles];
#pragma unroll
      for (int i = 0; i < kLinTiles; ++i) w[i] = *reinterpret_cast<const uint4*>(unit + (2 * i + h) * 512 + lane * 16);
      uint32_t xb[kBlocks][8];
#pragma unroll
      for (int j = 0; j < kBlocks; ++j) {
        const uint32_t* u = reinterpret_cast<const uint32_t*>(xv[h][j]);
#pragma unroll
        for (int e = 0; e < 8; ++e) xb[j][e] = times_bf16x2(u[e], up);
      }
      load_x(h, kb + kLinWarps);
      const uint32_t ones[4] = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
#pragma unroll
      for (int q = 0; q < 4; ++q) {
#pragma unroll
        for (int j = 0; j < kBlocks; ++j) mma(xs[j], ones, xb[j][2 * q], xb[j][2 * q + 1]);
#pragma unroll
        for (int i = 0; i < kLinTiles; ++i) {
          const uint32_t word = q == 0 ? w[i].x : q == 1 ? w[i].y : q == 2 ? w[i].z : w[i].w, next = word >> 8;
          const uint32_t a[4] = {int4_low(word), int4_high(word), int4_low(next), int4_high(next)};
#pragma unroll
          for (int j = 0; j < kBlocks; ++j) mma(part[i][j], a, xb[j][2 * q], xb[j][2 * q + 1]);
        }
      }
      if (h == 1 || kGroup == 64) {
#pragma unroll
        for (int i = 0; i < kLinTiles; ++i) {
          const uint2 u = *reinterpret_cast<const uint2*>(unit + L::kCodes + (i * L::kGroups + (kGroup == 64 ? h : 0)) * 64 + r * 8);
          // x carries kInt4Scale, its products with codes 1 / kInt4Back, those of the features r + 8 sixteen times that.
          const float s0 = pair_s(u.x) * kInt4Back, s1 = pair_s(u.y) * (kInt4Back / 16.f);
          const float m0 = pair_m(u.x) * (1.f / kInt4Scale), m1 = pair_m(u.y) * (1.f / kInt4Scale);
#pragma unroll
          for (int j = 0; j < kBlocks; ++j) {
            acc[i][j][0] = fmaf(s0, part[i][j][0], fmaf(m0, xs[j][0], acc[i][j][0]));
            acc[i][j][1] = fmaf(s0, part[i][j][1], fmaf(m0, xs[j][1], acc[i][j][1]));
            acc[i][j][2] = fmaf(s1, part[i][j][2], fmaf(m1, xs[j][0], acc[i][j][2]));
            acc[i][j][3] = fmaf(s1, part[i][j][3], fmaf(m1, xs[j][1], acc[i][j][3]));
          }
        }
      }
    }
    __syncwarp();  // the unit has been read
    if (kb + kLinStages * kLinWarps < hi) load(stage, kb + kLinStages * kLinWarps);
    cp_commit();
    if (++stage == kLinStages) stage = 0;
  }
  cp_wait_all();
  __syncthreads();  // the sums overlay the rings
  float* s_sum = reinterpret_cast<float*>(s_lin);
#pragma unroll
  for (int i = 0; i < kLinTiles; ++i)
#pragma unroll
    for (int j = 0; j < kBlocks; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        s_sum[(warp * L::kRows + j * 8 + 2 * c + (e & 1)) * L::kPitch + i * 16 + (e >> 1) * 8 + r] = acc[i][j][e];
  __syncthreads();
  const int rows = min(p.M, L::kRows);
  float* s_own = s_sum + kLinWarps * L::kRows * L::kPitch;
  for (int at = threadIdx.x; at < rows * L::kFeatures; at += kLinThreads) {
    const int row = at / L::kFeatures, n = at % L::kFeatures;
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kLinWarps; ++w) sum += s_sum[(w * L::kRows + row) * L::kPitch + n];
    s_own[row * L::kPitch + n] = sum;
  }
  if (p.splits > 1) cluster_sync_all();
  else __syncthreads();
  for (int at = threadIdx.x + split * kLinThreads; at < rows * L::kFeatures; at += p.splits * kLinThreads) {
    const int row = at / L::kFeatures, f = at % L::kFeatures, n = tile0 * 16 + f;
    if (n >= p.N) continue;
    float sum = 0.f;
    if (p.splits == 1) {
      sum = s_own[row * L::kPitch + f];
    } else {
      float v[kLinMaxSplits];
#pragma unroll
      for (int q = 0; q < kLinMaxSplits; ++q) v[q] = q < p.splits ? ld_cluster_f32(sptr(s_own + row * L::kPitch + f), q) : 0.f;
#pragma unroll
      for (int q = 0; q < kLinMaxSplits; ++q) sum += v[q];
    }
    __nv_bfloat16* dst = p.y + row * p.ldy + n;
    if (p.accumulate) sum += __bfloat162float(*dst);
    *dst = __float2bfloat16(sum);
  }
  if (p.splits > 1) cluster_sync_all();  // a CTA's shared memory outlives its readers
}

// W^T [N16 * 16, K128 * 128] in bf16: a warp two blocks, 16 features x 128 rows of W, a lane 16 neighbouring values of features
// r and r + 8 of each.  Lanes of a pair swap halves, so that a store fills whole sectors: [4096, 4096] 6.9 us (6.5 at the copy
// rate), 11.0 without.
__global__ void __launch_bounds__(256)
int4_expand_kernel(const uint4* codes, const uint2* pairs, __nv_bfloat16* out, int n16, int k128, int group) {
  const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  const int64_t units = static_cast<int64_t>(n16) * k128;
  for (int64_t unit = blockIdx.x * int64_t{8} + (threadIdx.x >> 5); unit < units; unit += gridDim.x * int64_t{8}) {
    const int64_t tile = unit / k128;
    const int kb = static_cast<int>(unit - tile * k128);
    uint4 w[2];
    uint2 u[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      w[h] = codes[(2 * unit + h) * 32 + lane];
      u[h] = pairs[(group == 64 ? 2 * unit + h : unit) * 8 + r];
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t words[4] = {w[h].x, w[h].y, w[h].z, w[h].w};
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint32_t pair = half ? u[h].y : u[h].x;
        const float s = pair_s(pair), m = pair_m(pair);
        uint32_t v[8];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e)  // rows 4j + 2e, + 1: bytes e and 2 + e
            v[2 * j + e] = pack2(fmaf(s, static_cast<float>((words[j] >> (8 * e + 4 * half)) & 15u), m),
                                 fmaf(s, static_cast<float>((words[j] >> (16 + 8 * e + 4 * half)) & 15u), m));
        // Even lanes keep their first half and get their neighbour's, odd ones the second halves: 16-byte pieces c & 2 and c & 1
        // of two neighbours' 64 bytes.
        uint32_t first[4], second[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t other = __shfl_xor_sync(0xffffffffu, c & 1 ? v[i] : v[4 + i], 1);
          first[i] = c & 1 ? other : v[i];
          second[i] = c & 1 ? v[4 + i] : other;
        }
        uint4* dst = reinterpret_cast<uint4*>(out + (tile * 16 + half * 8 + r) * (int64_t{128} * k128) + kb * 128 + h * 64 +
                                              (c >> 1) * 32 + (c & 1) * 8);
        dst[0] = make_uint4(first[0], first[1], first[2], first[3]);
        dst[2] = make_uint4(second[0], second[1], second[2], second[3]);
      }
    }
  }
}

template <int kBlocks, int kGroup>
static int launch_int4_linear(Int4LinearParams p, int splits, cudaStream_t stream) {
  using L = Int4Lin<kBlocks, kGroup>;
  constexpr auto kernel = int4_linear_kernel<kBlocks, kGroup>;
  static OptIn opt_in;
  if (!opt_in.done(kernel, L::kSmem)) return -3;
  p.splits = splits;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {static_cast<unsigned>(splits), 1, 1};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((p.N + L::kFeatures - 1) / L::kFeatures * splits));
  cfg.blockDim = dim3(kLinThreads);
  cfg.dynamicSmemBytes = L::kSmem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = static_cast<unsigned>(chain_attribute(attr, 1));
  return cudaLaunchKernelEx(&cfg, kernel, p) == cudaSuccess ? 0 : -4;
}

template <int kGroup>
static int int4_linear(const Int4LinearParams& p, int splits, cudaStream_t stream) {
  if (p.M <= 8) return launch_int4_linear<1, kGroup>(p, splits, stream);
  return launch_int4_linear<2, kGroup>(p, splits, stream);
}

}  // namespace axb

// x [M, K] bf16 with rows of ldx (K, ldx multiples of 8, 16-byte aligned), y [M, N] with rows of ldy; M <= 16.
extern "C" int axb_int4_linear(const void* x, const void* codes, const void* pairs, void* y, int M, int N, int K, int group,
                               int64_t ldx, int64_t ldy, int accumulate, int splits, cudaStream_t stream) {
  using namespace axb;
  const uintptr_t align = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(pairs);
  if (M < 0 || M > 16 || N < 1 || K < 1 || K % 8 || ldx % 8 || (align & 15) || (group != 64 && group != 128) ||
      splits < 1 || splits > kLinMaxSplits)
    return -10;
  if (M == 0) return 0;
  const Int4LinearParams p{static_cast<const __nv_bfloat16*>(x), static_cast<const uint4*>(codes),
                           static_cast<const uint2*>(pairs), static_cast<__nv_bfloat16*>(y), ldx, ldy, M, N, K, accumulate, 1};
  return group == 64 ? int4_linear<64>(p, splits, stream) : int4_linear<128>(p, splits, stream);
}

// out [ceil(N / 16) * 16, ceil(K / 128) * 128] bf16, 16-byte aligned: W^T with its padding.
extern "C" int axb_int4_expand(const void* codes, const void* pairs, void* out, int N, int K, int group, cudaStream_t stream) {
  using namespace axb;
  const uintptr_t align = reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(pairs);
  if (N < 1 || K < 1 || (align & 15) || (group != 64 && group != 128)) return -10;
  const int n16 = (N + 15) / 16, k128 = (K + 127) / 128;
  int64_t ctas = (static_cast<int64_t>(n16) * k128 + 7) / 8;
  if (ctas > 148 * 8) ctas = 148 * 8;
  int4_expand_kernel<<<static_cast<unsigned>(ctas), 256, 0, stream>>>(static_cast<const uint4*>(codes),
                                                                      static_cast<const uint2*>(pairs),
                                                                      static_cast<__nv_bfloat16*>(out), n16, k128, group);
  return cudaGetLastError() == cudaSuccess ? 0 : -4;
}
