// y[M, N] = x[M, K] W (+ y) for up to 128 rows with weights held in 4 bits (layout: int4_linear.cu), on the fifth-generation
// tensor cores: 128 features are the M side of the MMA, the rows of x its N side.
//
// Eight warps feed: each owns 16 features and turns their codes of 64 rows of W into bf16 values m + s c (one rounding, 2^-9 of
// a weight, as in the expansion for the GEMM of more rows), which `tcgen05.st` puts into tensor memory -- a lane's words are
// the fragment of the 16x256b shape as they lie --, so that weights never pass through shared memory once they are 16 bits
// wide: writing and reading them there would cost eight times the bytes of the codes.  They also bring x, 64 columns of it at
// a time, to shared memory in the order in which the codes run over K.  A ninth warp issues the MMAs.
// K slices are the CTAs of a cluster; partial sums meet in distributed shared memory in a fixed order.
//
// Launched in the ordinary way in a captured step, too: a successor that started early could hold the tensor memory that a
// CTA of this kernel has yet to get, and wait for it.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "cluster.cuh"
#include "int4.cuh"
#include "mma_sync.cuh"
#include "sm100.cuh"

namespace axb {

struct Int4GemmParams {
  const __nv_bfloat16* x;  // [M, ldx]
  const uint8_t* codes;    // [n16, k64, 512]
  const uint8_t* pairs;    // [n16, groups, 64]
  __nv_bfloat16* y;        // [M, ldy]
  int64_t ldx, ldy;
  int M, N, K, group_shift;  // rows of W a group, as a power of two of 64
  int accumulate, splits;
  int* status;
};

constexpr int kIgWarps = 8, kIgThreads = 32 * (kIgWarps + 1), kIgFeatures = 16 * kIgWarps;
constexpr int kIgMaxSplits = 8;
constexpr int kIgAStages = 4;  // of 64 rows of W in tensor memory: 32 columns

template <int BN>
struct Int4GemmCfg {
  static constexpr int kRing = BN <= 32 ? 10 : BN <= 64 ? 8 : 9;  // stages in shared memory
  static constexpr int kLag = 3;                                  // stages that the products may be behind
  static constexpr int kAhead = kRing - kLag;                     // stages on their way
  static constexpr int kX = BN * 128, kCodes = 576;               // bytes of a stage; of a warp's codes and pairs in it
  static constexpr int kStage = kX + kIgWarps * kCodes;
  static constexpr int kXRing = kRing * kX;
  static constexpr int kRingBytes = kRing * kStage;
  static constexpr int kSums = BN * kIgFeatures * 4;              // partial sums overlay the ring
  static constexpr int kBody = kRingBytes > kSums ? kRingBytes : kSums;
  static constexpr int kSmem = kBody + 256 + 1024;                // barriers, alignment slack
  static constexpr int kResident = BN <= 64 ? 2 : 1;
  static constexpr int kACol = BN <= 64 ? 64 : 128;
  static constexpr int kTmemCols = 256;
  static_assert(kACol + kIgAStages * 32 <= kTmemCols && kIgAStages > kLag, "tensor memory");
  static_assert(kResident * (kSmem + 1024) <= 228 * 1024, "resident CTAs");
};

__device__ __forceinline__ void ig_copy(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void ig_copy8(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(ok ? 8 : 0) : "memory");
}

// 16 lanes x 32 columns: thread (r, c) has columns 8 n + 2c, + 1 of lanes r (entries 4 n, 4 n + 1) and r + 8.
__device__ __forceinline__ void tmem_st_16x256(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// The codes in bits [4i, 4i + 4) and [16 + 4i, 20 + 4i) as values m + s c: 128 + c by one logic operation, c and the value
// by one packed operation each.
__device__ __forceinline__ uint32_t ig_values(uint32_t word, int i, __nv_bfloat162 s, __nv_bfloat162 m) {
  uint32_t u;
  asm("lop3.b32 %0, %1, 0x000f000f, 0x43004300, 0xEA;" : "=r"(u) : "r"(word >> (4 * i)));
  const __nv_bfloat162 c = __hsub2(reinterpret_cast<__nv_bfloat162&>(u), __float2bfloat162_rn(128.f));
  const __nv_bfloat162 v = __hfma2(c, s, m);
  return reinterpret_cast<const uint32_t&>(v);
}

template <int BN>
__global__ void __launch_bounds__(kIgThreads, Int4GemmCfg<BN>::kResident)
int4_gemm_kernel(Int4GemmParams p) {
  using S = Int4GemmCfg<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem =
      reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + S::kBody);
  uint64_t* empty_bar = full_bar + S::kRing;
  uint64_t* done_bar = empty_bar + S::kRing;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done_bar + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = static_cast<int>(blockIdx.x) % p.splits;
  const int n0 = static_cast<int>(blockIdx.x) / p.splits * kIgFeatures;
  const int k64 = (p.K + 127) / 128 * 2, num_kb = (p.K + 63) / 64;
  const int kb_lo = split * num_kb / p.splits, count = (split + 1) * num_kb / p.splits - kb_lo;

  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kRing; ++i) {
      mbar_init(&full_bar[i], kIgWarps);
      mbar_init(&empty_bar[i], 1);
    }
    mbar_init(done_bar, 1);
    fence_barrier_init();
  }
  if (warp == kIgWarps) {
    tmem_alloc(tmem_slot, S::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;

  bool ok = true;
  if (warp < kIgWarps) {
    // Tensor-memory lanes [32 (warp % 4) + 16 (warp / 4), + 16): features of this warp, in their order.
    const int sub = 2 * (warp & 3) + (warp >> 2);
    const int tile = n0 / 16 + sub;
    const bool have = tile < (p.N + 15) / 16;
    const uint32_t a_addr = tmem + (static_cast<uint32_t>(sub * 16) << 16) + S::kACol;
    const uint8_t* codes = p.codes + (static_cast<int64_t>(have ? tile : 0) * k64 + kb_lo) * 512 + lane * 16;
    const int groups = k64 >> p.group_shift;
    const uint8_t* pairs = p.pairs + static_cast<int64_t>(have ? tile : 0) * groups * 64 + lane * 16;
    const uint32_t own = smem_u32(smem) + S::kXRing + warp * S::kCodes;  // + stage * kIgWarps * kCodes
    // x: 16-byte pieces (row, i) of a stage, i of 8: columns 16 c + 8 q + 0 .. 7 with c = i / 2, q = i % 2.  Their halves go
    // to places 4c .. 4c + 3 of the k16 steps 2q and 2q + 1, where the codes of these columns are.
    constexpr int kPieces = BN * 8, kMine = (kPieces + 255) / 256;
    const __nv_bfloat16* x_src[kMine];
    uint32_t x_dst[kMine];
    int x_left[kMine];  // columns from this piece on, in the whole slice and behind it
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
      const int piece = j * 256 + static_cast<int>(threadIdx.x);
      const int row = piece >> 3, i = piece & 7, c = i >> 1, q = i & 1;
      const int unit = 4 * q + (c >> 1);  // of 16 bytes; the second half's is two further
      x_src[j] = p.x + (row < p.M ? row : 0) * p.ldx + kb_lo * 64 + c * 16 + q * 8;
      x_dst[j] = smem_u32(smem) + row * 128 + ((unit ^ (row & 7)) << 4) + (c & 1) * 8;
      x_left[j] = row < p.M && piece < kPieces ? p.K - kb_lo * 64 - c * 16 - q * 8 : 0;
    }
    auto load = [&](int it) {
      const int slot = it % S::kRing;
      const uint32_t dst = own + slot * (kIgWarps * S::kCodes) + lane * 16;
      ig_copy(dst, codes + static_cast<int64_t>(it) * 512, have);
      if (lane < 4) ig_copy(dst + 512, pairs + static_cast<int64_t>((kb_lo + it) >> p.group_shift) * 64, have);
#pragma unroll
      for (int j = 0; j < kMine; ++j) {
        if (kPieces < 256 && static_cast<int>(threadIdx.x) >= kPieces) break;
        const bool there = it * 64 < x_left[j];
        const __nv_bfloat16* src = there ? x_src[j] + it * 64 : p.x;
        const uint32_t at = x_dst[j] + slot * S::kX;
        ig_copy8(at, src, there);
        ig_copy8(at ^ 32, src + 4, there);  // two units further: bit 1 of the unit is 0, swapped or not
      }
    };
#pragma unroll 1
    for (int it = 0; it < S::kAhead; ++it) {
      if (it < count) load(it);
      cp_commit();
    }
#pragma unroll 1
    for (int it = 0; it < count; ++it) {
      // Products up to it - kLag are done: their places in the ring and in tensor memory are free.
      if (it >= S::kLag) {
        const int j = it - S::kLag;
        ok = mbar_wait_warp(&empty_bar[j % S::kRing], (j / S::kRing) & 1, p.status, kStatusWaitTimeoutProducer);
        if (!ok) break;
        tc_fence_after_sync();
      }
      if (it + S::kAhead < count) load(it + S::kAhead);
      cp_commit();
      cp_wait_group<S::kAhead>();
      __syncwarp();
      const uint8_t* unit = smem + S::kXRing + (it % S::kRing) * (kIgWarps * S::kCodes) + warp * S::kCodes;
      const uint4 w = *reinterpret_cast<const uint4*>(unit + lane * 16);
      const uint2 u = *reinterpret_cast<const uint2*>(unit + 512 + (lane >> 2) * 8);
      const __nv_bfloat162 pa = reinterpret_cast<const __nv_bfloat162&>(u.x), pb = reinterpret_cast<const __nv_bfloat162&>(u.y);
      const __nv_bfloat162 s0 = __low2bfloat162(pa), m0 = __high2bfloat162(pa), s1 = __low2bfloat162(pb), m1 = __high2bfloat162(pb);
      const uint32_t words[4] = {w.x, w.y, w.z, w.w};
      uint32_t v[16];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[4 * j] = ig_values(words[j], 0, s0, m0);
        v[4 * j + 1] = ig_values(words[j], 2, s0, m0);
        v[4 * j + 2] = ig_values(words[j], 1, s1, m1);
        v[4 * j + 3] = ig_values(words[j], 3, s1, m1);
      }
      tmem_st_16x256(a_addr + it % kIgAStages * 32, v);
      tmem_st_wait();
      fence_proxy_async();  // x
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&full_bar[it % S::kRing]);
    }
    cp_wait_all();
    if (ok) ok = mbar_wait_warp(done_bar, 0, p.status, kStatusWaitTimeoutEpilogue);
  } else if (elect_one()) {
    constexpr uint32_t idesc = umma_idesc_f16(kIgFeatures, BN, 1, 1, 0, 0);
    bool fed = true;
#pragma unroll 1
    for (int it = 0; it < count; ++it) {
      if (!mbar_wait(&full_bar[it % S::kRing], (it / S::kRing) & 1, p.status, kStatusWaitTimeoutMma)) {
        fed = false;
        break;
      }
      tc_fence_after_sync();
      const uint32_t sx = smem_u32(smem) + it % S::kRing * S::kX;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        tc_mma_f16_ts(tmem, tmem + S::kACol + it % kIgAStages * 32 + k * 8, umma_smem_desc(sx + k * 32, 16, 1024), idesc,
                      it > 0 || k > 0 ? 1u : 0u);
      tc_commit(&empty_bar[it % S::kRing]);
    }
    if (fed) tc_commit(done_bar);
  }
  __syncwarp();

  // All products have retired.  A thread owns one feature; warps 4 to 7 take the second half of the rows.
  const int feature = (warp & 3) * 32 + lane, n = n0 + feature;
  float* part = reinterpret_cast<float*>(smem);  // [row][feature]: the ring is free
  if (p.splits > 1) __syncthreads();
  if (warp < kIgWarps && ok) {
    tc_fence_after_sync();
    const uint32_t taddr = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    constexpr int kStep = BN >= 32 ? 16 : 8;
#pragma unroll 1
    for (int c0 = (warp >> 2) * (BN / 2); c0 < ((warp >> 2) + 1) * (BN / 2); c0 += kStep) {
      if (c0 >= p.M) break;
      uint32_t r[16];
      if constexpr (kStep == 16) tmem_ld_32x16(taddr + c0, r);
      else tmem_ld_32x16(taddr + (c0 & ~15), r);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        if (kStep == 8 && (j >> 3) != (c0 >> 3 & 1)) continue;
        const int row = (kStep == 16 ? c0 : (c0 & ~15)) + j;
        if (row >= p.M) continue;
        float v = __uint_as_float(r[j]);
        if (p.splits > 1) {
          part[row * kIgFeatures + feature] = v;
        } else if (n < p.N) {
          __nv_bfloat16* dst = p.y + row * p.ldy + n;
          if (p.accumulate) v += __bfloat162float(*dst);
          *dst = __float2bfloat16(v);
        }
      }
    }
  }
  if (p.splits > 1) {
    cluster_sync_all();
    if (warp < kIgWarps && ok && n < p.N) {
      for (int row = split + (warp >> 2) * p.splits; row < p.M; row += 2 * p.splits) {
        float v[kIgMaxSplits];
#pragma unroll
        for (int s = 0; s < kIgMaxSplits; ++s)
          v[s] = s < p.splits ? ld_cluster_f32(smem_u32(part) + (row * kIgFeatures + feature) * 4, s) : 0.f;
        float sum = v[0];
#pragma unroll
        for (int s = 1; s < kIgMaxSplits; ++s) sum += v[s];
        __nv_bfloat16* dst = p.y + row * p.ldy + n;
        if (p.accumulate) sum += __bfloat162float(*dst);
        *dst = __float2bfloat16(sum);
      }
    }
    cluster_sync_all();  // a CTA's shared memory outlives its readers
  }
  tc_fence_before_sync();
  const int gave_up = __syncthreads_or(!ok);
  if (warp == kIgWarps) {
    if (gave_up) {
      // A wait gave up: let what may still be in flight land before the CTA exits.
      for (int i = 0; i < 2000; ++i) __nanosleep(1000);
    }
    tc_fence_after_sync();
    tmem_dealloc(tmem, S::kTmemCols);
  }
}

template <int BN>
static int launch_int4_gemm(const Int4GemmParams& p, cudaStream_t stream) {
  using S = Int4GemmCfg<BN>;
  constexpr auto kernel = int4_gemm_kernel<BN>;
  static OptIn opt_in;
  if (!opt_in.done(kernel, S::kSmem)) return -3;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {static_cast<unsigned>(p.splits), 1, 1};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((p.N + kIgFeatures - 1) / kIgFeatures * p.splits));
  cfg.blockDim = dim3(kIgThreads);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p) == cudaSuccess ? 0 : -4;
}

}  // namespace axb

// x [M, K] bf16 with rows of ldx (K, ldx multiples of 8, 16-byte aligned), y [M, N] with rows of ldy; M <= 128.  `splits`:
// slices of K, up to 8 and one for every 64 rows of W at most.
extern "C" int axb_int4_gemm(const void* x, const void* codes, const void* pairs, void* y, int M, int N, int K, int group,
                             int64_t ldx, int64_t ldy, int accumulate, int splits, int* status, cudaStream_t stream) {
  using namespace axb;
  const uintptr_t align = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(pairs);
  if (M < 0 || M > 128 || N < 1 || K < 1 || K % 8 || ldx % 8 || (align & 15) || (group != 64 && group != 128) || splits < 1 ||
      splits > kIgMaxSplits || splits > (K + 63) / 64)
    return -10;
  if (M == 0) return 0;
  const Int4GemmParams p{static_cast<const __nv_bfloat16*>(x), static_cast<const uint8_t*>(codes),
                         static_cast<const uint8_t*>(pairs), static_cast<__nv_bfloat16*>(y), ldx, ldy, M, N, K,
                         group == 64 ? 0 : 1, accumulate, splits, status};
  if (M <= 16) return launch_int4_gemm<16>(p, stream);
  if (M <= 32) return launch_int4_gemm<32>(p, stream);
  if (M <= 64) return launch_int4_gemm<64>(p, stream);
  return launch_int4_gemm<128>(p, stream);
}
