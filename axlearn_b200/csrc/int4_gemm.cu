// y[M, N] = x[M, K] W (+ y) with weights held in 4 bits (layout: int4_linear.cu), on the fifth-generation tensor cores: 128
// features are the M side of the MMA, up to 128 rows of x its N side; more rows are blocks of 128.
//
// Up to eight warps feed: each owns 16 features and turns their codes of 128 rows of W into bf16 values m + s c (one rounding, up
// to 2^-8 of a weight, as in the expansion for the GEMM of more rows), which `tcgen05.st` puts into tensor memory, so that weights
// never pass through shared memory once they are 16 bits wide: writing and reading them there would cost eight times the
// bytes of the codes.  A 16x256b store takes from lane (r, c) the columns 2c, 2c + 1 of every k16 step, 4 rows of W: the word c of
// piece (r, s) of a block for step s.  `ldmatrix` hands out words that way, pieces being rows of its matrices, and x keeps its
// own order over K.  Codes (64-byte swizzle: no bank conflicts), pairs and x come by TMA: with 16-byte `cp.async` by the
// feeding warps the copies alone, about 32 cycles of the load unit for each of a warp, took 80% of the product's time.
//
// Measured (us; the codes at the copy rate): 64 x 4096 x 22016 22.9 (8.3), 64 x 14336 x 4096 17.1 (5.1), 64 x 4096 x 11008 15.5 (4.0),
// 128 x 4096 x 28672 40 (10.8).  A stage of one CTA an SM takes 0.35 us, a feeding warp's chain of waits, words, values and
// store; of two 0.27, by the instructions of both.  So the loop is short: with next codes and values ahead of the waits it
// was as fast or 4% slower, unrolled round the rings half as fast (the instruction caches).  One CTA an SM with sixteen
// feeding warps and clusters that share runs of tiles evenly was 26.2, 18.4 and 36.8.
// Blocks of 128 rows against one expansion and the GEMM: 256 x 4096 x 28672 77 / 121, 512 x 4096 x 4096 20.8 / 24.4, 1024 rows of
// it 40 / 35.
//
// K slices are the CTAs of a cluster; partial sums meet in distributed shared memory in a fixed order.
//
// Launched in the ordinary way in a captured step, too.  In the chain the wait for the predecessor would have to stand ahead of
// the allocation of tensor memory and the successor's start behind its release, since kernels that overlap could otherwise hold the
// tensor memory that each waits for; that has not been built.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "cluster.cuh"
#include "host_utils.cuh"
#include "int4.cuh"
#include "mma_sync.cuh"
#include "sm100.cuh"

namespace axb {

struct Int4GemmParams {
  __nv_bfloat16* y;        // [M, ldy]
  int64_t ldy;
  int M, N, K;
  int accumulate, splits, row_blocks;
  int warps;               // that feed: a tile is 16 features for each
  int* status;
};

constexpr int kIgWarps = 8, kIgThreads = 32 * (kIgWarps + 3), kIgFeatures = 16 * kIgWarps;
constexpr int kIgMaxSplits = 8;

// A stage is 128 rows of W: 64 columns of tensor memory, two 64-column tiles of x, eight warps' codes and pairs.  Codes, on
// their way from memory, have the deepest ring; x comes from the L2.
template <int BN>
struct Int4GemmCfg {
  static constexpr int kRing = BN <= 64 ? 3 : 4;             // places for x and for operands in tensor memory
  static constexpr int kCodeRing = BN <= 16 ? 9 : BN <= 32 ? 7 : BN <= 64 ? 6 : 8;
  static constexpr int kX = BN * 128, kCodes = kIgWarps * 1024, kPairs = kIgWarps * 128;  // bytes: a tile of x, codes, pairs
  static constexpr int kXBytes = kRing * 2 * kX, kCodeBytes = kCodeRing * kCodes;
  static constexpr int kRingBytes = kXBytes + kCodeBytes + kCodeRing * kPairs;
  static constexpr int kSums = BN * kIgFeatures * 4;         // partial sums overlay the rings
  static constexpr int kBody = kRingBytes > kSums ? kRingBytes : kSums;
  static constexpr int kSmem = kBody + 256 + 1024;           // barriers, alignment slack
  static constexpr int kResident = BN <= 64 ? 2 : 1;
  static constexpr int kACol = BN <= 64 ? 64 : 128;
  static constexpr int kTmemCols = BN <= 64 ? 256 : 512;
  static_assert(kACol + kRing * 64 <= kTmemCols, "tensor memory");
  static_assert(kResident * (kSmem + 1024) <= 228 * 1024 && kResident * kTmemCols <= 512, "resident CTAs");
};

// Slot and phase of a ring.
template <int N>
struct IgPlace {
  int slot = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next() {
    if (++slot == N) slot = 0, phase ^= 1;
  }
};

// 16 lanes x 32 columns: thread (r, c) has columns 8 n + 2c, + 1 of lanes r (entries 4 n, 4 n + 1) and r + 8.
__device__ __forceinline__ void tmem_st_16x256(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// The four registers of a word's k16 step: codes as denormal bf16 numbers (`int4.cuh`; the high nibbles are 16 times theirs),
// turned into 2^-37 (m + s c) by one operation.  s0 (s1) carries 2^(133 - 37) (a sixteenth of it), m0 and m1
// 2^-37, so that neither steps up to 2^31 nor values down to 2^-89 leave the range of bf16.
constexpr float kIgStep = 79228162514264337593543950336.f, kIgLow = 1.f / 137438953472.f;  // 2^(133 - 37), 2^-37

__device__ __forceinline__ void ig_values(uint32_t word, __nv_bfloat162 s0, __nv_bfloat162 m0, __nv_bfloat162 s1,
                                          __nv_bfloat162 m1, uint32_t* v) {
  const uint32_t next = word >> 8;
  auto value = [](uint32_t u, __nv_bfloat162 s, __nv_bfloat162 m) {
    const __nv_bfloat162 x = __hfma2(reinterpret_cast<__nv_bfloat162&>(u), s, m);
    return reinterpret_cast<const uint32_t&>(x);
  };
  v[0] = value(int4_low(word), s0, m0);
  v[1] = value(int4_low(next), s0, m0);
  v[2] = value(int4_high(word), s1, m1);
  v[3] = value(int4_high(next), s1, m1);
}

// kGroup: 64 or 128.
template <int BN, int kGroup>
__global__ void __launch_bounds__(kIgThreads, Int4GemmCfg<BN>::kResident)
int4_gemm_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_codes,
                 const __grid_constant__ CUtensorMap map_pairs, Int4GemmParams p) {
  using S = Int4GemmCfg<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem =
      reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + S::kBody);
  uint64_t* empty_bar = full_bar + S::kRing;
  uint64_t* code_full = empty_bar + S::kRing;
  uint64_t* code_empty = code_full + S::kCodeRing;
  uint64_t* done_bar = code_empty + S::kCodeRing;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done_bar + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // Blocks of rows of one tile run side by side: its codes come from memory once.
  const int split = static_cast<int>(blockIdx.x) % p.splits, block = static_cast<int>(blockIdx.x) / p.splits;
  const int row0 = block % p.row_blocks * BN, n0 = block / p.row_blocks * (16 * p.warps);
  const int rows = min(p.M - row0, BN);
  const int k128 = (p.K + 127) / 128;
  const int kb_lo = split * k128 / p.splits, count = (split + 1) * k128 / p.splits - kb_lo;

  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kRing; ++i) {
      mbar_init(&full_bar[i], p.warps + 1);
      mbar_init(&empty_bar[i], 1);
    }
    for (int i = 0; i < S::kCodeRing; ++i) {
      mbar_init(&code_full[i], 1);
      mbar_init(&code_empty[i], p.warps);
    }
    mbar_init(done_bar, 1);
    fence_barrier_init();
  }
  constexpr int kXWarp = kIgWarps, kCodeWarp = kIgWarps + 1, kMmaWarp = kIgWarps + 2;
  if (warp == kMmaWarp) {
    tmem_alloc(tmem_slot, S::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;

  constexpr int kPairBytes = kGroup == 64 ? 128 : 64;  // of a stage and 16 features
  bool ok = true;
  if (warp < kIgWarps) {
    // Features 16 warp .. + 15 of the tile are the tensor-memory lanes from 32 (warp % 4) + 16 (warp / 4) on.
    const uint32_t a_addr = tmem + (static_cast<uint32_t>((warp & 3) * 32 + (warp >> 2) * 16) << 16) + S::kACol;
    const int r = lane >> 2;
    // Row lane % 8 of matrix lane / 8: the copy swaps 16-byte units as the 64-byte swizzle does.
    const uint8_t* mine = smem + S::kXBytes + warp * 1024 + (lane & 7) * 64 + (((lane >> 3) ^ (lane >> 1 & 3)) << 4);
    const uint8_t* mine_pairs = smem + S::kXBytes + S::kCodeBytes + warp * kPairBytes + r * 8;
    IgPlace<S::kCodeRing> code;
    const int mine_count = warp < p.warps ? count : 0;
    IgPlace<S::kRing> a;
#pragma unroll 1
    for (int it = 0; ok && it < mine_count; ++it) {
      ok = mbar_wait_warp(&code_full[code.slot], code.phase, p.status, kStatusWaitTimeoutProducer);
      if (!ok) break;
      if (it >= S::kRing) {
        ok = mbar_wait_warp(&empty_bar[a.slot], a.phase ^ 1, p.status, kStatusWaitTimeoutProducer);
        if (!ok) break;
        tc_fence_after_sync();
      }
      __nv_bfloat162 s0, m0, s1, m1;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        if (half == 0 || kGroup == 64) {
          const uint2 pair = *reinterpret_cast<const uint2*>(mine_pairs + code.slot * S::kPairs + half * 64);
          const __nv_bfloat162 pa = reinterpret_cast<const __nv_bfloat162&>(pair.x),
                               pb = reinterpret_cast<const __nv_bfloat162&>(pair.y), low = __float2bfloat162_rn(kIgLow);
          s0 = __hmul2(__low2bfloat162(pa), __float2bfloat162_rn(kIgStep)), m0 = __hmul2(__high2bfloat162(pa), low);
          s1 = __hmul2(__low2bfloat162(pb), __float2bfloat162_rn(kIgStep / 16.f)), m1 = __hmul2(__high2bfloat162(pb), low);
        }
        uint32_t w[4], v[16];
        ldsm4(w, mine + code.slot * S::kCodes + half * 512);
#pragma unroll
        for (int q = 0; q < 4; ++q) ig_values(w[q], s0, m0, s1, m1, v + 4 * q);
        tmem_st_16x256(a_addr + a.slot * 64 + half * 32, v);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&code_empty[code.slot]);
      code.next();
      tmem_st_wait();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&full_bar[a.slot]);
      a.next();
    }
    if (ok) ok = mbar_wait_warp(done_bar, 0, p.status, kStatusWaitTimeoutEpilogue);
  } else if (warp == kXWarp) {
    if (elect_one()) {
      IgPlace<S::kRing> x;
#pragma unroll 1
      for (int it = 0; it < count; ++it) {
        if (it >= S::kRing && !mbar_wait(&empty_bar[x.slot], x.phase ^ 1, p.status, kStatusWaitTimeoutProducer)) break;
        uint8_t* tile = smem + x.slot * (2 * S::kX);
        mbar_arrive_expect_tx(&full_bar[x.slot], 2 * S::kX);
        tma_load_2d(tile, &map_x, &full_bar[x.slot], (kb_lo + it) * 128, row0);
        tma_load_2d(tile + S::kX, &map_x, &full_bar[x.slot], (kb_lo + it) * 128 + 64, row0);
        x.next();
      }
    }
  } else if (warp == kCodeWarp) {
    if (elect_one()) {
      IgPlace<S::kCodeRing> code;
#pragma unroll 1
      for (int it = 0; it < count; ++it) {
        if (it >= S::kCodeRing && !mbar_wait(&code_empty[code.slot], code.phase ^ 1, p.status, kStatusWaitTimeoutProducer)) break;
        mbar_arrive_expect_tx(&code_full[code.slot], p.warps * (1024 + kPairBytes));
        tma_load_3d(smem + S::kXBytes + code.slot * S::kCodes, &map_codes, &code_full[code.slot], 0, (kb_lo + it) * 16, n0 / 16);
        tma_load_2d(smem + S::kXBytes + S::kCodeBytes + code.slot * S::kPairs, &map_pairs, &code_full[code.slot],
                    (kb_lo + it) * kPairBytes, n0 / 16);
        code.next();
      }
    }
  } else if (elect_one()) {
    constexpr uint32_t idesc = umma_idesc_f16(kIgFeatures, BN, 1, 1, 0, 0);
    bool fed = true;
    IgPlace<S::kRing> at;
#pragma unroll 1
    for (int it = 0; it < count; ++it) {
      if (!mbar_wait(&full_bar[at.slot], at.phase, p.status, kStatusWaitTimeoutMma)) {
        fed = false;
        break;
      }
      tc_fence_after_sync();
      const uint32_t sx = smem_u32(smem) + at.slot * (2 * S::kX), sa = tmem + S::kACol + at.slot * 64;
#pragma unroll
      for (int k = 0; k < 8; ++k)
        tc_mma_f16_ts(tmem, sa + k * 8, umma_smem_desc(sx + (k >> 2) * S::kX + (k & 3) * 32, 16, 1024), idesc,
                      it > 0 || k > 0 ? 1u : 0u);
      tc_commit(&empty_bar[at.slot]);
      at.next();
    }
    if (fed) tc_commit(done_bar);
  }
  __syncwarp();

  // All products have retired.  A thread owns one lane of tensor memory; warps 4 to 7 take the second half of the rows.
  const int feature = (warp & 3) * 32 + lane, n = n0 + 16 * ((warp & 3) + (lane >> 4) * 4) + (lane & 15);
  const bool there = n < min(p.N, n0 + 16 * p.warps);
  float* part = reinterpret_cast<float*>(smem);  // [row][lane]: the ring is free
  if (p.splits > 1) __syncthreads();
  if (warp < kIgWarps && ok) {
    tc_fence_after_sync();
    const uint32_t taddr = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    constexpr int kStep = BN >= 32 ? 16 : 8;
#pragma unroll 1
    for (int c0 = (warp >> 2) * (BN / 2); c0 < ((warp >> 2) + 1) * (BN / 2); c0 += kStep) {
      if (c0 >= rows) break;
      uint32_t r[16];
      if constexpr (kStep == 16) tmem_ld_32x16(taddr + c0, r);
      else tmem_ld_32x16(taddr + (c0 & ~15), r);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        if (kStep == 8 && (j >> 3) != (c0 >> 3 & 1)) continue;
        const int row = (kStep == 16 ? c0 : (c0 & ~15)) + j;
        if (row >= rows) continue;
        float v = __uint_as_float(r[j]) * (1.f / kIgLow);
        if (p.splits > 1) {
          part[row * kIgFeatures + feature] = v;
        } else if (there) {
          __nv_bfloat16* dst = p.y + (row0 + row) * p.ldy + n;
          if (p.accumulate) v += __bfloat162float(*dst);
          *dst = __float2bfloat16(v);
        }
      }
    }
  }
  if (p.splits > 1) {
    cluster_sync_all();
    if (warp < kIgWarps && ok && there) {
      for (int row = split + (warp >> 2) * p.splits; row < rows; row += 2 * p.splits) {
        float v[kIgMaxSplits];
#pragma unroll
        for (int s = 0; s < kIgMaxSplits; ++s)
          v[s] = s < p.splits ? ld_cluster_f32(smem_u32(part) + (row * kIgFeatures + feature) * 4, s) : 0.f;
        float sum = v[0];
#pragma unroll
        for (int s = 1; s < kIgMaxSplits; ++s) sum += v[s];
        __nv_bfloat16* dst = p.y + (row0 + row) * p.ldy + n;
        if (p.accumulate) sum += __bfloat162float(*dst);
        *dst = __float2bfloat16(sum);
      }
    }
    cluster_sync_all();  // a CTA's shared memory outlives its readers
  }
  tc_fence_before_sync();
  const int gave_up = __syncthreads_or(!ok);
  if (warp == kMmaWarp) {
    if (gave_up) {
      // A wait gave up: let what may still be in flight land before the CTA exits.
      for (int i = 0; i < 2000; ++i) __nanosleep(1000);
    }
    tc_fence_after_sync();
    tmem_dealloc(tmem, S::kTmemCols);
  }
}

template <int BN, int kGroup>
static int launch_int4_gemm(const void* x, int64_t ldx, const void* codes, const void* pairs, const Int4GemmParams& p,
                            cudaStream_t stream) {
  using S = Int4GemmCfg<BN>;
  constexpr auto kernel = int4_gemm_kernel<BN, kGroup>;
  static OptIn opt_in;
  if (!opt_in.done(kernel, S::kSmem)) return -3;
  CUtensorMap map_x, map_codes, map_pairs;
  const uint64_t n16 = (p.N + 15) / 16, k128 = (p.K + 127) / 128, pair_bytes = kGroup == 64 ? 128 : 64;
  const uint64_t x_dims[2] = {static_cast<uint64_t>(p.K), static_cast<uint64_t>(p.M)}, x_stride[1] = {static_cast<uint64_t>(ldx) * 2};
  const uint32_t x_box[2] = {64, BN};
  const uint64_t code_dims[3] = {64, k128 * 16, n16}, code_strides[2] = {64, k128 * 1024};
  const uint32_t warps = static_cast<uint32_t>(p.warps), code_box[3] = {64, 16, warps};
  const uint64_t pair_dims[2] = {k128 * pair_bytes, n16}, pair_stride[1] = {k128 * pair_bytes};
  const uint32_t pair_box[2] = {static_cast<uint32_t>(pair_bytes), warps};
  if (make_tensor_map(&map_x, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, x, x_dims, x_stride, x_box, CU_TENSOR_MAP_SWIZZLE_128B) != 0 ||
      make_tensor_map(&map_codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, codes, code_dims, code_strides, code_box,
                      CU_TENSOR_MAP_SWIZZLE_64B) != 0 ||
      make_tensor_map(&map_pairs, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, pairs, pair_dims, pair_stride, pair_box,
                      CU_TENSOR_MAP_SWIZZLE_NONE) != 0)
    return -2;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {static_cast<unsigned>(p.splits), 1, 1};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((p.N + 16 * p.warps - 1) / (16 * p.warps) * p.row_blocks * p.splits));
  cfg.blockDim = dim3(kIgThreads);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, map_x, map_codes, map_pairs, p) == cudaSuccess ? 0 : -4;
}

template <int kGroup>
static int int4_gemm(const void* x, int64_t ldx, const void* codes, const void* pairs, const Int4GemmParams& p, cudaStream_t stream) {
  if (p.M <= 16) return launch_int4_gemm<16, kGroup>(x, ldx, codes, pairs, p, stream);
  if (p.M <= 32) return launch_int4_gemm<32, kGroup>(x, ldx, codes, pairs, p, stream);
  if (p.M <= 64) return launch_int4_gemm<64, kGroup>(x, ldx, codes, pairs, p, stream);
  return launch_int4_gemm<128, kGroup>(x, ldx, codes, pairs, p, stream);
}

}  // namespace axb

// x [M, K] bf16 with rows of ldx (K, ldx multiples of 8, 16-byte aligned), y [M, N] with rows of ldy; M <= 65536.  `splits`:
// slices of K, up to 8 and one for every 128 rows of W at most.
extern "C" int axb_int4_gemm(const void* x, const void* codes, const void* pairs, void* y, int M, int N, int K, int group,
                             int64_t ldx, int64_t ldy, int accumulate, int warps, int splits, int* status, cudaStream_t stream) {
  using namespace axb;
  const uintptr_t align = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(pairs);
  if (M < 0 || M > 65536 || N < 1 || K < 1 || K % 8 || ldx % 8 || (align & 15) || (group != 64 && group != 128) || warps < 1 ||
      warps > kIgWarps || splits < 1 || splits > kIgMaxSplits || splits > (K + 127) / 128)
    return -10;
  if (M == 0) return 0;
  const Int4GemmParams p{static_cast<__nv_bfloat16*>(y), ldy, M, N, K, accumulate, splits, (M + 127) / 128, warps, status};
  return group == 64 ? int4_gemm<64>(x, ldx, codes, pairs, p, stream) : int4_gemm<128>(x, ldx, codes, pairs, p, stream);
}
