// y[M, N] = x[M, K] W (+ y) for up to 128 rows with weights held in 4 bits (layout: int4_linear.cu), on the fifth-generation
// tensor cores: 128 features are the M side of the MMA, the rows of x its N side.
//
// Eight warps feed: each owns 16 features and turns their codes of 128 rows of W into bf16 values m + s c (one rounding, 2^-9
// of a weight, as in the expansion for the GEMM of more rows), which `tcgen05.st` puts into tensor memory -- a lane's words
// are the fragment of the 16x256b shape as they lie --, so that weights never pass through shared memory once they are 16
// bits wide: writing and reading them there would cost eight times the bytes of the codes.  Other warps bring x, 128 columns
// of it at a time, to shared memory in the order in which the codes run over K, and one issues the MMAs.
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
  int M, N, K;
  int accumulate, splits;
  int* status;
};

constexpr int kIgWarps = 8, kIgFeatures = 16 * kIgWarps;
constexpr int kIgMaxSplits = 8;

// A stage is 128 rows of W: 64 columns of tensor memory, two 64-column tiles of x, eight warps' codes and pairs.  Codes, on
// their way from memory, have the deepest ring; x comes from the L2.
template <int BN>
struct Int4GemmCfg {
  static constexpr int kXRing = BN == 64 ? 3 : 4;            // each place has a warp of its own
  static constexpr int kThreads = 32 * (kIgWarps + kXRing + 1);
  static constexpr int kCodeRing = BN <= 16 ? 9 : BN <= 32 ? 7 : BN <= 64 ? 6 : 8;
  static constexpr int kX = BN * 128, kCodes = 1024 + 128;   // bytes of a tile of x; of a warp's codes and pairs
  static constexpr int kXBytes = kXRing * 2 * kX;
  static constexpr int kRingBytes = kXBytes + kCodeRing * kIgWarps * kCodes;
  static constexpr int kSums = BN * kIgFeatures * 4;         // partial sums overlay the rings
  static constexpr int kBody = kRingBytes > kSums ? kRingBytes : kSums;
  static constexpr int kSmem = kBody + 256 + 1024;           // barriers, alignment slack
  static constexpr int kResident = BN <= 64 ? 2 : 1;
  static constexpr int kACol = BN <= 64 ? 64 : 128, kARing = BN <= 64 ? 3 : 4;
  static constexpr int kTmemCols = BN <= 64 ? 256 : 512;
  static_assert(kACol + kARing * 64 <= kTmemCols, "tensor memory");
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

// The four registers of a word's k16 step: codes as denormal bf16 numbers (`int4.cuh`; the high nibbles are 16 times theirs),
// turned into 2^-kIgDown (m + s c) by one operation.  s0 (s1) carries 2^(133 - kIgDown) (a sixteenth of it), m0 and m1
// 2^-kIgDown, so that neither steps up to 2^31 nor values down to 2^-89 leave the range of bf16.
constexpr int kIgDown = 37;
constexpr float kIgStep = 79228162514264337593543950336.f, kIgLow = 1.f / 137438953472.f;  // 2^(133 - kIgDown), 2^-kIgDown

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
__global__ void __launch_bounds__(Int4GemmCfg<BN>::kThreads, Int4GemmCfg<BN>::kResident)
int4_gemm_kernel(Int4GemmParams p) {
  using S = Int4GemmCfg<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem =
      reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* x_full = reinterpret_cast<uint64_t*>(smem + S::kBody);
  uint64_t* x_empty = x_full + S::kXRing;
  uint64_t* a_full = x_empty + S::kXRing;
  uint64_t* a_empty = a_full + S::kARing;
  uint64_t* done_bar = a_empty + S::kARing;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done_bar + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = static_cast<int>(blockIdx.x) % p.splits;
  const int n0 = static_cast<int>(blockIdx.x) / p.splits * kIgFeatures;
  const int k128 = (p.K + 127) / 128;
  const int kb_lo = split * k128 / p.splits, count = (split + 1) * k128 / p.splits - kb_lo;

  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kXRing; ++i) {
      mbar_init(&x_full[i], 1);
      mbar_init(&x_empty[i], 1);
    }
    for (int i = 0; i < S::kARing; ++i) {
      mbar_init(&a_full[i], kIgWarps);
      mbar_init(&a_empty[i], 1);
    }
    mbar_init(done_bar, 1);
    fence_barrier_init();
  }
  constexpr int kMmaWarp = kIgWarps + S::kXRing;
  if (warp == kMmaWarp) {
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
    const int64_t block = static_cast<int64_t>(have ? tile : 0) * k128 + kb_lo;
    const uint8_t* codes = p.codes + block * 1024 + lane * 16;
    constexpr int kPairBytes = kGroup == 64 ? 128 : 64;  // of a stage
    const uint8_t* pairs = p.pairs + block * kPairBytes + lane * 16;
    constexpr int kStride = kIgWarps * S::kCodes;        // of a stage in the ring
    const uint8_t* own = smem + S::kXBytes + warp * S::kCodes;
    const uint32_t dst0 = smem_u32(own) + lane * 16;
    uint32_t dst = dst0;
    auto load = [&] {  // the next stage
      ig_copy(dst, codes, have);
      ig_copy(dst + 512, codes + 512, have);
      if (lane * 16 < kPairBytes) ig_copy(dst + 1024, pairs, have);
      codes += 1024;
      pairs += kPairBytes;
      dst += kStride;
      if (dst == dst0 + S::kCodeRing * kStride) dst = dst0;
    };
#pragma unroll 1
    for (int it = 0; it < S::kCodeRing; ++it) {
      if (it < count) load();
      cp_commit();
    }
    IgPlace<S::kCodeRing> code;
    IgPlace<S::kARing> a;
#pragma unroll 1
    for (int it = 0; it < count; ++it) {
      if (it >= S::kARing) {
        ok = mbar_wait_warp(&a_empty[a.slot], a.phase ^ 1, p.status, kStatusWaitTimeoutProducer);
        if (!ok) break;
        tc_fence_after_sync();
      }
      cp_wait_group<S::kCodeRing - 1>();
      __syncwarp();
      const uint8_t* mine = own + code.slot * kStride;
      const uint32_t a_stage_addr = a_addr + a.slot * 64;
      __nv_bfloat162 s0, m0, s1, m1;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint4 w = *reinterpret_cast<const uint4*>(mine + half * 512 + lane * 16);
        if (half == 0 || kGroup == 64) {
          const uint2 u = *reinterpret_cast<const uint2*>(mine + 1024 + half * 64 + (lane >> 2) * 8);
          const __nv_bfloat162 pa = reinterpret_cast<const __nv_bfloat162&>(u.x), pb = reinterpret_cast<const __nv_bfloat162&>(u.y);
          const __nv_bfloat162 low = __float2bfloat162_rn(kIgLow);
          s0 = __hmul2(__low2bfloat162(pa), __float2bfloat162_rn(kIgStep)), m0 = __hmul2(__high2bfloat162(pa), low);
          s1 = __hmul2(__low2bfloat162(pb), __float2bfloat162_rn(kIgStep / 16.f)), m1 = __hmul2(__high2bfloat162(pb), low);
        }
        uint32_t v[16];
        ig_values(w.x, s0, m0, s1, m1, v);
        ig_values(w.y, s0, m0, s1, m1, v + 4);
        ig_values(w.z, s0, m0, s1, m1, v + 8);
        ig_values(w.w, s0, m0, s1, m1, v + 12);
        tmem_st_16x256(a_stage_addr + half * 32, v);
      }
      tmem_st_wait();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&a_full[a.slot]);
      if (it + S::kCodeRing < count) load();  // into the place that has been read
      cp_commit();
      code.next();
      a.next();
    }
    cp_wait_all();
    if (ok) ok = mbar_wait_warp(done_bar, 0, p.status, kStatusWaitTimeoutEpilogue);
  } else if (warp < kMmaWarp) {
    // x: 16-byte pieces (row, h, i), tile h of 2 and i of 8: columns 64 h + 16 c + 8 q + 0 .. 7 with c = i / 2, q = i % 2.
    // Their halves go to places 4c .. 4c + 3 of the k16 steps 2q and 2q + 1, where the codes of these columns are.  A warp fills
    // one place of the ring, a lane the pieces (h, i) of every second row.
    constexpr int kMine = BN / 2;
    const int place = warp - kIgWarps;
    const int i = lane & 7, h = lane >> 3 & 1, row0 = lane >> 4;
    const int c = i >> 1, q = i & 1, unit = 4 * q + (c >> 1);  // of 16 bytes; the second half's is two further
    const int column = (kb_lo + place) * 128 + h * 64 + c * 16 + q * 8;
    const __nv_bfloat16* src = p.x + row0 * p.ldx + column;
    int left = p.K - column;                                   // columns from this piece on
    const int rows = min(kMine, (p.M - row0 + 1) / 2);         // of this lane
    const uint32_t at = smem_u32(smem) + place * (2 * S::kX) + h * S::kX + row0 * 128 + (c & 1) * 8;
    uint32_t phase = 1;
#pragma unroll 1
    for (int it = place; it < count; it += S::kXRing) {
      if (it >= S::kXRing) {
        ok = mbar_wait_warp(&x_empty[place], phase, p.status, kStatusWaitTimeoutProducer);
        if (!ok) break;
      }
      phase ^= 1;
      const int there = left > 0 ? rows : 0;
      const __nv_bfloat16* from = src;
#pragma unroll 8
      for (int j = 0; j < kMine; ++j) {
        // Rows of the lane are two apart: the swizzle takes the row mod 8.
        const uint32_t to = at + j * 256 + ((unit ^ ((row0 + 2 * j) & 7)) << 4);
        const __nv_bfloat16* piece = j < there ? from : p.x;
        ig_copy8(to, piece, j < there);
        ig_copy8(to ^ 32, piece + 4, j < there);  // two units further: bit 1 of the unit is 0, swapped or not
        from += 2 * p.ldx;
      }
      src += S::kXRing * 128;
      left -= S::kXRing * 128;
      cp_wait_all();
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&x_full[place]);
    }
  } else if (elect_one()) {
    constexpr uint32_t idesc = umma_idesc_f16(kIgFeatures, BN, 1, 1, 0, 0);
    bool fed = true;
    IgPlace<S::kXRing> x;
    IgPlace<S::kARing> a;
#pragma unroll 1
    for (int it = 0; it < count; ++it) {
      if (!mbar_wait(&x_full[x.slot], x.phase, p.status, kStatusWaitTimeoutMma) ||
          !mbar_wait(&a_full[a.slot], a.phase, p.status, kStatusWaitTimeoutMma)) {
        fed = false;
        break;
      }
      tc_fence_after_sync();
      const uint32_t sx = smem_u32(smem) + x.slot * (2 * S::kX), sa = tmem + S::kACol + a.slot * 64;
#pragma unroll
      for (int k = 0; k < 8; ++k)
        tc_mma_f16_ts(tmem, sa + k * 8, umma_smem_desc(sx + (k >> 2) * S::kX + (k & 3) * 32, 16, 1024), idesc,
                      it > 0 || k > 0 ? 1u : 0u);
      tc_commit(&x_empty[x.slot]);
      tc_commit(&a_empty[a.slot]);
      x.next();
      a.next();
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
        float v = __uint_as_float(r[j]) * (1.f / kIgLow);
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
static int launch_int4_gemm(const Int4GemmParams& p, cudaStream_t stream) {
  using S = Int4GemmCfg<BN>;
  constexpr auto kernel = int4_gemm_kernel<BN, kGroup>;
  static OptIn opt_in;
  if (!opt_in.done(kernel, S::kSmem)) return -3;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {static_cast<unsigned>(p.splits), 1, 1};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((p.N + kIgFeatures - 1) / kIgFeatures * p.splits));
  cfg.blockDim = dim3(S::kThreads);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p) == cudaSuccess ? 0 : -4;
}

template <int kGroup>
static int int4_gemm(const Int4GemmParams& p, cudaStream_t stream) {
  if (p.M <= 16) return launch_int4_gemm<16, kGroup>(p, stream);
  if (p.M <= 32) return launch_int4_gemm<32, kGroup>(p, stream);
  if (p.M <= 64) return launch_int4_gemm<64, kGroup>(p, stream);
  return launch_int4_gemm<128, kGroup>(p, stream);
}

}  // namespace axb

// x [M, K] bf16 with rows of ldx (K, ldx multiples of 8, 16-byte aligned), y [M, N] with rows of ldy; M <= 128.  `splits`:
// slices of K, up to 8 and one for every 128 rows of W at most.
extern "C" int axb_int4_gemm(const void* x, const void* codes, const void* pairs, void* y, int M, int N, int K, int group,
                             int64_t ldx, int64_t ldy, int accumulate, int splits, int* status, cudaStream_t stream) {
  using namespace axb;
  const uintptr_t align = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(pairs);
  if (M < 0 || M > 128 || N < 1 || K < 1 || K % 8 || ldx % 8 || (align & 15) || (group != 64 && group != 128) || splits < 1 ||
      splits > kIgMaxSplits || splits > (K + 127) / 128)
    return -10;
  if (M == 0) return 0;
  const Int4GemmParams p{static_cast<const __nv_bfloat16*>(x), static_cast<const uint8_t*>(codes),
                         static_cast<const uint8_t*>(pairs), static_cast<__nv_bfloat16*>(y), ldx, ldy, M, N, K,
                         accumulate, splits, status};
  return group == 64 ? int4_gemm<64>(p, stream) : int4_gemm<128>(p, stream);
}
