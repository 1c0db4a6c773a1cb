// Skinny bf16 GEMM for sm_100a: C[M, N] = X[M, K] * W[K, N] (+ C) with M <= 128 -- the products of a decoding
// step and of short prompts.  Every weight byte is used once, so the bound is the rate at which W comes
// out of HBM; the shape of the kernel follows from that:
//
//   * operands are swapped: 128 output FEATURES are the M side of the tcgen05 tile and the (16 .. 128) rows of X
//     its N side, so a pipeline stage is 16 KB of weights and 2 KB of X per 16 rows, not 16 KB of mostly
//     zero-filled X rows beside 8 KB of weights (the 128-row tile of gemm.cu);
//   * two CTAs fit one SM (<= 113 KB each), so about 190 KB of weights per SM are on their way at any time and the
//     prologue / epilogue of one CTA runs under the stream of the other;
//   * the K slices of a tile are the CTAs of one cluster: partial sums meet through distributed shared
//     memory (no fp32 workspace in global memory, no counters, no fence), each CTA finishing every
//     split-th row of X in a fixed order, so results are reproducible.
//
// Warp 0 streams tiles with TMA, one thread of warp 1 issues the MMAs, warps 2-5 read the accumulator (thread =
// feature, so a warp stores 32 neighbouring features of a row).  Either layout of W is read in place.
//
// In a chain of small products neither HBM nor the L2 is the bound (1 x 2048 x 2048 took 4.8 us with its weights in HBM
// and 4.6 with them in the L2) but what a launch does one after the other, so for up to 32 rows:
//   * a stage is two k-blocks (up to 16 rows): the thread that issues the MMAs spends 40 clocks on each and about 110
//     on a stage's wait and commit; a stage that is not filled again is not committed;
//   * partial sums are stored into the inbox of the CTA that finishes their row (behind the stages), which then reads
//     its own shared memory: one cluster barrier behind the products and no round trip between SMs, where fetching them
//     took both and a second barrier (2.0 -> 1.0 us);
//   * C is read while the products run, and no CTA looks at the status word in memory before it leaves (0.6 us).
//
// us, chained launches with weights from HBM, before these / now, the weights alone at 6.55 TB/s in brackets:
//   1 x 512 x 2048    4.5 /  3.4 (0.3)     1 x 2048 x 2048  4.8 /  3.6 (1.3)     1 x 2048 x 8192  9.0 / 7.7 (5.1)
//   1 x 16384 x 2048 12.7 / 11.3 (10.2)   16 x 4096 x 4096  9.4 /  7.9 (5.1)    16 x 4096 x 14336 22.8 / 19.9 (17.9)
// Separate launches, this file's first form (64-column tiles with a split-K workspace before it in brackets) and the
// library:
//  16 x 28672 x 4096 37.0 (38.8) / 37.1    64 x 4096 x 11008 21.1 (26.4) / 18.1   64 x 32768 x 4096 49.2 (49.4) / 46.8
// Half tiles (64 features, twice the CTAs) were no faster: an MMA costs its issuer the same 40 clocks.
#include <atomic>

#include "chain.cuh"
#include "cluster.cuh"
#include "host_utils.cuh"
#include "int8.cuh"
#include "opt_in.cuh"
#include "sm100.cuh"

namespace axb {

constexpr int kSkTile = 128;  // features of one MMA
constexpr int kSkRow = 128;  // bytes of a k-block in a row of either operand: 64 bf16 or 128 8-bit values
constexpr int kSkThreads = 192;
constexpr int kSkMaxSplit = 8;  // portable cluster size

// BN rows of X; `LAYOUT`: how a CTA fills its SM.
//   kPair  one 128-feature tile, half an SM's shared memory: two CTAs per SM;
//   kDeep  one tile, the whole SM: twice the stages in flight, for grids of at most one CTA per SM;
//   kWide  two tiles side by side, the whole SM: 512 contiguous bytes per K row of an N-major W where one tile has 256;
//   kEven  8-bit operands in place of kWide: two tiles of which the second has as few features as spread N evenly over the SMs (us
//          kPair / kWide / kEven: 1 x 4096 x 19200 21.0 19.1 16.3, x 22016 21.8 20.2 18.7, x 28672 24.1 23.0 22.4; 64 rows of these
//          25.5 20.5 19.6, 26.5 22.3 21.4, 28.8 25.7 25.8).
enum SkinnyLayout { kPair, kDeep, kWide, kEven };

template <int BN, SkinnyLayout LAYOUT>
struct SkinnyCfg {
  static constexpr int kTiles = LAYOUT == kWide || LAYOUT == kEven ? 2 : 1;
  static constexpr int kFeatures = kTiles * kSkTile;  // (kEven: at most)
  static constexpr int kWBytes = kFeatures * kSkRow;
  static constexpr int kXBytes = BN * kSkRow;
  static constexpr int kBlockBytes = kWBytes + kXBytes;
  static constexpr int kBlocks = (LAYOUT == kPair ? 110 * 1024 : 200 * 1024) / kBlockBytes;
  // A stage, the unit of waits and commits, is one or two k-blocks.
  static constexpr int kGroup = BN <= 16 && LAYOUT != kEven ? 2 : 1;
  // Stages of kEven: MMAs read the second tile's 128 rows whole, also in the last stage, and what lies behind its features makes
  // sums that nobody reads.
  static constexpr int kEvenRing = 200 * 1024, kEvenLeast = kSkTile + 8;
  __host__ __device__ static constexpr int even_stages(int features) {
    const int block = features * kSkRow + kXBytes;
    return (kEvenRing - (block > kWBytes ? block : kWBytes)) / block + 1;
  }
  static constexpr int kStages = LAYOUT == kEven ? even_stages(kEvenLeast) : kBlocks / kGroup;
  // A split tile of few rows receives the other slices' partial sums behind the stages: [slice][own row][feature].
  static constexpr bool kPush = kTiles == 1 && BN <= 32;
  static constexpr int kInboxBytes = kPush ? (BN + kSkMaxSplit - 1) * kSkTile * 4 : 0;
  static constexpr int kSplitStages = kPush ? (kBlocks * kBlockBytes - kInboxBytes) / (kGroup * kBlockBytes) : kStages;
  static constexpr int kRingBytes = LAYOUT == kEven ? kEvenRing : kBlocks * kBlockBytes;
  static constexpr int kSmem = kRingBytes + 512 + 1024;  // barriers, alignment slack
  static constexpr int kResident = LAYOUT == kPair ? 2 : 1;
  static constexpr int kTmemCols = kTiles * BN < 32 ? 32 : kTiles * BN;
  static_assert(kResident * (kSmem + 1024) <= 228 * 1024 && kSmem <= 227 * 1024, "resident CTAs per SM");
  static_assert(kSplitStages >= 2, "a ring");
  static_assert(kTiles > 1 || kPush || BN * kSkTile * 4 <= kRingBytes, "partial sums reuse the stages");
};

struct SkinnyGemmParams {
  int M, N, K;
  void* C;
  int64_t ldc;
  int* status;
  int accumulate;
  int split;
  int w_resident;  // in a chained launch: nothing that runs just before this kernel writes W
  const float *x_scales, *w_scales;  // 8-bit operands: of the rows of X and of the features
  int features;                      // kEven: of a CTA, a multiple of 8
};

// Operands in 8 bits (`int8_t`) are products of whole numbers in 32-bit integers, exact in any order; a sum counts times the
// scale of its row and of its feature.  Everything up to there moves the same bytes as bf16 operands of half the K.
template <typename In>
struct SkinnyIn {
  static constexpr bool kWhole = sizeof(In) == 1;
  static constexpr int kK = kSkRow / static_cast<int>(sizeof(In));  // values of a k-block
  static constexpr CUtensorMapDataType kType = kWhole ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;

  static __device__ __forceinline__ constexpr uint32_t idesc(int n, int w_mn, int x_mn) {
    return kWhole ? umma_idesc_i8(kSkTile, n) : umma_idesc_f16(kSkTile, n, 1, 1, w_mn, x_mn);
  }
  static __device__ __forceinline__ void mma(uint32_t d, uint64_t w, uint64_t x, uint32_t idesc, uint32_t accumulate) {
    if constexpr (kWhole) tc_mma_i8(d, w, x, idesc, accumulate);
    else tc_mma_f16(d, w, x, idesc, accumulate);
  }
  // Bits of a partial sum that stand for zero in both forms; the sum of two.
  static __device__ __forceinline__ float add(float a, float b) {
    if constexpr (kWhole) return __int_as_float(__float_as_int(a) + __float_as_int(b));
    else return a + b;
  }
  static __device__ __forceinline__ float value(float sum, float x_scale, float w_scale) {
    if constexpr (kWhole) return __int2float_rn(__float_as_int(sum)) * x_scale * w_scale;
    else return sum;
  }
};

template <typename OutT>
__device__ __forceinline__ float skinny_read(const OutT* src) {
  if constexpr (sizeof(OutT) == 2) return __bfloat162float(*src);
  else return *src;
}

template <typename OutT>
__device__ __forceinline__ void skinny_write(OutT* dst, float v) {
  if constexpr (sizeof(OutT) == 2) *dst = __float2bfloat16(v);
  else *dst = v;
}

__device__ __forceinline__ float ld_shared_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}

template <int BN, SkinnyLayout LAYOUT, bool X_MN, bool W_MN, typename OutT, typename In>
__global__ void __launch_bounds__(kSkThreads, LAYOUT == kPair ? 2 : 1)
gemm_skinny_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x,
                   SkinnyGemmParams p) {
  using S = SkinnyCfg<BN, LAYOUT>;
  using I = SkinnyIn<In>;
  static_assert(!I::kWhole || (!X_MN && !W_MN), "8-bit operands are read along K");
  static_assert(I::kWhole ? LAYOUT != kWide : LAYOUT != kEven, "two tiles");
  constexpr int kGroup = S::kGroup, kSkK = I::kK;
  extern __shared__ uint8_t smem_raw[];
  __shared__ float x_scales[I::kWhole ? BN : 1];  // read by the epilogue while the products run
  uint8_t* smem =
      reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + S::kRingBytes);
  uint64_t* empty_bar = full_bar + S::kStages;
  uint64_t* done_bar = empty_bar + S::kStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done_bar + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = p.split;
  const bool splits = S::kTiles == 1 && split > 1;
  const int features = LAYOUT == kEven ? p.features : S::kFeatures;
  const int w_bytes = LAYOUT == kEven ? features * kSkRow : S::kWBytes, block_bytes = w_bytes + S::kXBytes;
  const int stages = LAYOUT == kEven ? S::even_stages(features) : splits ? S::kSplitStages : S::kStages;
  const int rank = splits ? static_cast<int>(cluster_rank()) : 0;
  const int n0 = static_cast<int>(blockIdx.x) / split * features;
  const int num_kb = (p.K + kSkK - 1) / kSkK;
  const int kb_lo = rank * num_kb / split, kb_hi = (rank + 1) * num_kb / split;

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmap_w);
    tma_prefetch_desc(&tmap_x);
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    mbar_init(done_bar, 1);
    fence_barrier_init();
    fence_proxy_async();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, S::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (S::kPush && splits) cluster_arrive();  // waited for ahead of the first store to another CTA: it runs by then
  const uint32_t tmem = *tmem_slot;
  chain_start_next();

  // TMEM lanes [32 * (warp & 3), +32) belong to an epilogue warp; a thread owns one feature.
  const int feature = (warp & 3) * 32 + lane;
  OutT* out = static_cast<OutT*>(p.C) + n0 + feature;
  // C of up to 16 rows is read while the products run: rows rank, rank + split, ...
  constexpr int kEarlyC = BN <= 16 && S::kTiles == 1 ? 16 : 1;
  float before[kEarlyC];

  bool ok = true;
  if (warp == 0) {
    if (elect_one()) {
      auto block_at = [&](int stage, int j) { return smem + (stage * kGroup + j) * block_bytes; };
      auto load_w = [&](int stage, int kb) {
        const int blocks = kb_hi - kb < kGroup ? kb_hi - kb : kGroup;
        mbar_arrive_expect_tx(&full_bar[stage], blocks * block_bytes);
#pragma unroll
        for (int j = 0; j < kGroup; ++j) {
          if (j >= blocks) break;
          uint8_t* sw = block_at(stage, j);
          const int k0 = (kb + j) * kSkK;
          if constexpr (LAYOUT == kEven) {
            tma_load_2d(sw, &tmap_w, &full_bar[stage], k0, n0);  // all features
          } else if constexpr (!W_MN) {
#pragma unroll
            for (int t = 0; t < S::kTiles; ++t)
              tma_load_2d(sw + t * (kSkTile * kSkRow), &tmap_w, &full_bar[stage], k0, n0 + t * kSkTile);
          } else {
            // (A box that starts beyond the last feature reads the fill value like any other out-of-range column.)
#pragma unroll
            for (int i = 0; i < S::kFeatures / 64; ++i)
              tma_load_2d(sw + i * 8192, &tmap_w, &full_bar[stage], n0 + i * 64, k0);
          }
        }
      };
      // The stages are empty at the start: in a chained launch with resident weights they fill with weights while the
      // kernels before this one still run, and only X waits for them.
      const int early = p.w_resident ? min((kb_hi - kb_lo + kGroup - 1) / kGroup, stages) : 0;
      for (int i = 0; i < early; ++i) load_w(i, kb_lo + i * kGroup);
      chain_wait();
      int stage = 0;
      uint32_t phase = 0;
      for (int kb = kb_lo; kb < kb_hi; kb += kGroup) {
        if (kb - kb_lo >= early * kGroup) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1, p.status, kStatusWaitTimeoutProducer)) break;
          load_w(stage, kb);
        }
#pragma unroll
        for (int j = 0; j < kGroup; ++j) {
          if (kb + j >= kb_hi) break;
          uint8_t* sx = block_at(stage, j) + w_bytes;
          const int k0 = (kb + j) * kSkK;
          if constexpr (!X_MN) {
            tma_load_2d(sx, &tmap_x, &full_bar[stage], k0, 0);
          } else {
#pragma unroll
            for (int i = 0; i < BN / 64; ++i) tma_load_2d(sx + i * 8192, &tmap_x, &full_bar[stage], i * 64, k0);
          }
        }
        if (++stage == stages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      chain_wait();
      constexpr uint32_t idesc = I::idesc(BN, W_MN ? 1 : 0, X_MN ? 1 : 0);
      int stage = 0;
      uint32_t phase = 0;
      bool fed = true;
      for (int kb = kb_lo; kb < kb_hi; kb += kGroup) {
        if (!mbar_wait(&full_bar[stage], phase, p.status, kStatusWaitTimeoutMma)) {
          fed = false;
          break;
        }
        tc_fence_after_sync();
#pragma unroll
        for (int j = 0; j < kGroup; ++j) {
          if (kb + j >= kb_hi) break;
          const uint32_t sw = smem_u32(smem + (stage * kGroup + j) * block_bytes);
          const uint32_t sx = sw + w_bytes;
#pragma unroll
          for (int k = 0; k < kSkRow / 32; ++k) {
            const uint64_t dx =
                X_MN ? umma_smem_desc(sx + k * 2048, 8192, 1024) : umma_smem_desc(sx + k * 32, 16, 1024);
#pragma unroll
            for (int t = 0; t < S::kTiles; ++t) {
              const uint32_t st = sw + t * (kSkTile * kSkRow);
              const uint64_t dw =
                  W_MN ? umma_smem_desc(st + k * 2048, 8192, 1024) : umma_smem_desc(st + k * 32, 16, 1024);
              I::mma(tmem + t * BN, dw, dx, idesc, (kb + j > kb_lo || k > 0) ? 1u : 0u);
            }
          }
        }
        if (kb + stages * kGroup < kb_hi) tc_commit(&empty_bar[stage]);  // a stage that is filled again
        if (++stage == stages) {
          stage = 0;
          phase ^= 1;
        }
      }
      if (fed) tc_commit(done_bar);
    }
  } else {
    chain_wait();  // ahead of the first read or write of C
    if (I::kWhole) {
      const int row = static_cast<int>(threadIdx.x) - 64;
      if (row < BN && row < p.M) x_scales[row] = p.x_scales[row];
    }
    if (kEarlyC > 1 && p.accumulate && n0 + feature < p.N) {
#pragma unroll
      for (int i = 0; i < kEarlyC; ++i)
        if (rank + i * split < p.M) before[i] = skinny_read(out + static_cast<int64_t>(rank + i * split) * p.ldc);
    }
    ok = mbar_wait_warp(done_bar, 0, p.status, kStatusWaitTimeoutEpilogue);
    if (I::kWhole) asm volatile("bar.sync 1, 128;" ::: "memory");  // of the epilogue's warps: the scales are there
  }
  __syncwarp();
  if (S::kPush && splits) cluster_wait();

  // All MMAs of this CTA have retired.  Partial sums of a split tile go to the CTA that finishes their row, or, where
  // they are too many for its inbox, to the own stages (which are free), to be fetched from there.
  const int own_rows = (p.M + split - 1) / split;
  float* part = reinterpret_cast<float*>(smem);
  const uint32_t inbox = smem_u32(smem + S::kRingBytes - S::kInboxBytes);
  if (warp >= 2 && ok) {
    tc_fence_after_sync();
#pragma unroll
    for (int t = 0; t < S::kTiles; ++t) {
      const uint32_t taddr = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + t * BN;
      const bool stores = n0 + t * kSkTile + feature < p.N && (LAYOUT != kEven || t * kSkTile + feature < features);
      const float w_scale = I::kWhole && stores ? p.w_scales[n0 + t * kSkTile + feature] : 0.f;
#pragma unroll 1
      for (int c = 0; c < BN; c += 16) {
        if (c >= p.M) break;
        uint32_t r[16];
        tmem_ld_32x16(taddr + c, r);
        tmem_ld_wait();
        if (splits && S::kPush) {
          int to = c % split, row = c / split;
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            if (c + j >= p.M) break;
            st_cluster_f32(inbox + ((rank * own_rows + row) * kSkTile + feature) * 4, to, __uint_as_float(r[j]));
            if (++to == split) to = 0, ++row;
          }
        } else if (splits) {
#pragma unroll
          for (int j = 0; j < 16; ++j) part[(c + j) * kSkTile + feature] = __uint_as_float(r[j]);
        } else if (stores) {
          OutT* dst = out + t * kSkTile + static_cast<int64_t>(c) * p.ldc;
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            if (c + j >= p.M) break;
            float v = I::value(__uint_as_float(r[j]), I::kWhole ? x_scales[c + j] : 0.f, w_scale);
            if (p.accumulate) v += kEarlyC > 1 ? before[j] : skinny_read(dst + j * p.ldc);
            skinny_write(dst + j * p.ldc, v);
          }
        }
      }
    }
  }
  if (splits) {
    cluster_sync_all();
    if (warp >= 2 && ok && n0 + feature < p.N) {
      const float w_scale = I::kWhole ? p.w_scales[n0 + feature] : 0.f;
      auto finish = [&](int i, int row, float old) {
        float v[kSkMaxSplit];
#pragma unroll
        for (int s = 0; s < kSkMaxSplit; ++s) {
          if (s >= split) v[s] = 0.f;
          else if (S::kPush) v[s] = ld_shared_f32(inbox + ((s * own_rows + i) * kSkTile + feature) * 4);
          else v[s] = ld_cluster_f32(smem_u32(part) + (row * kSkTile + feature) * 4, s);
        }
        float sum = v[0];
#pragma unroll
        for (int s = 1; s < kSkMaxSplit; ++s) sum = I::add(sum, v[s]);
        sum = I::value(sum, I::kWhole ? x_scales[row] : 0.f, w_scale);
        skinny_write(out + static_cast<int64_t>(row) * p.ldc, p.accumulate ? sum + old : sum);
      };
      if constexpr (kEarlyC > 1) {
#pragma unroll
        for (int i = 0; i < kEarlyC / 2; ++i)
          if (rank + i * split < p.M) finish(i, rank + i * split, before[i]);
      } else {
#pragma unroll 4
        for (int row = rank, i = 0; row < p.M; row += split, ++i)
          finish(i, row, p.accumulate ? skinny_read(out + static_cast<int64_t>(row) * p.ldc) : 0.f);
      }
    }
    if (!S::kPush) cluster_sync_all();  // a CTA's shared memory outlives its readers
  }

  tc_fence_before_sync();
  const int gave_up = __syncthreads_or(!ok);
  if (warp == 1) {
    if (gave_up) {
      // A wait gave up (whichever it was, the epilogue's did, too): let copies that may still be in flight land before
      // the CTA exits.
      for (int i = 0; i < 2000; ++i) __nanosleep(1000);
    }
    tc_fence_after_sync();
    tmem_dealloc(tmem, S::kTmemCols);
  }
}

// CTAs of clusters of `split` that the GPU holds at once (GPCs hold whole clusters only).
template <typename Kernel>
static int resident_ctas(Kernel kernel, int smem, int split, std::atomic<int>* cache) {
  int n = cache[split].load(std::memory_order_relaxed);
  if (n > 0) return n;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(split));
  cfg.blockDim = dim3(kSkThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {static_cast<unsigned>(split), 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int clusters = 0;
  if (cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) != cudaSuccess || clusters < 1) {
    cudaGetLastError();
    clusters = 1;
  }
  cache[split].store(clusters * split, std::memory_order_relaxed);
  return clusters * split;
}

template <int BN, SkinnyLayout LAYOUT, bool X_MN, bool W_MN, typename OutT, typename In>
struct SkinnyKernel {
  using S = SkinnyCfg<BN, LAYOUT>;
  static constexpr auto kernel = gemm_skinny_kernel<BN, LAYOUT, X_MN, W_MN, OutT, In>;

  static bool configure() {
    static OptIn opt_in;
    return opt_in.done(kernel, S::kSmem);
  }

  // Expected time in us of N features cut into `split` slices of `num_kb` k-blocks: what a k-block takes at the slowest
  // of an SM's port to the L2 (110 GB/s), the thread that issues its MMAs (0.21 us a tile, more for many rows) and the
  // memory that all CTAs share; every wave starts and drains, and a split pays for its hand-over, an uneven cluster a
  // little more.  Fitted to chained launches of every split and layout over N of 640 to 32768, K of 1024 to 14336 and 1
  // to 100 rows: the choice is 2 % behind the fastest on average (6 % with the constants of the kernel before this
  // one).
  static float cost(int N, int num_kb, int split, int features = S::kFeatures) {
    static std::atomic<int> cache[kSkMaxSplit + 1];
    const int ctas = (N + features - 1) / features * split;
    const int resident = resident_ctas(kernel, S::kSmem, split, cache);
    const float sms = static_cast<float>(resident_ctas(kernel, S::kSmem, 1, cache)) / S::kResident;
    const int waves = (ctas + resident - 1) / resident;
    const int stages = ((num_kb + split - 1) / split + S::kGroup - 1) / S::kGroup;
    const float at_once = static_cast<float>(ctas < resident ? ctas : resident);
    const float port = (features * kSkRow + S::kXBytes) * fmaxf(1.f, at_once / sms) / 1.1e5f;
    const float memory = at_once * (features * kSkRow) / 7.1e6f;
    const float issue = (BN > 16 ? 0.23f : 0.21f) * S::kTiles;
    const float work = static_cast<float>(stages * S::kGroup) * fmaxf(fmaxf(port, memory), issue);
    const float rows = S::kPush ? 0.01f * BN : 0.13f * BN / split;
    const float meet = 1.5f + 0.15f * split + rows + ((split & (split - 1)) != 0 ? 0.15f : 0.f);
    return static_cast<float>(waves) * (work + 1.25f) + (split > 1 ? meet : 0.f);
  }

  // Of a CTA, for as many waves as kFeatures would take.
  static int even_features(int N) {
    static std::atomic<int> cache[2];
    const int sms = resident_ctas(kernel, S::kSmem, 1, cache), most = sms * S::kFeatures;
    const int ctas = (N + most - 1) / most * sms;
    return ((N + ctas - 1) / ctas + 7) / 8 * 8;
  }

  static int launch(const CUtensorMap& tw, const CUtensorMap& tx, const SkinnyGemmParams& p, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    const int features = LAYOUT == kEven ? p.features : S::kFeatures;
    cfg.gridDim = dim3(static_cast<unsigned>((p.N + features - 1) / features * p.split));
    cfg.blockDim = dim3(kSkThreads);
    cfg.dynamicSmemBytes = S::kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {static_cast<unsigned>(p.split), 1, 1};
    cfg.attrs = attr;
    cfg.numAttrs = static_cast<unsigned>(chain_attribute(attr, p.split > 1 ? 1 : 0));
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, tw, tx, p);
    if (e != cudaSuccess) {
      fprintf(stderr, "axb skinny gemm: launch failed: %s\n", cudaGetErrorString(e));
      return -4;
    }
    return 0;
  }
};

// The cheapest layout and split, and kEven's features; `forced` split (0 = free).
template <int BN, bool X_MN, bool W_MN, typename OutT, typename In = __nv_bfloat16>
static bool skinny_plan(int N, int K, int forced, int* split, SkinnyLayout* layout, int* features) {
  constexpr SkinnyLayout kBoth = SkinnyIn<In>::kWhole ? kEven : kWide;
  using Pair = SkinnyKernel<BN, kPair, X_MN, W_MN, OutT, In>;
  using Deep = SkinnyKernel<BN, kDeep, X_MN, W_MN, OutT, In>;
  using Both = SkinnyKernel<BN, kBoth, X_MN, W_MN, OutT, In>;
  if (!Deep::configure() || !Pair::configure() || !Both::configure()) return false;
  *features = kBoth == kEven ? Both::even_features(N) : 2 * kSkTile;
  constexpr int kSkK = SkinnyIn<In>::kK;
  const int num_kb = (K + kSkK - 1) / kSkK;
  float best = 0.f;
  *split = 0;
  auto consider = [&](float cost, int s, SkinnyLayout l) {
    if (*split != 0 && cost >= best) return;
    best = cost;
    *split = s;
    *layout = l;
  };
  for (int s = 1; s <= kSkMaxSplit && s <= num_kb; ++s) {
    if (forced > 0 ? s != forced : (s > 1 && num_kb / s < 2)) continue;
    consider(Deep::cost(N, num_kb, s), s, kDeep);
    consider(Pair::cost(N, num_kb, s), s, kPair);
    if (s == 1 && *features > kSkTile) consider(Both::cost(N, num_kb, 1, *features), 1, kBoth);
  }
  return *split > 0;
}

template <int BN, bool X_MN, bool W_MN, typename OutT, typename In = __nv_bfloat16>
static int launch_skinny(const void* X, const void* W, int64_t ldx, int64_t ldw, SkinnyGemmParams p,
                         cudaStream_t stream) {
  SkinnyLayout layout = kPair;
  if (!skinny_plan<BN, X_MN, W_MN, OutT, In>(p.N, p.K, p.split, &p.split, &layout, &p.features)) return -15;
  CUtensorMap tw, tx;
  constexpr int kSkK = SkinnyIn<In>::kK;
  const uint64_t k = static_cast<uint64_t>(p.K), n = static_cast<uint64_t>(p.N), m = static_cast<uint64_t>(p.M);
  const uint64_t wdims[2] = {W_MN ? n : k, W_MN ? k : n};
  const uint64_t wstride[1] = {static_cast<uint64_t>(ldw) * sizeof(In)};
  const uint32_t wbox[2] = {W_MN ? 64 : kSkK, static_cast<uint32_t>(W_MN ? kSkK : layout == kEven ? p.features : kSkTile)};
  int rc = make_tensor_map(&tw, SkinnyIn<In>::kType, 2, W, wdims, wstride, wbox,
                           CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc != 0) return rc;
  static_assert(!X_MN || BN >= 64, "an M-major tile of X is at least one 128-byte row wide");
  const uint64_t xdims[2] = {X_MN ? m : k, X_MN ? k : m};
  const uint64_t xstride[1] = {static_cast<uint64_t>(ldx) * sizeof(In)};
  const uint32_t xbox[2] = {X_MN ? 64 : kSkK, X_MN ? static_cast<uint32_t>(kSkK) : static_cast<uint32_t>(BN)};
  rc = make_tensor_map(&tx, SkinnyIn<In>::kType, 2, X, xdims, xstride, xbox, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc != 0) return rc;
  switch (layout) {
    case kDeep: return SkinnyKernel<BN, kDeep, X_MN, W_MN, OutT, In>::launch(tw, tx, p, stream);
    case kWide:
    case kEven: return SkinnyKernel<BN, SkinnyIn<In>::kWhole ? kEven : kWide, X_MN, W_MN, OutT, In>::launch(tw, tx, p, stream);
    default: return SkinnyKernel<BN, kPair, X_MN, W_MN, OutT, In>::launch(tw, tx, p, stream);
  }
}

}  // namespace axb

// Chains the launches of the calling thread (chain.cuh) from here on; returns the previous setting.
extern "C" int axb_chain_launches(int on) {
  const int before = axb::chain_launches ? 1 : 0;
  axb::chain_launches = on != 0;
  return before;
}

// K slices that the kernel would choose for a problem with K-major X and N-major W (1 = no split).
extern "C" int axb_gemm_splitk_plan(int M, int N, int K) {
  using namespace axb;
  int split = 1, features = 0;
  SkinnyLayout layout;
  bool ok;
  if (M <= 16) ok = skinny_plan<16, false, true, __nv_bfloat16>(N, K, 0, &split, &layout, &features);
  else if (M <= 32) ok = skinny_plan<32, false, true, __nv_bfloat16>(N, K, 0, &split, &layout, &features);
  else if (M <= 64) ok = skinny_plan<64, false, true, __nv_bfloat16>(N, K, 0, &split, &layout, &features);
  else if (M <= 128) ok = skinny_plan<128, false, true, __nv_bfloat16>(N, K, 0, &split, &layout, &features);
  else ok = false;
  return ok ? split : 1;
}

// C[M, N] (bf16 or fp32, row pitch ldc) = X * W (+ C when accumulate), M <= 128.
//   x_mn_major = 0: X is [M, K] row-major (pitch ldx);         1: X is stored [K, M] row-major.
//   w_mn_major = 0: W is stored [N, K] row-major (pitch ldw);  1: W is [K, N] row-major.
// `w_resident`: W is not written by what runs before it on the stream (weights); counts in chained launches only.
// `split`: K slices per tile, 0 = the kernel's own choice.  Alignment as for axb_gemm_bf16; -20 = not one of mine.
extern "C" int axb_gemm_skinny(const void* X, const void* W, void* C, int M, int N, int K, int64_t ldx, int64_t ldw,
                               int64_t ldc, int x_mn_major, int w_mn_major, int out_fp32, int accumulate, int split,
                               int w_resident, int* status, cudaStream_t stream) {
  using namespace axb;
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  // One wave of two-tile CTAs at most: beyond it the persistent 256-column tiles of gemm.cu, which overlap a tile's
  // epilogue with the next tile's stream, are faster (64 x 128256 x 2048: 89 us, here 102; 32 x 40960 x 4096: 71 and
  // 79).  Above 64 rows X weighs as much as W in every stage, and they win as soon as they fill half the SMs
  // (128 x 12288 x 4096: 23.2 and 24.5; 128 x 4096 x 4096: 20.7 and 15.7).
  if (M > 128 || N > (M <= 64 ? 148 * 256 : 8192)) return -20;
  if ((ldx % 8) || (ldw % 8) || (reinterpret_cast<uintptr_t>(X) & 15) || (reinterpret_cast<uintptr_t>(W) & 15) ||
      (reinterpret_cast<uintptr_t>(C) & 15) || (ldc % (out_fp32 ? 4 : 8)))
    return -10;
  if (split < 0 || split > kSkMaxSplit || split > (K + SkinnyIn<__nv_bfloat16>::kK - 1) / SkinnyIn<__nv_bfloat16>::kK) return -15;
  const SkinnyGemmParams p{M, N, K, C, ldc, status, accumulate, split, w_resident && chain_launches ? 1 : 0, nullptr, nullptr, 0};
#define AXB_SKINNY_BN(BN, XM, WM, T) return launch_skinny<BN, XM, WM, T>(X, W, ldx, ldw, p, stream)
#define AXB_SKINNY(WM, T)                                  \
  do {                                                     \
    if (x_mn_major && M <= 64) AXB_SKINNY_BN(64, true, WM, T); \
    if (x_mn_major) AXB_SKINNY_BN(128, true, WM, T);       \
    if (M <= 16) AXB_SKINNY_BN(16, false, WM, T);          \
    if (M <= 32) AXB_SKINNY_BN(32, false, WM, T);          \
    if (M <= 64) AXB_SKINNY_BN(64, false, WM, T);          \
    AXB_SKINNY_BN(128, false, WM, T);                      \
  } while (0)
  if (w_mn_major) {
    if (out_fp32) AXB_SKINNY(true, float);
    AXB_SKINNY(true, __nv_bfloat16);
  }
  if (out_fp32) AXB_SKINNY(false, float);
  AXB_SKINNY(false, __nv_bfloat16);
#undef AXB_SKINNY
#undef AXB_SKINNY_BN
}

// y[M, N] (bf16) = x_scales[m] w_scales[n] sum_k x[m, k] w[n, k] (+ y when accumulate) of 8-bit whole numbers, x [M, K] and w [N, K]
// one row behind the other and 16-byte aligned, M <= 128, K a multiple of 16.  The weight's bytes bound it: 1 x 4096 x 28672 22.4 us
// (18.0 at the copy rate), 16 x 14336 x 4096 with the rows' own kernel 15.0 (9.1), 2 of each a launch and its first loads.
// `plan`: slices of K; `resident`: as above.
extern "C" int axb_gemm_skinny_int8(const axb::Int8LinearCall* call, cudaStream_t stream) {
  using namespace axb;
  const Int8LinearCall& a = *call;
  if (a.M <= 0 || a.N <= 0 || a.K <= 0) return 0;
  if (a.M > 128) return -20;
  if (a.N > 0x40000000 || a.K > (1 << 17) || a.K % 16 || (reinterpret_cast<uintptr_t>(a.x) & 15) ||
      (reinterpret_cast<uintptr_t>(a.w) & 15) || (reinterpret_cast<uintptr_t>(a.y) & 1))
    return -10;
  if (a.plan < 0 || a.plan > kSkMaxSplit || a.plan > (a.K + SkinnyIn<int8_t>::kK - 1) / SkinnyIn<int8_t>::kK) return -15;
  const int M = static_cast<int>(a.M);
  const SkinnyGemmParams p{M, static_cast<int>(a.N), static_cast<int>(a.K), a.y, a.N, a.status, a.accumulate != 0,
                           static_cast<int>(a.plan), a.resident && chain_launches ? 1 : 0, a.x_scales, a.w_scales, 0};
  if (M <= 16) return launch_skinny<16, false, false, __nv_bfloat16, int8_t>(a.x, a.w, a.K, a.K, p, stream);
  if (M <= 32) return launch_skinny<32, false, false, __nv_bfloat16, int8_t>(a.x, a.w, a.K, a.K, p, stream);
  if (M <= 64) return launch_skinny<64, false, false, __nv_bfloat16, int8_t>(a.x, a.w, a.K, a.K, p, stream);
  return launch_skinny<128, false, false, __nv_bfloat16, int8_t>(a.x, a.w, a.K, a.K, p, stream);
}
